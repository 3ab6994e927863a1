// Rounding to MXFP4, shared by the quantizing kernels (mxfp4_cast.hip,
// gemm_mxfp4_skinny.hip).
#pragma once

#include "mfma.h"

namespace ntops {

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

// fp32 value of scale byte s (< 255): 2^(s - 127).
__device__ __forceinline__ float scale_value(uint32_t s) {
  return __builtin_bit_cast(float, s == 0 ? 0x00400000u : s << 23);
}

// Scale byte of a block whose largest |x| has these fp32 bits: floor(log2) is its
// exponent field less 127, so e + 127 is that field less 2; 255 for what is not
// finite.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  const uint32_t exponent = top >> 23;
  return exponent == 255 ? 255 : exponent > 2 ? exponent - 2 : 0;
}

// 8 values to 8 codes (value i in nibble i) under `scale`.
template <typename T>
__device__ __forceinline__ uint32_t codes8(const T (&v)[8], float scale) {
  uint32_t r = 0;
  if constexpr (std::is_same<T, __bf16>::value) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, bf16x2_t{v[0], v[1]}, scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, bf16x2_t{v[2], v[3]}, scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, bf16x2_t{v[4], v[5]}, scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, bf16x2_t{v[6], v[7]}, scale, 3);
  } else if constexpr (std::is_same<T, _Float16>::value) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, f16x2_t{v[0], v[1]}, scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, f16x2_t{v[2], v[3]}, scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, f16x2_t{v[4], v[5]}, scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, f16x2_t{v[6], v[7]}, scale, 3);
  } else {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], scale, 3);
  }
  return r;
}

// A whole block of 32 16-bit values: its codes and, in s, its scale byte.
template <typename T>
__device__ __forceinline__ u32x4 quantize32(const u32x4 (&x)[4], uint32_t& s) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  u16x2 most = {0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, x[i >> 2][i & 3] & 0x7fff7fffu));
  const uint16_t top = max(most.x, most.y);
  s = scale_byte(__builtin_bit_cast(uint32_t, static_cast<float>(__builtin_bit_cast(T, top))));
  const float scale = scale_value(s == 255 ? 127 : s);
  u32x4 c;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    T v[8];
    __builtin_memcpy(v, &x[i], 16);
    c[i] = s == 255 ? 0 : codes8<T>(v, scale);
  }
  return c;
}

}  // namespace ntops
