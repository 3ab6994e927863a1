// MXFP4 (microscaled 4-bit floating point) and back.
//
// A row is cut into blocks of 32 values (the last padded with zeros).  With
// amax = max |x| of a block its scale is 2^e, e = max(-127, floor(log2 amax) -
// 2), kept as the byte e + 127; the values are x / 2^e rounded to the nearest
// of 0, .5, 1, 1.5, 2, 3, 4, 6 (ties to the even code) and cut at 6 (amax / 2^e
// lies in [4, 8)).  A block with a NaN or an infinity has the scale byte 255
// (NaN) and zero codes.  Every step but the one rounding is exact: a division
// by a power of two, the hardware's v_cvt_scalef32_pk_fp4.
//
// Bound by memory: es read and 17 / 32 written per value.  A lane takes 8
// values (one or two 16-byte loads, 4 bytes of codes), four neighbouring lanes
// a block, so the block's maximum is two DPP steps.  The exponent of amax is
// read off its bits: the largest |x| as an integer, under which a NaN is larger
// than an infinity and that than any number.  (14336, 4096) bf16 26.7 us (5.6 TB/s)
// and 27.1 back, fp32 48.0 and 66.4 (a lane's 32 bytes go out in two stores, half a
// line each); rows of 4095 bf16 28.1 and 30.7, where single accesses took 57.3 and
// 82.6.
#include <algorithm>

#include "mxfp4.h"

namespace ntops {
namespace {

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, false));
}

// 16 bytes at any address (the hardware takes them unaligned), as whole accesses.
typedef u32x4 u32x4_any __attribute__((aligned(2), may_alias));

template <typename T>
__device__ __forceinline__ void load8(const T* p, T (&v)[8]) {
  u32x4 raw[sizeof(T) / 2];
#pragma unroll
  for (int h = 0; h < static_cast<int>(sizeof(T)) / 2; ++h) raw[h] = reinterpret_cast<const u32x4_any*>(p)[h];
  __builtin_memcpy(v, raw, sizeof(v));
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const T (&v)[8]) {
  u32x4 raw[sizeof(T) / 2];
  __builtin_memcpy(raw, v, sizeof(v));
#pragma unroll
  for (int h = 0; h < static_cast<int>(sizeof(T)) / 2; ++h) reinterpret_cast<u32x4_any*>(p)[h] = raw[h];
}

// Index type I: 32 bits where every count fits.  Only the
// last values of a row whose length is no multiple of 8 go one by one.
template <typename T, typename I, int U>
__global__ __launch_bounds__(256) void k_quantize_mxfp4(const T* x, int64_t ld, I cols, I packs, I total,
                                                        uint32_t* codes, uint8_t* scales) {
  const I first = static_cast<I>(block_id()) * (256 * U) + threadIdx.x;
  T v[U][8];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const I p = first + u * 256;  // pack: 8 values, `packs` (a multiple of 4) a row
    const I row = p / packs, c = (p - row * packs) * 8;
    const T* at = x + static_cast<int64_t>(row) * ld + c;
    if (p < total && c + 8 <= cols) {
      load8(at, v[u]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[u][e] = p < total && c + e < cols ? at[e] : static_cast<T>(0.f);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const I p = first + u * 256;
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      top = max(top, __builtin_bit_cast(uint32_t, static_cast<float>(v[u][e])) & 0x7fffffffu);
    top = max(top, dpp_u32<kDppXor1>(top));  // (a block's four lanes are in a quad, whole waves active)
    top = max(top, dpp_u32<kDppXor2>(top));
    const uint32_t s = scale_byte(top);
    if (p < total) {
      codes[p] = s == 255 ? 0 : codes8<T>(v[u], scale_value(s));
      if ((threadIdx.x & 3) == 0) scales[p >> 2] = static_cast<uint8_t>(s);
    }
  }
}

// 8 codes to fp32 (each product with the power of two is exact).
template <typename T>
__device__ __forceinline__ void values8(uint32_t codes, uint32_t s, T (&v)[8]) {
  const float scale = s == 255 ? __builtin_nanf("") : 1.f;
  const float up = scale_value(s == 255 ? 127 : s);
  f32x2_t f[4];
  f[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 0);
  f[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 1);
  f[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 2);
  f[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 3);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = static_cast<T>(f[i].x * up * scale);
    v[2 * i + 1] = static_cast<T>(f[i].y * up * scale);
  }
}

template <typename T, typename I, int U>
__global__ __launch_bounds__(256) void k_dequantize_mxfp4(const uint32_t* codes, int64_t codes_ld,
                                                          const uint8_t* scales, int64_t scales_ld, I cols, I packs,
                                                          I total, T* y) {
  const I first = static_cast<I>(block_id()) * (256 * U) + threadIdx.x;
  uint32_t q[U], s[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const I p = first + u * 256;
    const I row = p / packs, c = p - row * packs;
    q[u] = p < total ? codes[static_cast<int64_t>(row) * codes_ld + c] : 0;
    s[u] = p < total ? scales[static_cast<int64_t>(row) * scales_ld + (c >> 2)] : 0;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const I p = first + u * 256;
    if (p >= total) continue;
    const I row = p / packs, c = (p - row * packs) * 8;
    T v[8];
    values8<T>(q[u], s[u], v);
    T* at = y + static_cast<int64_t>(row) * cols + c;
    if (c + 8 <= cols) {
      store8(at, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < cols) at[e] = v[e];
    }
  }
}

// Packs a lane takes: one while that leaves every CU a block, four from there on.
int lane_packs(int64_t total) { return total >= static_cast<int64_t>(cu_count_cached()) * 1024 * 4 ? 4 : 1; }

}  // namespace
}  // namespace ntops

using namespace ntops;

extern "C" int ntops_quantize_mxfp4(int dtype, int64_t rows, int64_t cols, const void* x, int64_t x_row_stride,
                                    void* codes, void* scales, void* stream) {
  if (rows < 0 || cols < 0) return set_error(NTOPS_ERR_INVALID, "quantize_mxfp4: negative size");
  return dispatch_float16_32(dtype, "quantize_mxfp4", [&](auto tag) -> int {
    using T = decltype(tag);
    if (rows == 0 || cols == 0) return NTOPS_OK;
    if (!x || !codes || !scales) return set_error(NTOPS_ERR_INVALID, "quantize_mxfp4: null pointer");
    if ((reinterpret_cast<uintptr_t>(codes) & 3u) != 0)
      return set_error(NTOPS_ERR_INVALID, "quantize_mxfp4: codes not aligned to 4 bytes");
    if (rows > (int64_t(1) << 56) / cols) return set_error(NTOPS_ERR_UNSUPPORTED, "quantize_mxfp4: too many values");
    int64_t r = rows, c = cols;
    if (c % 32 == 0 && (x_row_stride == c || r == 1)) {  // one long row: the same blocks
      c *= r;
      r = 1;
    }
    const int64_t packs = ceil_div(c, 32) * 4, total = r * packs;
    const int u = lane_packs(total);
    const int64_t blocks = ceil_div(total, 256 * u);
    if (blocks > (int64_t(1) << 31)) return set_error(NTOPS_ERR_UNSUPPORTED, "quantize_mxfp4: too many values");
    const auto go = [&](auto index, auto utag) {
      using I = decltype(index);
      constexpr int U = decltype(utag)::value;
      hipLaunchKernelGGL((k_quantize_mxfp4<T, I, U>), blocks_2d(blocks), dim3(256), 0,
                         static_cast<hipStream_t>(stream), static_cast<const T*>(x), x_row_stride, static_cast<I>(c),
                         static_cast<I>(packs), static_cast<I>(total), static_cast<uint32_t*>(codes),
                         static_cast<uint8_t*>(scales));
      return check_launch("quantize_mxfp4");
    };
    const auto pick = [&](auto index) {
      return u == 4 ? go(index, std::integral_constant<int, 4>{}) : go(index, std::integral_constant<int, 1>{});
    };
    return total * 8 + 65536 < (int64_t(1) << 31) ? pick(uint32_t{}) : pick(int64_t{});
  });
}

extern "C" int ntops_dequantize_mxfp4(int dtype, int64_t rows, int64_t cols, const void* codes, int64_t codes_row_stride,
                                      const void* scales, int64_t scales_row_stride, void* y, void* stream) {
  if (rows < 0 || cols < 0) return set_error(NTOPS_ERR_INVALID, "dequantize_mxfp4: negative size");
  return dispatch_float16_32(dtype, "dequantize_mxfp4", [&](auto tag) -> int {
    using T = decltype(tag);
    if (rows == 0 || cols == 0) return NTOPS_OK;
    if (!y || !codes || !scales) return set_error(NTOPS_ERR_INVALID, "dequantize_mxfp4: null pointer");
    if ((reinterpret_cast<uintptr_t>(codes) & 3u) != 0 || codes_row_stride % 4 != 0)
      return set_error(NTOPS_ERR_INVALID, "dequantize_mxfp4: codes not aligned to 4 bytes");
    if (rows > (int64_t(1) << 56) / cols) return set_error(NTOPS_ERR_UNSUPPORTED, "dequantize_mxfp4: too many values");
    int64_t r = rows, c = cols;
    if (c % 32 == 0 && (r == 1 || (codes_row_stride == c / 2 && scales_row_stride == c / 32))) {
      c *= r;
      r = 1;
    }
    const int64_t packs = ceil_div(c, 8), total = r * packs;
    const int u = lane_packs(total);
    const int64_t blocks = ceil_div(total, 256 * u);
    if (blocks > (int64_t(1) << 31)) return set_error(NTOPS_ERR_UNSUPPORTED, "dequantize_mxfp4: too many values");
    const auto go = [&](auto index, auto utag) {
      using I = decltype(index);
      constexpr int U = decltype(utag)::value;
      hipLaunchKernelGGL((k_dequantize_mxfp4<T, I, U>), blocks_2d(blocks), dim3(256), 0,
                         static_cast<hipStream_t>(stream), static_cast<const uint32_t*>(codes), codes_row_stride / 4,
                         static_cast<const uint8_t*>(scales), scales_row_stride, static_cast<I>(c),
                         static_cast<I>(packs), static_cast<I>(total), static_cast<T*>(y));
      return check_launch("dequantize_mxfp4");
    };
    const auto pick = [&](auto index) {
      return u == 4 ? go(index, std::integral_constant<int, 4>{}) : go(index, std::integral_constant<int, 1>{});
    };
    return total * 8 + 65536 < (int64_t(1) << 31) ? pick(uint32_t{}) : pick(int64_t{});
  });
}
