// Shared by the kernels on a key / value cache held in 8 bits (kv_cache.hip,
// attn_cache*.hip): e4m3 values under an fp32 scale for each block of
// consecutive tokens of a head.
#pragma once

#include "mfma.h"

namespace ntops {

// Element i of an I32 / I64 index vector (null: `other`).
__device__ __forceinline__ int64_t index_at(const void* p, int dtype, int64_t i, int64_t other) {
  if (p == nullptr) return other;
  return dtype == NTOPS_I32 ? static_cast<const int32_t*>(p)[i] : static_cast<const int64_t*>(p)[i];
}

typedef float f32x2 __attribute__((ext_vector_type(2)));

// 8 e4m3 values to fp32.
__device__ __forceinline__ void from_e4m3(u32x2 c, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(c[i]), false);
    const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(c[i]), true);
    v[4 * i] = lo.x;
    v[4 * i + 1] = lo.y;
    v[4 * i + 2] = hi.x;
    v[4 * i + 3] = hi.y;
  }
}

// 8 fp32 values, each at most 448 in magnitude or not finite, to e4m3 (nearest,
// ties to even; what is not finite becomes NaN).
__device__ __forceinline__ u32x2 to_e4m3(const float (&v)[8]) {
  u32x2 c;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], w, true);
    c[i] = static_cast<uint32_t>(w);
  }
  return c;
}

inline bool index_dtype(int dt) { return dt == NTOPS_I32 || dt == NTOPS_I64; }
// Tokens of a block of scales: a power of two from 16 on (a matrix
// instruction's 16 keys then share a scale).
inline bool block_ok(int64_t block) { return block >= 16 && block <= (1 << 24) && (block & (block - 1)) == 0; }

}  // namespace ntops
