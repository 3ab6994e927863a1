// Shared by the MXFP4 product's kernels (gemm_mxfp4*.hip): out = A B^T (+ a
// bias row) for A (M, K) and B (N, K) of 4-bit codes with a scale byte per 32.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 on 4-bit data: lane l holds the 16 bytes
// (32 codes, one block) of row l & 15 and k block l >> 4 of A / B, and that
// block's scale in one byte of a register, which the instruction selects; of the
// result it holds column l & 15 and rows 4 (l >> 4) .. + 3.
//
// Blocks keep their order in the LDS: with neighbouring blocks in one lane, whose
// scales would be neighbouring bytes, the DMA's lanes gathered every second (or
// eighth) 16 bytes of a line: (16, 4096, 14336) 10.9 -> 13.1 us.
#pragma once

#include "mfma.h"

namespace ntops {

struct Mx4Args {
  const uint8_t* a;    // codes: 16 bytes a block
  const uint8_t* as;   // scales: a byte a block
  const uint8_t* b;
  const uint8_t* bs;
  const void* bias;    // N values of the output's type, or null
  void* d;
  int64_t lda, ldas, ldb, ldbs;  // row strides in bytes
  int64_t ldd;         // elements
  int M, N, kb;        // kb: blocks of 32 along K
  const void* x;       // A not yet quantized: 16-bit rows of K values, ldx apart (elements)
  int64_t ldx;
  int K;
  float* part;         // split K: fp32 partial products, slice s at s * M * N
  int split, kchunk;   // slices, and the blocks of each
};

typedef int i32x8 __attribute__((ext_vector_type(8)));

// c += A B over 4 blocks; SA / SB: the byte of sa / sb that holds the scales.
template <int SA, int SB>
__device__ __forceinline__ f32x4 mfma_mx4(u32x4 a, uint32_t sa, u32x4 b, uint32_t sb, f32x4 c) {
  // (4-bit data fills the first half of the 256-bit operands)
  const i32x8 x = {static_cast<int>(a.x), static_cast<int>(a.y), static_cast<int>(a.z), static_cast<int>(a.w), 0, 0, 0, 0};
  const i32x8 y = {static_cast<int>(b.x), static_cast<int>(b.y), static_cast<int>(b.z), static_cast<int>(b.w), 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, SA, static_cast<int>(sa), SB, static_cast<int>(sb));
}

// A lane's 4 consecutive columns n .. n + 3 of row m, rounded; whole: the output's
// rows are runs that 4 elements at a time can be stored to.
template <typename T>
__device__ __forceinline__ void store4(T* d, int64_t ldd, int m, int n, int M, int N, f32x4 v, const T* bias, bool whole) {
  if (m >= M) return;
  T* at = d + static_cast<int64_t>(m) * ldd + n;
  T o[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float b = bias != nullptr && n + e < N ? static_cast<float>(bias[n + e]) : 0.f;
    o[e] = static_cast<T>(v[e] + b);
  }
  if (whole && n + 4 <= N) {
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<u32x2*>(at) = __builtin_bit_cast(u32x2, o);
    else
      *reinterpret_cast<u32x4*>(at) = __builtin_bit_cast(u32x4, o);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < N) at[e] = o[e];
  }
}

// 16-bit out on 256 x 256 tiles, from 33 blocks of K on, with a workspace.
bool mx4_large_serves(int out_dtype, const Mx4Args& g);
int64_t mx4_large_workspace(int64_t M, int64_t N, int64_t kb);
int mx4_large(int out_dtype, Mx4Args g, void* workspace, hipStream_t st);

constexpr int kSkinnyRows = 32;
// out for M <= kSkinnyRows, bound by streaming B.
int mx4_skinny(int out_dtype, const Mx4Args& g, hipStream_t st);
// The same with A quantized by the blocks themselves (g.x), for up to kFusedRows
// rows.
constexpr int kFusedRows = 4;
int mx4_skinny_fused(int x_dtype, int out_dtype, const Mx4Args& g, hipStream_t st);

}  // namespace ntops
