// Shared by the attention kernels on a cache in 8 bits (attn_cache*.hip).
#pragma once

#include "attention.h"
#include "kv_cache.h"

namespace ntops {

struct CacheAttnArgs {
  const void* q;       // (B, Hq, Sq, D)
  const uint8_t* k;    // (B, Hkv, C, D) e4m3
  const uint8_t* v;
  const float* ks;     // (B, Hkv, blocks)
  const float* vs;
  void* o;
  int64_t qst[3], kst[3], vst[3], kss[2], vss[2], ost[3];
  const void* lengths;  // tokens of each sequence (null: C)
  int lengths_dtype;
  int64_t C;
  int B, Hq, Hkv, Sq, D, shift;  // a block of scales: 1 << shift tokens
  int causal;            // row i sees keys up to length - Sq + i
  float scale_log2;      // scale * log2(e)
};

// 8 probabilities as bf16 operands: rounded, as the 16-bit attention of this library
// rounds them, and for f16 queries, whose results keep 11 bits, what the rounding left
// as a second operand (17 bits in all).  Against 64 bits, relative to the whole result:
// bf16 prompts (4, 32 / 8, 2048 over 2048, 128) 0.0017, with fp32 probabilities, of
// which only the result's own rounding is left, 0.0014; (16, 32 / 8, 1 over 2048 ..
// 4096, 128) 0.0015 and 0.0015; f16 prompts 0.00018 and 0.00018.
template <bool LO>
__device__ __forceinline__ void pack_p(const float* x, u32x4& hi, u32x4& lo) {
  hi = pack8<__bf16>(x);
  if constexpr (LO) {
    float d[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t w = hi[e >> 1];
      d[e] = x[e] - __builtin_bit_cast(float, e & 1 ? w & 0xffff0000u : w << 16);
    }
    lo = pack8<__bf16>(d);
  }
}

// 1 in every byte of w that is a NaN of e4m3 (all of its low 7 bits set).
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  return (((w & 0x7f7f7f7fu) + 0x01010101u) >> 7) & 0x01010101u;
}
// Bits 0, 8, 16 and 24 as bits 0 .. 3.
__device__ __forceinline__ uint32_t byte_bits(uint32_t w) { return (w * 0x01020408u) >> 24; }

__device__ __forceinline__ int64_t length_of(const CacheAttnArgs& a, int b) {
  return max(int64_t(0), min(a.C, index_at(a.lengths, a.lengths_dtype, b, a.C)));
}

// Most query rows per cache head of cache_decode: with more, its registers are spent.
// 5 positions of 4 heads, bf16 of 128: (16, 32 / 8, 5, 2048 .. 4096) 30.7 us, by
// cache_tile 46.3; (1, 32 / 8, 8, 131000) 57.5 and 92.6; (64, 32 / 8, 8, 1024 .. 2048)
// 48.6 and 76.3.
constexpr int kDecodeRows = 32;

// 16-bit queries of head dims and layouts that the matrix cores' kernels read.
bool cache_matrix_layout(const CacheAttnArgs& a, int dtype);

// True when cache_decode serves this problem: such a layout, and at most kDecodeRows
// query rows per cache head.
bool cache_decode_serves(const CacheAttnArgs& a, int dtype);
// Bytes of workspace with which it spreads the keys over more blocks (0: one
// block per cache head is as good).
int64_t cache_decode_workspace(int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t C, int64_t D);
// Runs it; a missing or short workspace runs one block per cache head.
int cache_decode(int dtype, const CacheAttnArgs& a, void* workspace, int64_t workspace_bytes, hipStream_t st);

// The same for any number of query rows.
bool cache_tile_serves(const CacheAttnArgs& a, int dtype);
int64_t cache_tile_workspace(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t C, int64_t D);
int cache_tile(int dtype, const CacheAttnArgs& a, void* workspace, int64_t workspace_bytes, hipStream_t st);

// Combines the slices' partial results of every query row in slice order: part
// holds, per row (batch, head, position) and slice, the unnormalised O row, then
// for each the pair (max in base 2, sum).
void cache_merge(int dtype, const CacheAttnArgs& a, int nsplit, const float* part, hipStream_t st);

}  // namespace ntops
