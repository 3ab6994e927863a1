// Shared by the attention kernels (attention.hip, attn_decode.hip).
#pragma once

#include "mfma.h"

namespace ntops {

struct AttnArgs {
  const void* q;
  const void* k;
  const void* v;
  const void* mask;
  void* o;
  int64_t qs[4], ks[4], vs[4], ms[4], os[4];
  int B, Hq, Hkv, Sq, Skv, D;
  int mask_dtype;    // -1: none; NTOPS_BOOL (true = attend), NTOPS_F32 / F16 / BF16 (additive)
  int causal;        // 0: none, 1: upper-left (kv <= q), 2: lower-right (kv <= q + Skv - Sq)
  float scale_log2;  // scale * log2(e)
};

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float neg_inf() { return -__builtin_huge_valf(); }

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Chunk slot of 16-byte chunk c of key row r in the V tile ([kv][d] with
// D / 8 chunks per row), conflict-free for the transposing fragment reads.
template <int D>
__device__ __forceinline__ int vslot(int r, int c) {
  if constexpr (D == 128)
    return mnslot(r, c);
  else
    return c ^ (((r >> 1) & 1) << 2);
}

// max(a, b, c) in one instruction, without the NaN-quieting moves the
// compiler puts in front of fmaxf in IEEE mode (a NaN operand may be
// dropped; a NaN score still reaches the output through its exponential).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// From here on a result cut to [0, 1] keeps a NaN (it is 0 by default): the
// wave's MODE register, bit 8 (DX10_CLAMP).
__device__ __forceinline__ void clamp_keeps_nan() { __builtin_amdgcn_s_setreg(1 | 8 << 6 | 0 << 11, 0); }

// B fragment of S = Q K^T: key rows n0 .. n0 + 31 (lane l: row n0 + (l & 31)),
// d = 16 ks + 8 (l >> 5) .. + 7.
template <int D>
__device__ __forceinline__ u32x4 k_frag(const char* tile, int n0, int ks, int lane) {
  const int r = n0 + (lane & 31);
  const int c = ks * 2 + (lane >> 5);
  return *reinterpret_cast<const u32x4*>(tile + r * (D * 2) + kslot<D>(r, c) * 16);
}

// B fragment of O += P V for the 16-key slice sl and output columns
// n0 .. n0 + 31: lane l receives column n0 + (l & 31) at keys
// 16 sl + 4 (l >> 5) + 0..3 (elements 0..3) and 16 sl + 8 + 4 (l >> 5) + 0..3
// (elements 4..7) -- the key order in which the S accumulator holds P.
template <int D>
__device__ __forceinline__ u32x4 v_frag(const char* tile, int n0, int sl, int lane) {
  const int i = lane & 15;
  const int n = n0 + ((lane >> 4) & 1) * 16 + (i & 3) * 4;
  const int c = n >> 3, half = (n >> 2) & 1;
  s16x4 v[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int k = sl * 16 + h * 8 + (lane >> 5) * 4 + (i >> 2);
    const char* p = tile + k * (D * 2) + vslot<D>(k, c) * 16 + half * 8;
    v[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(p));
  }
  u32x4 r;
  r.x = static_cast<uint16_t>(v[0][0]) | (static_cast<uint32_t>(static_cast<uint16_t>(v[0][1])) << 16);
  r.y = static_cast<uint16_t>(v[0][2]) | (static_cast<uint32_t>(static_cast<uint16_t>(v[0][3])) << 16);
  r.z = static_cast<uint16_t>(v[1][0]) | (static_cast<uint32_t>(static_cast<uint16_t>(v[1][1])) << 16);
  r.w = static_cast<uint16_t>(v[1][2]) | (static_cast<uint32_t>(static_cast<uint16_t>(v[1][3])) << 16);
  return r;
}

// True when attn_decode serves this problem: 16-bit data whose head dim and
// rows suit the matrix cores, no explicit mask, at most 16 query rows per key
// / value head, and more than kDecodeMinKeys keys -- or any but none, where
// every CU gets a key / value head.
bool attn_decode_serves(const AttnArgs& a);
// Bytes of workspace with which attn_decode splits the keys over more blocks
// (0: one block per key / value head is as good).
int64_t attn_decode_workspace(int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t Skv, int64_t D);
// Runs it; a missing or short workspace runs one block per key / value head.
int attn_decode(int dtype, const AttnArgs& a, void* workspace, int64_t workspace_bytes, hipStream_t st);

}  // namespace ntops
