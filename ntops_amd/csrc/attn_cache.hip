// Attention over a key / value cache held in 8 bits: the kernel for any head dim
// and layout, and the C entry points.
//
//   O = softmax(scale Q K^T) V over the first n tokens of a sequence's cache, K
//   = k8 ks, V = v8 vs with a scale of each for every block of tokens; causal:
//   row i sees the keys up to n - Sq + i (the last query row is the last token).
//   A row that sees no key is 0.
//
// The scale of a key's block multiplies its score, that of a value's block its
// probability, both in fp32, so the cache is never expanded.
#include <algorithm>

#include "attn_cache.h"

namespace ntops {
namespace {

// One wave per query row: 64 keys at a time, a lane a key for the scores and a
// lane every 64th column for P V.  For head dims and layouts that the matrix
// cores' kernels do not take, and fp32 queries.
constexpr int kMaxDim = 256;
constexpr int64_t kMaxCount = 0x7fffffff;

template <typename T>
__global__ __launch_bounds__(64) void k_cache_attn_rows(CacheAttnArgs a) {
  __shared__ float q[kMaxDim];
  const int lane = threadIdx.x;
  const int64_t row = block_id();
  if (row >= static_cast<int64_t>(a.B) * a.Hq * a.Sq) return;
  const int i = static_cast<int>(row % a.Sq);
  const int64_t bh = row / a.Sq;
  const int b = static_cast<int>(bh / a.Hq), h = static_cast<int>(bh % a.Hq);
  const int hk = h / (a.Hq / a.Hkv);
  const T* Q = static_cast<const T*>(a.q) + b * a.qst[0] + h * a.qst[1] + i * a.qst[2];
  const uint8_t* K = a.k + b * a.kst[0] + hk * a.kst[1];
  const uint8_t* V = a.v + b * a.vst[0] + hk * a.vst[1];
  const float* KS = a.ks + b * a.kss[0] + hk * a.kss[1];
  const float* VS = a.vs + b * a.vss[0] + hk * a.vss[1];
  for (int d = lane; d < a.D; d += 64) q[d] = static_cast<float>(Q[d]);
  __syncthreads();
  const int64_t n = length_of(a, b);
  const int64_t end = a.causal ? max(int64_t(0), n - a.Sq + i + 1) : n;
  float m = neg_inf(), l = 0.f;
  float o[kMaxDim / 64] = {};
  for (int64_t k0 = 0; k0 < end; k0 += 64) {
    const int64_t key = k0 + lane;
    float s = neg_inf(), vscale = 0.f;
    if (key < end) {
      const uint8_t* kr = K + key * a.kst[2];
      float dot = 0.f;
      for (int d = 0; d < a.D; ++d) dot = fmaf(q[d], __builtin_amdgcn_cvt_f32_fp8(kr[d], 0), dot);
      s = dot * KS[key >> a.shift] * a.scale_log2;
      vscale = VS[key >> a.shift];
    }
    const float m_new = fmaxf(m, wave_max(s));
    const float m_use = m_new == neg_inf() ? 0.f : m_new;
    const float alpha = fast_exp2(m - m_use);
    const float p = fast_exp2(s - m_use);
    l = l * alpha + wave_sum(p);
    m = m_new;
#pragma unroll
    for (int t = 0; t < kMaxDim / 64; ++t) o[t] *= alpha;
    const float w = key < end ? p * vscale : 0.f;
    const int keys = static_cast<int>(min(int64_t(64), end - k0));
    for (int u = 0; u < keys; ++u) {
      const float pu = lane_read(w, u);
      const uint8_t* vr = V + (k0 + u) * a.vst[2];
#pragma unroll
      for (int t = 0; t < kMaxDim / 64; ++t)
        if (t * 64 + lane < a.D) o[t] = fmaf(pu, __builtin_amdgcn_cvt_f32_fp8(vr[t * 64 + lane], 0), o[t]);
    }
  }
  // (a NaN sum, from a NaN score, passes through)
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* O = static_cast<T*>(a.o) + b * a.ost[0] + h * a.ost[1] + i * a.ost[2];
#pragma unroll
  for (int t = 0; t < kMaxDim / 64; ++t)
    if (t * 64 + lane < a.D) O[t * 64 + lane] = static_cast<T>(o[t] * inv);
}

template <typename T>
int run_rows(const CacheAttnArgs& a, hipStream_t st) {
  note_kernel("kv_cache_attention rows");
  hipLaunchKernelGGL((k_cache_attn_rows<T>), blocks_2d(static_cast<int64_t>(a.B) * a.Hq * a.Sq), dim3(64), 0, st, a);
  return check_launch("kv_cache_attention");
}

}  // namespace
}  // namespace ntops

using namespace ntops;

extern "C" int64_t ntops_kv_cache_attention_workspace(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq,
                                                      int64_t C, int64_t D) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Sq <= 0 || C <= 0 || D <= 0 || Hq % Hkv != 0 || dtype == NTOPS_F32) return 0;
  if (B > kMaxCount || Hq > kMaxCount || Sq > kMaxCount || C > (int64_t(1) << 40) || B * Hq > kMaxCount ||
      B * Hq * Sq > kMaxCount)
    return 0;  // (the call is refused)
  return Sq * (Hq / Hkv) <= kDecodeRows ? cache_decode_workspace(B, Hq, Hkv, Sq, C, D) : cache_tile_workspace(dtype, B, Hq, Hkv, Sq, C, D);
}

extern "C" int ntops_kv_cache_attention(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t C, int64_t D,
                                        int64_t block, const void* q, const int64_t* q_strides, const void* key_cache,
                                        const int64_t* key_cache_strides, const void* value_cache,
                                        const int64_t* value_cache_strides, const float* key_scale,
                                        const int64_t* key_scale_strides, const float* value_scale,
                                        const int64_t* value_scale_strides, const void* lengths, int lengths_dtype,
                                        int causal, double scale, void* out, const int64_t* out_strides, void* workspace,
                                        int64_t workspace_bytes, void* stream) {
  if (B < 0 || Hq < 0 || Hkv < 0 || Sq < 0 || C < 0 || D < 0)
    return set_error(NTOPS_ERR_INVALID, "kv_cache_attention: negative size");
  if (dtype != NTOPS_F32 && dtype != NTOPS_F16 && dtype != NTOPS_BF16)
    return set_error(NTOPS_ERR_UNSUPPORTED, "kv_cache_attention: unsupported dtype %d (F32/F16/BF16 only)", dtype);
  if (!block_ok(block))
    return set_error(NTOPS_ERR_INVALID, "kv_cache_attention: a block is a power of two of 16 to 2^24 tokens");
  if (lengths && !index_dtype(lengths_dtype))
    return set_error(NTOPS_ERR_INVALID, "kv_cache_attention: lengths are I32 or I64");
  if (causal != 0 && causal != 1) return set_error(NTOPS_ERR_INVALID, "kv_cache_attention: causal is 0 or 1");
  if (B == 0 || Hq == 0 || Sq == 0 || D == 0) return NTOPS_OK;
  if (Hkv == 0 || Hq % Hkv != 0)
    return set_error(NTOPS_ERR_INVALID, "kv_cache_attention: query heads are not a multiple of cache heads");
  if (!q || !out || !q_strides || !out_strides)
    return set_error(NTOPS_ERR_INVALID, "kv_cache_attention: null pointer");
  if (C > 0 && (!key_cache || !value_cache || !key_scale || !value_scale || !key_cache_strides || !value_cache_strides ||
                !key_scale_strides || !value_scale_strides))
    return set_error(NTOPS_ERR_INVALID, "kv_cache_attention: null pointer");
  if (D > kMaxDim) return set_error(NTOPS_ERR_UNSUPPORTED, "kv_cache_attention: head dim over %d", kMaxDim);
  if (B > kMaxCount || Hq > kMaxCount || Sq > kMaxCount || C > (int64_t(1) << 40) || B * Hq > kMaxCount || B * Hq * Sq > kMaxCount)
    return set_error(NTOPS_ERR_UNSUPPORTED, "kv_cache_attention: problem too large");
  CacheAttnArgs a{};
  a.q = q;
  a.k = static_cast<const uint8_t*>(key_cache);
  a.v = static_cast<const uint8_t*>(value_cache);
  a.ks = key_scale;
  a.vs = value_scale;
  a.o = out;
  if (D > 1 && (q_strides[3] != 1 || out_strides[3] != 1))
    return set_error(NTOPS_ERR_INVALID, "kv_cache_attention: the head dims need unit strides");
  for (int d = 0; d < 3; ++d) {
    a.qst[d] = q_strides[d];
    a.ost[d] = out_strides[d];
  }
  if (C > 0) {
    if ((D > 1 && (key_cache_strides[3] != 1 || value_cache_strides[3] != 1)) ||
        (C > block && (key_scale_strides[2] != 1 || value_scale_strides[2] != 1)))
      return set_error(NTOPS_ERR_INVALID, "kv_cache_attention: the last dims need unit strides");
    for (int d = 0; d < 3; ++d) {
      a.kst[d] = key_cache_strides[d];
      a.vst[d] = value_cache_strides[d];
    }
    for (int d = 0; d < 2; ++d) {
      a.kss[d] = key_scale_strides[d];
      a.vss[d] = value_scale_strides[d];
    }
  }
  a.lengths = lengths;
  a.lengths_dtype = lengths_dtype;
  a.C = C;
  a.B = static_cast<int>(B);
  a.Hq = static_cast<int>(Hq);
  a.Hkv = static_cast<int>(Hkv);
  a.Sq = static_cast<int>(Sq);
  a.D = static_cast<int>(D);
  a.shift = __builtin_ctzll(static_cast<unsigned long long>(block));
  a.causal = causal;
  a.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (workspace_bytes < 0 || (workspace != nullptr && !aligned16(workspace)))
    return set_error(NTOPS_ERR_INVALID, "kv_cache_attention: workspace not aligned to 16 bytes");
  if (cache_decode_serves(a, dtype)) return cache_decode(dtype, a, workspace, workspace_bytes, st);
  if (cache_tile_serves(a, dtype)) return cache_tile(dtype, a, workspace, workspace_bytes, st);
  return dispatch_float16_32(dtype, "kv_cache_attention", [&](auto tag) { return run_rows<decltype(tag)>(a, st); });
}
