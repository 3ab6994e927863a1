// Many query rows over an 8-bit cache (prompts, chunks of prompts).
//
// Rows are those of all query heads that share a cache head, in the order
// (position, head): row r is position r / group of head r % group, so a tile of
// 128 rows sees one cache head up to nearly the same key, and the tile's keys
// are widened once for all of them.  Four waves of 32 rows; key tiles of 64.
//
//  * A tile's e4m3 keys and values come through registers (16-byte loads a tile
//    ahead) and go to the LDS widened to 16 bits, in the layouts that the
//    fragment reads of attention.h expect: each byte is converted once per block
//    where converting fragments would do it in each of the four waves.
//  * Values are widened to bf16 times the power of two in their block's scale
//    (exact), whatever the query's type; what is left of a scale that is no
//    power of two, in [1, 2), multiplies the probabilities, in a branch that
//    stores made by this library never take.  The probabilities are rounded to
//    bf16 for the product (f16 queries: with the rest as a second operand): only
//    bf16 holds values under scales of any size.
//  * The scale of a key's block times the softmax scale is a factor per 16 keys:
//    the maximum is taken over raw scores in each 16 and scaled then, and the
//    exponent is one fma per score.
//  * A NaN value reaches the rows that see it and no others, though P = 0 times it
//    is NaN: a tile that not every row of the block sees whole is searched for NaNs
//    before its products; they are noted for the rows that see them, whose results
//    become NaN at the end, and cleared.  Without the search (4, 32 / 8, 2048 over
//    2048, 128) causal bf16 took 163 us instead of 164, of 64 values 101 instead of
//    105.
//  * Few tiles over many keys are split over slices of the keys, fp32 partial
//    results combined in slice order (k_cache_merge).
#include <algorithm>
#include <atomic>

#include "attn_cache.h"

namespace ntops {
namespace {

constexpr int kRows = 128;
constexpr int kKeys = 64;
constexpr int kAhead = 4;  // fragments read ahead of the MFMA that uses them
// A row's reference, which its exponents are taken from, follows its maximum when
// that is past it by more than this (base 2): the largest probability is then at
// most 2^8, in fp32 sums and in bf16 products as good as 1, and O is rescaled on
// few tiles instead of most.
constexpr float kSlack = 8.f;

// Two e4m3 values of a word to 16-bit ones; bf16: times the power of two in scale.
template <typename T, bool HI>
__device__ __forceinline__ uint32_t widen2(uint32_t w, float scale) {
  if constexpr (std::is_same<T, __bf16>::value)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI));
}

// The 16 values of a 16-byte chunk, as two 16-byte chunks.
template <typename T>
__device__ __forceinline__ void widen16(u32x4 c, float scale, u32x4 (&o)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    o[i] = u32x4{widen2<T, false>(c[2 * i], scale), widen2<T, true>(c[2 * i], scale),
                 widen2<T, false>(c[2 * i + 1], scale), widen2<T, true>(c[2 * i + 1], scale)};
}

__device__ __forceinline__ float max8(const float* v) {
  return max3(max3(v[0], v[1], v[2]), max3(v[3], v[4], v[5]), max3(v[6], v[7], v[7]));
}

// Blocks that a CU holds: by registers.
constexpr int blocks_per_cu(bool bf16, int d) { return bf16 && d <= 64 ? 3 : 2; }

// part: fp32 partial results (null: one slice, O normalised into a.o).
template <typename T, int D>
__global__ __launch_bounds__(256, blocks_per_cu(std::is_same<T, __bf16>::value, D)) void k_cache_tile(CacheAttnArgs a, int nqb, int total, int nsplit, float* part) {
  constexpr int KS = D / 16;          // k-steps of S = Q K^T
  constexpr int DT = D / 32;          // 32-column tiles of O
  constexpr bool LO = std::is_same<T, _Float16>::value;  // probabilities in two operands
  constexpr int kTile = kKeys * D * 2;  // bytes of a widened tile
  constexpr int CPR = D / 16;         // 16-byte chunks of a cache row
  constexpr int NL = kKeys * CPR / 256;  // chunks a thread loads of a tile's keys (and values)
  __shared__ __attribute__((aligned(1024))) char smem[2 * 2 * kTile];  // [stage][keys, values]
  __shared__ uint8_t nans[kKeys][D / 8];     // a bit per value of a tile that is NaN
  __shared__ uint8_t nan_rows[kRows][D / 8];  // and per result that one has reached
  __shared__ int nan_waves[4];               // whether a wave has found any
  bool nan_seen = false;                     // (nan_rows is in use)

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int64_t pid = block_id();
  if (pid >= total) return;  // the tail of a 2-D grid (the whole block)
  // An XCD (workgroups go round them) walks whole cache heads, every eighth one, so
  // that sequences of different lengths spread over the XCDs; the tiles with the
  // most keys first.
  const int per = nqb * nsplit;
  int bh, in;
  if (((a.B * a.Hkv) & 7) == 0) {
    const int at = static_cast<int>(pid >> 3);
    bh = at / per * 8 + static_cast<int>(pid & 7);
    in = at % per;
  } else {
    bh = static_cast<int>(pid / per);
    in = static_cast<int>(pid - static_cast<int64_t>(bh) * per);
  }
  const int qb = nqb - 1 - in / nsplit, sp = in % nsplit;
  const int b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int group = a.Hq / a.Hkv;
  const int nrows = group * a.Sq;
  const int64_t n_all = length_of(a, b);
  // keys that the tile's last row sees
  const int r_last = min(qb * kRows + kRows, nrows) - 1;
  const int64_t seen = a.causal ? max(int64_t(0), n_all - a.Sq + r_last / group + 1) : n_all;
  const int64_t chunk = (seen + nsplit * kKeys - 1) / (nsplit * kKeys) * kKeys;
  const int64_t t0 = sp * chunk;
  const int n = __builtin_amdgcn_readfirstlane(static_cast<int>(max(int64_t(0), min(seen - t0, chunk))));
  const int nt = (n + kKeys - 1) / kKeys;

  const int my_r = qb * kRows + wave * 32 + (lane & 31);
  const bool in_rows = my_r < nrows;
  const int my_q = my_r / group, my_h = hk * group + my_r - my_q * group;
  // last key of the slice that this lane's row sees
  const int my_lim = a.causal ? static_cast<int>(max(int64_t(-1), min(int64_t(n), n_all - a.Sq + my_q + 1 - t0))) - 1 : n - 1;
  const int w_first = min(qb * kRows + wave * 32, nrows - 1) / group;  // the wave's first position
  const int w_lim = a.causal ? static_cast<int>(max(int64_t(-1), min(int64_t(n), n_all - a.Sq + w_first + 1 - t0))) - 1 : n - 1;

  // last key that the block's first row sees: a tile past it is cut for some rows
  const int b_lim = a.causal ? static_cast<int>(max(int64_t(-1), min(int64_t(n), n_all - a.Sq + qb * kRows / group + 1 - t0))) - 1 : n - 1;

  // Q fragments (A operand of S); a negative softmax scale: -Q under its magnitude
  u32x4 qf[KS];
  const T* Q = static_cast<const T*>(a.q) + b * a.qst[0] + my_h * a.qst[1] + my_q * a.qst[2];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int d0 = ks * 16 + 8 * (lane >> 5);
    qf[ks] = in_rows && d0 < a.D ? *reinterpret_cast<const u32x4*>(Q + d0) : u32x4{0, 0, 0, 0};
    if (a.scale_log2 < 0.f) qf[ks] ^= 0x80008000u;
  }
  const float c0 = fabsf(a.scale_log2);

  // this thread's chunks of a tile: chunk id threadIdx.x + 256 i, row id / CPR
  const __amdgpu_buffer_rsrc_t rk = buffer_rsrc_uniform(
      a.k + b * a.kst[0] + hk * a.kst[1] + t0 * a.kst[2], n > 0 ? static_cast<uint32_t>((n - 1) * a.kst[2] + a.D) : 0u);
  const __amdgpu_buffer_rsrc_t rv = buffer_rsrc_uniform(
      a.v + b * a.vst[0] + hk * a.vst[1] + t0 * a.vst[2], n > 0 ? static_cast<uint32_t>((n - 1) * a.vst[2] + a.D) : 0u);
  const int64_t blk0 = t0 >> a.shift;
  const int first_part = static_cast<int>(t0 - (blk0 << a.shift));
  const uint32_t sbytes = n > 0 ? static_cast<uint32_t>(((first_part + n - 1) >> a.shift) * 4 + 4) : 0u;
  const __amdgpu_buffer_rsrc_t rks = buffer_rsrc_uniform(a.ks + b * a.kss[0] + hk * a.kss[1] + blk0, sbytes);
  const __amdgpu_buffer_rsrc_t rvs = buffer_rsrc_uniform(a.vs + b * a.vss[0] + hk * a.vss[1] + blk0, sbytes);
  uint32_t koff[NL], voff[NL];
  int lrow[NL], lchunk[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int id = threadIdx.x + 256 * i;
    lrow[i] = id / CPR;
    lchunk[i] = id % CPR;
    const bool ok = lchunk[i] * 16 < a.D;
    koff[i] = ok ? static_cast<uint32_t>(lrow[i] * a.kst[2] + lchunk[i] * 16) : kOOB;
    voff[i] = ok ? static_cast<uint32_t>(lrow[i] * a.vst[2] + lchunk[i] * 16) : kOOB;
  }
  // two tiles on their way: tile j's chunks in set j & 1
  u32x4 kc[2][NL], vc[2][NL];
  float kscale[2], vscale[2];  // of the tile's 16-key part lane & 3
  const auto load = [&](auto set, int j) __attribute__((always_inline)) {
    constexpr int S = decltype(set)::value;
    const uint32_t kt = static_cast<uint32_t>(j) * static_cast<uint32_t>(kKeys * a.kst[2]);
    const uint32_t vt = static_cast<uint32_t>(j) * static_cast<uint32_t>(kKeys * a.vst[2]);
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      kc[S][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, koff[i] == kOOB ? kOOB : koff[i] + kt, 0, 0));
      vc[S][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rv, voff[i] == kOOB ? kOOB : voff[i] + vt, 0, 0));
    }
    const int at = ((first_part + j * kKeys + (lane & 3) * 16) >> a.shift) * 4;
    kscale[S] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rks, at, 0, 0));
    vscale[S] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rvs, at, 0, 0));
  };
  const auto put = [&](auto set) __attribute__((always_inline)) {  // into the stage of the same number
    constexpr int S = decltype(set)::value;
    char* sk = smem + S * 2 * kTile;
    char* sv = sk + kTile;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      u32x4 w[2];
      widen16<T>(kc[S][i], 1.f, w);
#pragma unroll
      for (int u = 0; u < 2; ++u)
        *reinterpret_cast<u32x4*>(sk + lrow[i] * (D * 2) + kslot<D>(lrow[i], lchunk[i] * 2 + u) * 16) = w[u];
      // (a wave's value rows of one i lie in one part: its first lane's)
      widen16<__bf16>(vc[S][i], lane_read(vscale[S], (i * (256 / CPR) + wave * (64 / CPR)) >> 4), w);
#pragma unroll
      for (int u = 0; u < 2; ++u)
        *reinterpret_cast<u32x4*>(sv + lrow[i] * (D * 2) + vslot<D>(lrow[i], lchunk[i] * 2 + u) * 16) = w[u];
    }
  };

  f32x16 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[t][e] = 0.f;
  float m_i = neg_inf(), l_i = 0.f;  // reference (base 2) of row my_r; this lane's half of its sum
  float c[4], f[4];  // of the current tile's parts: the scores' factor, the rest of the values' scale
  const auto factors = [&](auto set) __attribute__((always_inline)) {
    constexpr int S = decltype(set)::value;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      // at least the least factor there is, so that a masked score (-inf) stays one under a zero scale
      const float x = lane_read(kscale[S], p) * c0, y = lane_read(vscale[S], p);
      c[p] = x < 0x1p-149f ? 0x1p-149f : x;
      f[p] = y < 0x1p-126f ? 0.f : __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, y) & 0x7fffffu) | 0x3f800000u);
    }
  };
  constexpr std::integral_constant<int, 0> even{};
  constexpr std::integral_constant<int, 1> odd{};
  if (nt > 0) {
    load(even, 0);
    load(odd, 1);
    put(even);
    factors(even);
  }
  __syncthreads();

  // Notes and clears the NaNs of tile j's values (bf16, at sv).
  const auto clear_nans = [&](char* sv, int j) __attribute__((always_inline)) {
    constexpr int kChunks = D / 8;  // 16-byte chunks of a row
    int tid = threadIdx.x;  // (opaque, so that nothing of this sits in registers in other tiles)
    asm volatile("" : "+v"(tid));
    const auto chunk = [&](int id) { return reinterpret_cast<u32x4*>(sv + id / kChunks * (D * 2) + vslot<D>(id / kChunks, id % kChunks) * 16); };
    const auto bad = [](uint32_t w) { return (((w & 0x7fff7fffu) + 0x007f007fu) >> 15) & 0x00010001u; };  // in bits 0 and 16
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < kKeys * kChunks / 256; ++i) {
      const u32x4 w = *chunk(tid + i * 256);
      any |= bad(w.x) | bad(w.y) | bad(w.z) | bad(w.w);
    }
    any = __any(any != 0);
    if ((tid & 63) == 0) nan_waves[tid >> 6] = static_cast<int>(any);
    __syncthreads();
    if ((nan_waves[0] | nan_waves[1] | nan_waves[2] | nan_waves[3]) == 0) return;
#pragma unroll 1
    for (int id = tid; id < kKeys * kChunks; id += 256) {
      u32x4 w = *chunk(id);
      uint32_t bits = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t b = bad(w[e]);
        w[e] &= ~(b * 0xffffu);
        bits |= ((b | b >> 15) & 3u) << (2 * e);
      }
      *chunk(id) = w;
      nans[id / kChunks][id % kChunks] = static_cast<uint8_t>(bits);
    }
    __syncthreads();
    const int row = (tid >> 6) * 32 + (tid & 31), last = min(my_lim - j * kKeys, kKeys - 1);
#pragma unroll 1
    for (int c = tid >> 5 & 1; c < kChunks; c += 2) {
      uint32_t bits = nan_seen ? nan_rows[row][c] : 0;
      for (int k = 0; k <= last; ++k) bits |= nans[k][c];
      nan_rows[row][c] = static_cast<uint8_t>(bits);
    }
    nan_seen = true;
  };

  // tile j, of stage set; other: the other one (loads past the last tile bring zeros)
  const auto tile = [&](auto set, auto other, int j) __attribute__((always_inline)) {
    const char* sk = smem + decltype(set)::value * 2 * kTile;
    const char* sv = sk + kTile;
    if (b_lim < n - 1 && j * kKeys + kKeys - 1 > b_lim) clear_nans(const_cast<char*>(sv), j);
    load(set, j + 2);
    f32x16 s[2];
    // (the other block's wave on this SIMD has its vector work under these MFMAs)
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[t][e] = 0.f;
    {
      constexpr int nm = 2 * KS;  // MFMA i: d slice i / 2, key half i % 2
      u32x4 fr[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) fr[i] = k_frag<D>(sk, (i % 2) * 32, i / 2, lane);
#pragma unroll
      for (int i = 0; i < nm; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        s[i % 2] = mfma32<T>(fr[i % kAhead], qf[i / 2], s[i % 2]);
        if (i + kAhead < nm) fr[i % kAhead] = k_frag<D>(sk, ((i + kAhead) % 2) * 32, (i + kAhead) / 2, lane);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    // element 4q + e of half t is key 64 j + 32 t + 8 q + 4 (lane >> 5) + e
    if (j * kKeys + kKeys - 1 > w_lim) {
      const int rel = my_lim - j * kKeys - 4 * (lane >> 5);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[t][e] = 32 * t + 8 * (e >> 2) + (e & 3) <= rel ? s[t][e] : neg_inf();
    }
    float x[2][16];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) x[t][e] = s[t][e];
    const float th = fmaxf(max3(max8(&x[0][0]) * c[0], max8(&x[0][8]) * c[1], max8(&x[1][0]) * c[2]), max8(&x[1][8]) * c[3]);
    if (__any(th > m_i + kSlack)) {
      const auto h2 = __builtin_amdgcn_permlane32_swap(__float_as_uint(th), __float_as_uint(th), false, false);
      const float tmax = fmaxf(__uint_as_float(h2[0]), __uint_as_float(h2[1]));  // of lanes l and l ^ 32
      const bool up = tmax > m_i + kSlack;
      const float alpha = up ? fast_exp2(m_i - tmax) : 1.f;
      m_i = up ? tmax : m_i;
      l_i *= alpha;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[t][e] *= alpha;
    }
    const float mb = m_i == neg_inf() ? 0.f : m_i;  // nothing seen so far: P = 0
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) x[t][e] = fast_exp2(fmaf(s[t][e], c[2 * t + (e >> 3)], -mb));
    {
      float r[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) r[e] = x[0][e] + x[1][e];
#pragma unroll
      for (int w = 8; w >= 1; w >>= 1)
#pragma unroll
        for (int e = 0; e < w; ++e) r[e] += r[e + w];
      l_i += r[0];
    }
    {
      u32x4 pf[4], pl[4];
      if (f[0] == 1.f && f[1] == 1.f && f[2] == 1.f && f[3] == 1.f) {
#pragma unroll
        for (int sl = 0; sl < 4; ++sl) pack_p<LO>(&x[sl >> 1][8 * (sl & 1)], pf[sl], pl[sl]);
      } else {
#pragma unroll
        for (int sl = 0; sl < 4; ++sl) {
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = x[sl >> 1][8 * (sl & 1) + e] * f[sl];
          pack_p<LO>(y, pf[sl], pl[sl]);
        }
      }
      __builtin_amdgcn_s_setprio(1);
      constexpr int kAheadV = LO ? 2 : kAhead;  // (two MFMAs a fragment)
      constexpr int nm = 4 * DT;  // MFMA i: key slice i / DT, d tile i % DT
      u32x4 fr[kAheadV];
#pragma unroll
      for (int i = 0; i < kAheadV; ++i) fr[i] = v_frag<D>(sv, (i % DT) * 32, i / DT, lane);
#pragma unroll
      for (int i = 0; i < nm; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        o[i % DT] = mfma32<__bf16>(fr[i % kAheadV], pf[i / DT], o[i % DT]);
        if constexpr (LO) o[i % DT] = mfma32<__bf16>(fr[i % kAheadV], pl[i / DT], o[i % DT]);
        if (i + kAheadV < nm) fr[i % kAheadV] = v_frag<D>(sv, ((i + kAheadV) % DT) * 32, (i + kAheadV) / DT, lane);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    // the other stage was last read before the barrier that ended the previous tile
    if (j + 1 < nt) {
      put(other);
      factors(other);
    }
    __syncthreads();
  };
  for (int j = 0; j < nt; j += 2) {
    tile(even, odd, j);
    if (j + 1 < nt) tile(odd, even, j + 1);
  }

  l_i += __shfl_xor(l_i, 32, 64);
  if (!in_rows) return;
  // A row that sees none of these keys is 0 whatever it met of the values: one past
  // fp32's range, which 256 times a scale of 2^120 is, times P = 0 is NaN.  (A row
  // whose scores are all NaN has a NaN sum.)
  const bool none = m_i == neg_inf();
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[t][e] = none ? 0.f : o[t][e];
  if (nan_seen)
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t bits = nan_rows[wave * 32 + (lane & 31)][4 * t + q] >> 4 * (lane >> 5);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][4 * q + e] = bits >> e & 1 ? __builtin_nanf("") : o[t][4 * q + e];
      }
  if (part) {
    const int64_t nrow = static_cast<int64_t>(a.B) * a.Hq * a.Sq;
    const int64_t at = ((static_cast<int64_t>(b) * a.Hq + my_h) * a.Sq + my_q) * nsplit + sp;
    float* ml = part + nrow * nsplit * a.D;
    if (lane < 32) {
      ml[2 * at] = m_i;
      ml[2 * at + 1] = l_i;
    }
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int qq = 0; qq < 4; ++qq) {
        const int col = t * 32 + 8 * qq + 4 * (lane >> 5);
        if (col < a.D)
          *reinterpret_cast<f32x4*>(part + at * a.D + col) =
              f32x4{o[t][4 * qq], o[t][4 * qq + 1], o[t][4 * qq + 2], o[t][4 * qq + 3]};
      }
    return;
  }
  const float inv = l_i == 0.f ? 0.f : 1.f / l_i;  // (a NaN sum passes through)
  T* O = static_cast<T*>(a.o) + b * a.ost[0] + my_h * a.ost[1] + my_q * a.ost[2];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int qq = 0; qq < 4; ++qq) {
      T v4[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v4[e] = static_cast<T>(o[t][4 * qq + e] * inv);
      const int col = t * 32 + 8 * qq + 4 * (lane >> 5);
      if (col < a.D)  // a.D % 16 == 0: the 4 columns are all in or all out
        *reinterpret_cast<u32x2*>(O + col) = __builtin_bit_cast(u32x2, v4);
    }
}

// Slices of the keys: as many as fill the CUs (half as many: (3, 24 / 8, 101 over
// 5001, 64) f16 34.7 -> 41.9 us, twice as many 36.7), none under four key tiles at
// full length.
int tile_split(int dtype, int64_t heads, int64_t rows, int64_t C, int64_t D) {
  const int64_t tiles = heads * ceil_div(rows, kRows);
  const int64_t n = std::min({static_cast<int64_t>(64), blocks_per_cu(dtype == NTOPS_BF16, static_cast<int>(D)) * cu_count_cached() / tiles, ceil_div(C, 4 * kKeys)});
  return static_cast<int>(std::max<int64_t>(n, 1));
}

template <typename T, int D>
int launch_tile(const CacheAttnArgs& a, int nsplit, float* part, hipStream_t st) {
  const int64_t rows = static_cast<int64_t>(a.Hq / a.Hkv) * a.Sq;
  const int64_t nqb = ceil_div(rows, kRows);
  const int64_t total = nqb * nsplit * a.B * a.Hkv;
  note_kernel("kv_cache_tile d%d split%d", D, nsplit);
  hipLaunchKernelGGL((k_cache_tile<T, D>), blocks_2d(total), dim3(256), 0, st, a, static_cast<int>(nqb),
                     static_cast<int>(total), nsplit, part);
  if (part) cache_merge(std::is_same<T, __bf16>::value ? NTOPS_BF16 : NTOPS_F16, a, nsplit, part, st);
  return check_launch("kv_cache_attention");
}

template <typename T>
int run_tile(const CacheAttnArgs& a, void* ws, int64_t ws_bytes, hipStream_t st) {
  constexpr int dt = std::is_same<T, __bf16>::value ? NTOPS_BF16 : NTOPS_F16;
  int nsplit = tile_split(dt, static_cast<int64_t>(a.B) * a.Hkv, static_cast<int64_t>(a.Hq / a.Hkv) * a.Sq, a.C, a.D);
  const int64_t need = cache_tile_workspace(dt, a.B, a.Hq, a.Hkv, a.Sq, a.C, a.D);
  if (need == 0 || ws == nullptr || ws_bytes < need) {
    nsplit = 1;
    ws = nullptr;
  }
  float* part = static_cast<float*>(ws);
  return a.D > 64 ? launch_tile<T, 128>(a, nsplit, part, st) : launch_tile<T, 64>(a, nsplit, part, st);
}

}  // namespace

bool cache_tile_serves(const CacheAttnArgs& a, int dtype) {
  const int64_t rows = static_cast<int64_t>(a.Hq / a.Hkv) * a.Sq;
  return cache_matrix_layout(a, dtype) && rows < (int64_t(1) << 30) &&
         ceil_div(rows, kRows) * a.B * a.Hkv <= 0x7fffffffLL / 64;
}

int64_t cache_tile_workspace(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t C, int64_t D) {
  if (D % 16 != 0 || D > 128 || C == 0) return 0;
  const int nsplit = tile_split(dtype, B * Hkv, Hq / Hkv * Sq, C, D);
  return nsplit > 1 ? B * Hq * Sq * nsplit * (D + 2) * 4 : 0;
}

int cache_tile(int dtype, const CacheAttnArgs& a, void* workspace, int64_t workspace_bytes, hipStream_t st) {
  return dtype == NTOPS_BF16 ? run_tile<__bf16>(a, workspace, workspace_bytes, st)
                             : run_tile<_Float16>(a, workspace, workspace_bytes, st);
}

}  // namespace ntops
