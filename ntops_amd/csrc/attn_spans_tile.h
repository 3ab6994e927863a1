// Many query rows a cache head (prompts, chunks of prompts, all sequences of a shared
// prefix together): windowed and shared-prefix attention on the matrix cores.
//
// A block is 128 of the rows that share a cache head -- with grouped queries 128 / group
// tokens, so that the keys that a window leaves to a block are little more than the
// window -- over the 64-key tiles of both spans, or a slice of them.  Wave w owns rows
// 32 w .. + 31 with their queries in registers and skips the tiles that none of them
// sees; tiles go global -> LDS by direct DMA into one of two stages while the other is
// used, one barrier a tile.  Two blocks a CU (up to 96 columns: three; over 128, whose
// stages fill the LDS: one) that nothing synchronizes: the maxima and exponentials of one
// run under the MFMAs of the other.  (Rows of 96 columns in the LDS of 128, two blocks: 57
// against 49 us for narrow windows, 840 against 777 for long rows.)
//
// Blocks see few keys at a prompt's start and many at its end, so the order in which they
// are handed out decides where two a CU start at once: (1, 16 / 4, 4096 causal) of 128 97 us,
// set after set 119.
//
// Eight waves of 32 rows that alternate the two kinds of phase between barriers (256
// rows, four stages, one block a CU) took 2 % less for long rows of 128 columns -- (16,
// 32 / 8, 500 over a shared 8192) bf16 1070 against 1088 us -- 28 % more of 64 columns,
// (1, 32 / 8, 16384, window 4096) 748 against 583, and half as long again for narrow
// windows, (7, 16, 2001, window 255) of 80 columns 100 against 57.
//
// A row's reference (from which its exponents are taken) follows its maximum when that
// is past it by more than 2^8.  Masked scores are -inf whatever their key holds; a
// value that is not finite times P = 0 is NaN, so a row whose result is NaN, or past fp32's
// range, under a sum that is a number is computed again by itself, from the keys that it
// sees.
//
// Bound by the vector instructions of the softmax beside the matrix cores (55 % busy over
// long rows of 128 columns), at few tiles a block by its start and end, and of one row a
// head over 128 columns by the loads.  Measured, bf16: (1, 32 / 8, 16384 tokens, window
// 4096 and 4 sinks) of 128 931 us, 1.03 PFLOP/s; (16, 32 / 8, 500 over a shared 8192) of 128
// 1042 us, 1.05 PFLOP/s; (7, 16, 2001, window 255) of 80 46 us; (1, 16 / 4, 1000 behind 1000)
// of 192 42 us, of 256 50 us; (64, 32 / 8, 1 over 4100) of 256 381 us, 5.6 TB/s, by the
// kernel of one wave per row 8.4 ms.
#pragma once

#include "attn_spans.h"

namespace ntops {
namespace span_tile {

constexpr int kWaves = 4;
constexpr int kRowsBlock = 32 * kWaves;
static_assert(kRowsBlock == kTileRows, "the plans count on it");
constexpr int kKeys = 64;
constexpr uint32_t kCus = 256;
constexpr int kAhead = 4;  // fragments read ahead of the MFMA that uses them
constexpr float kSlack = 8.f;

// DMA of one tile of 64 keys of D: 1 KiB an instruction, spread evenly over the waves.
template <int D, bool IS_V>
struct SpanDma {
  static constexpr int kChunks = D / 8;  // of a row
  static constexpr int kInst = kKeys * kChunks / 64 / kWaves;
  static_assert(kInst * kWaves * 64 == kKeys * kChunks, "tile must split evenly over the waves");
  uint32_t voff[kInst];
  int lds_off;

  __device__ __forceinline__ void init(int64_t ld, int wave, int lane, int dt) {
    lds_off = wave * kInst * 1024;
#pragma unroll
    for (int i = 0; i < kInst; ++i) {
      const int id = (wave * kInst + i) * 64 + lane, row = id / kChunks, slot = id % kChunks;
      const int c = IS_V ? vslot<D>(row, slot) : kslot<D>(row, slot);
      voff[i] = c * 8 < dt ? static_cast<uint32_t>(row * ld * 2 + c * 16) : kOOB;
    }
  }
  // `n` rows at `base` (those past them are zeros) into the LDS
  __device__ __forceinline__ void issue(const char* base, int64_t ld, int n, int dt, uint32_t tile) const {
    const u32x4 r = make_rsrc(base, ((n - 1) * ld + dt) * 2);
#pragma unroll
    for (int i = 0; i < kInst; ++i) dma16(r, __builtin_amdgcn_readfirstlane(tile + lds_off + i * 1024), voff[i]);
  }
};

// A tile whose rows below `cut` come from `front` and the others from `base` (the row
// that would be the tile's first), `n` rows in all; once a block, so in few instructions.
template <int D, bool IS_V>
__device__ __forceinline__ void dma_two(const char* front, int64_t front_ld, const char* base, int64_t ld, int cut, int n, int dt, uint32_t tile,
                                        int wave, int lane) {
  constexpr int kInst = SpanDma<D, IS_V>::kInst, kChunks = SpanDma<D, IS_V>::kChunks;
#pragma unroll 1
  for (int i = 0; i < kInst; ++i) {
    const int inst = wave * kInst + i, row = (inst * 64 + lane) / kChunks, slot = (inst * 64 + lane) % kChunks;
    const int c = IS_V ? vslot<D>(row, slot) : kslot<D>(row, slot);
#pragma unroll 1
    for (int part = 0; part < 2; ++part) {
      const int64_t of = part ? ld : front_ld;
      const u32x4 r = make_rsrc(part ? base : front, ((part ? n : cut) - 1) * of * 2 + dt * 2);
      const uint32_t off = c * 8 < dt ? static_cast<uint32_t>(row * of * 2 + c * 16) : kOOB;
      if ((row < cut) == (part == 0)) dma16(r, __builtin_amdgcn_readfirstlane(tile + inst * 1024), off);  // (a lane that is off writes nothing)
    }
  }
}

__device__ __forceinline__ float max32(const f32x16 (&s)[2]) {
  float v[32];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int e = 0; e < 16; ++e) v[16 * u + e] = s[u][e];
  float m[11];
  const uint32_t seen = read_of(v[15], v[31]);
  m[10] = max3_after(v[15], v[31], v[31], seen);
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    m[i] = max3_after(v[3 * i], v[3 * i + 1], v[3 * i + 2], seen);
    m[5 + i] = max3_after(v[16 + 3 * i], v[17 + 3 * i], v[18 + 3 * i], seen);
  }
  return max3(max3(max3(m[0], m[1], m[2]), max3(m[3], m[4], m[5]), m[6]), max3(m[7], m[8], m[9]), m[10]);
}

template <int D>
constexpr int kTileLds = 2 * 2 * kKeys * D * 2;

// Block `pid` of `total`: D columns of a row in the LDS, DM that are multiplied, at least
// the head dim.
template <typename T, int D, int DM>
__device__ __forceinline__ void tile_block(const SpanArgs& a, int mode, int nqb, int slices, uint32_t total, const SpanPart& part, uint32_t pid,
                                           char* smem) {
  constexpr int KS = DM / 16;  // k-steps of S = Q K^T
  constexpr int DT = DM / 32;  // 32-column tiles of O
  constexpr int kTile = kKeys * D * 2;
  constexpr int kStage = 2 * kTile;                      // K tile, then V tile
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Long rows of keys first.  An XCD (workgroups go round them) walks whole sets, every
  // eighth one; up to two blocks a CU, which all start at once, the CUs with the longest
  // of the first half get the shortest of the second.
  const uint32_t per = static_cast<uint32_t>(nqb * slices), sets = total / per;
  uint32_t set, in;
  if (total > 2 * kCus && (sets & 7) == 0) {
    const uint32_t at = pid >> 3, of = at / per;
    set = of * 8 + (pid & 7);
    in = at - of * per;
  } else {
    const uint32_t at = total <= 2 * kCus && pid >= kCus ? total - 1 - (pid - kCus) : pid;
    in = at / sets;
    set = at - in * sets;
  }
  const uint32_t back = in / static_cast<uint32_t>(slices);
  const int qb = nqb - 1 - static_cast<int>(back), slice = static_cast<int>(in - back * slices);
  const int group = a.group, ro = group * a.Sq;
  const int nrows = mode == kFront ? ro * a.per : ro;
  const int r0 = qb * kRowsBlock, r1 = min(r0 + kRowsBlock, nrows);
  const bool front_only = mode == kFront;
  const auto token = [&](int row) { return static_cast<int>(static_cast<uint32_t>(row) / static_cast<uint32_t>(group)); };
  const Spans s = make_spans<2>(a, mode, set, front_only ? 0 : token(r0), front_only ? 0 : token(r1 - 1));

  const int qw = r0 + wave * 32;
  const bool active = qw < nrows;
  const int my_r = qw + (lane & 31);
  const bool in_rows = my_r < nrows;
  const SpanRow x = span_row(a, mode, s, min(my_r, nrows - 1));
  const int tw0 = front_only ? 0 : token(min(qw, nrows - 1)), tw1 = front_only ? 0 : token(min(qw + 31, nrows - 1));
  // The front's keys and the main ones behind them, as one sequence: of it [lo, hi) and
  // all below `sinks` are seen by some row of the wave, between lo_all and hi_all by every row
  const int nf = s.n[0], keys = nf + s.n[1];
  const int sinks = nf + max(0, s.sinks);
  const int w_hi = nf + s.hi(tw1), w_lo = nf + s.lo(tw0), w_hi_all = nf + s.hi(tw0), w_lo_all = nf + s.lo(tw1);

  u32x4 qf[KS];  // Q fragments (A operand of S): row my_r, d = 16 ks + 8 (lane >> 5) .. + 7
  {
    const T* Q = static_cast<const T*>(a.q) + x.b * a.qst[0] + x.h * a.qst[1] + x.t * a.qst[2];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d0 = ks * 16 + 8 * (lane >> 5);
      qf[ks] = in_rows && d0 < a.D ? *reinterpret_cast<const u32x4*>(Q + d0) : u32x4{0, 0, 0, 0};
      if (a.scale_log2 < 0.f) qf[ks] ^= 0x80008000u;
    }
  }
  // (under a zero scale the least factor there is, so that a masked score stays -inf)
  const float c = a.scale_log2 == 0.f ? 0x1p-149f : fabsf(a.scale_log2);

  const int nt = (keys + kKeys - 1) / kKeys;
  const int share = (nt + slices - 1) / slices;
  const int i0 = min(slice * share, nt);
  const int nkv = min(i0 + share, nt) - i0;  // tiles of this item

  SpanDma<D, false> kd[2];  // of the front, of the main span
  SpanDma<D, true> vd[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    kd[i].init(s.kld[i], wave, lane, a.D);
    vd[i].init(s.vld[i], wave, lane, a.D);
  }
  const uint32_t smem_addr = lds_addr(smem);
  // tile g of the item into its stage
  const auto dma = [&](int g) __attribute__((always_inline)) {
    const uint32_t st = smem_addr + static_cast<uint32_t>((g & 1) * kStage);
    const int k0 = (i0 + g) * kKeys;
    if (k0 >= nf) {
      const int row0 = k0 - nf;
      kd[1].issue(s.k[1] + row0 * s.kld[1] * 2, s.kld[1], s.n[1] - row0, a.D, st);
      vd[1].issue(s.v[1] + row0 * s.vld[1] * 2, s.vld[1], s.n[1] - row0, a.D, st + kTile);
    } else if (k0 + kKeys <= nf || s.n[1] == 0) {
      kd[0].issue(s.k[0] + k0 * s.kld[0] * 2, s.kld[0], nf - k0, a.D, st);
      vd[0].issue(s.v[0] + k0 * s.vld[0] * 2, s.vld[0], nf - k0, a.D, st + kTile);
    } else {  // the front's last keys and the first main ones
      const int cut = nf - k0;
      dma_two<D, false>(s.k[0] + k0 * s.kld[0] * 2, s.kld[0], s.k[1] - cut * s.kld[1] * 2, s.kld[1], cut, keys - k0, a.D, st, wave, lane);
      dma_two<D, true>(s.v[0] + k0 * s.vld[0] * 2, s.vld[0], s.v[1] - cut * s.vld[1] * 2, s.vld[1], cut, keys - k0, a.D, st + kTile, wave, lane);
    }
  };
  if (nkv > 0) dma(0);
  // the queries settle here, with tile 0
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) asm volatile("" ::"v"(qf[ks]));
  // whether the wave has rows that see keys of tile g
  const auto need = [&](int g) __attribute__((always_inline)) {
    const int k0 = (i0 + g) * kKeys;
    return active && k0 < w_hi && (k0 + kKeys > w_lo || k0 < sinks);
  };
  // limits of row my_r relative to this lane's column group: element (u, e) of a tile is
  // its key 32 u + 8 (e >> 2) + (e & 3) past that origin
  const int my_hi = nf + s.hi(x.t) - 4 * (lane >> 5), my_lo = nf + s.lo(x.t) - 4 * (lane >> 5);

  f32x16 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[t][e] = 0.f;
  float m_run = neg_inf();  // reference (base 2) of row my_r
  float l_half = 0.f;       // this lane's half of the row's sum of exponentials
  uint32_t far = 0;         // span_far of some row's reference, wave-uniform
  f32x16 sc[2];             // S of the tile being softmaxed
  u32x4 pf[4];              // P of that tile, as MFMA A operands per 16-key slice

  // O += P_j V_j; fragment i + kAhead is read while MFMA i runs, and a scheduling fence
  // per step pins that order
  const auto pv_part = [&](int j) __attribute__((always_inline)) {
    const char* sv = smem + (j & 1) * kStage + kTile;
    constexpr int nm = 4 * DT;  // MFMA i: key slice i / DT, d tile i % DT
    u32x4 f[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) f[i] = v_frag<D>(sv, (i % DT) * 32, i / DT, lane);
#pragma unroll
    for (int i = 0; i < nm; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      o[i % DT] = mfma32<T>(f[i % kAhead], pf[i / DT], o[i % DT]);
      if (i + kAhead < nm) f[i % kAhead] = v_frag<D>(sv, ((i + kAhead) % DT) * 32, (i + kAhead) / DT, lane);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // S = Q K_j^T
  const auto qk_part = [&](int j) __attribute__((always_inline)) {
    const char* sk = smem + (j & 1) * kStage;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[u][e] = 0.f;
    constexpr int nm = 2 * KS;  // MFMA i: d slice i / 2, key half i % 2
    u32x4 f[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) f[i] = k_frag<D>(sk, (i % 2) * 32, i / 2, lane);
#pragma unroll
    for (int i = 0; i < nm; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      sc[i % 2] = mfma32<T>(f[i % kAhead], qf[i / 2], sc[i % 2]);
      if (i + kAhead < nm) f[i % kAhead] = k_frag<D>(sk, ((i + kAhead) % 2) * 32, (i + kAhead) / 2, lane);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  const auto vector_phase = [&](int g) __attribute__((always_inline)) {
    const int k0 = (i0 + g) * kKeys;
    if (k0 + kKeys > w_hi_all) {
      const int up = my_hi - k0;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[u][e] = 32 * u + 8 * (e >> 2) + (e & 3) < up ? sc[u][e] : neg_inf();
    }
    if (k0 < w_lo_all && k0 + kKeys > sinks) {  // hidden: [sinks, my_lo)
      const int sink = sinks - 4 * (lane >> 5) - k0;
      const uint32_t hidden = static_cast<uint32_t>(max(0, my_lo - k0 - sink));
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          sc[u][e] = static_cast<uint32_t>(32 * u + 8 * (e >> 2) + (e & 3) - sink) < hidden ? neg_inf() : sc[u][e];
    }
    const float th = max32(sc) * c;  // of this lane's half of the row (base 2)
    if (__any(th > m_run + kSlack)) {
      const float tmax = fmaxf(th, __shfl_xor(th, 32, 64));
      const bool up = tmax > m_run + kSlack;
      const float alpha = up ? fast_exp2(m_run - tmax) : 1.f;
      m_run = up ? tmax : m_run;
      l_half *= alpha;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[t][e] *= alpha;
      far |= __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(__ballot(span_far(m_run)) != 0));
    }
    float mb = m_run == neg_inf() ? 0.f : m_run;  // nothing seen so far: P = 0
    float by = c;
    if (far != 0) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[u][e] = product(sc[u][e], c) - mb;
      by = 1.f;
      mb = 0.f;
    }
    float p[2][16];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) p[u][e] = fast_exp2(fmaf(sc[u][e], by, -mb));
    float r[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) r[e] = p[0][e] + p[1][e];
#pragma unroll
    for (int w = 8; w >= 1; w >>= 1)
#pragma unroll
      for (int e = 0; e < w; ++e) r[e] += r[e + w];
    l_half += r[0];
    // The second product takes probabilities of the type, half a step each, as the framework's
    // other attention does; their sum, and all that is summed with them, keeps 32 bits.  In
    // parts of higher and lower bits it would be two products, of which this kernel is full.
    // Against 64 bits, of the whole result: bf16 0.0020 to 0.0023, of which 0.0017 are the
    // result's own rounding; f16 0.00026 to 0.00029 of which 0.00021.
#pragma unroll
    for (int sl = 0; sl < 4; ++sl) pf[sl] = pack8<T>(&p[sl >> 1][8 * (sl & 1)]);
  };

  for (int k = 0; k < nkv; ++k) {
    wait_vmcnt<0>();
    block_barrier();  // tile k is in, and every wave is done with tile k - 1
    if (k + 1 < nkv) dma(k + 1);
    if (!need(k)) continue;
    // (the other block's wave on this SIMD has its vector work under these MFMAs)
    __builtin_amdgcn_s_setprio(1);
    qk_part(k);
    __builtin_amdgcn_s_setprio(0);
    vector_phase(k);
    __builtin_amdgcn_s_setprio(1);
    pv_part(k);
    __builtin_amdgcn_s_setprio(0);
  }

  const float l = l_half + __shfl_xor(l_half, 32, 64);
  const float inv = l == 0.f ? 0.f : 1.f / l;  // (a NaN sum passes through)
  // what a row met of values without seeing a key of theirs: nothing
  const bool none = m_run == neg_inf();
  float any = 0.f;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      o[t][e] = none ? 0.f : o[t][e];
      any += o[t][e];
    }
  if (in_rows) {
    if (part.p) {
      const int64_t at = part.at(a, x, slice);
      if (lane < 32) {
        float* ml = part.ml(a, at);
        ml[0] = m_run;
        ml[1] = l;
      }
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int col = t * 32 + 8 * q + 4 * (lane >> 5);
          if (col < a.D)
            *reinterpret_cast<f32x4*>(part.row(at) + col) = f32x4{o[t][4 * q], o[t][4 * q + 1], o[t][4 * q + 2], o[t][4 * q + 3]};
        }
    } else {
      T* O = static_cast<T*>(a.o) + x.b * a.ost[0] + x.h * a.ost[1] + x.t * a.ost[2];
      float by_sum = inv;
      if constexpr (std::is_same<T, _Float16>::value) {
        // as mean_as, in fewer instructions: the row is divided by what its probabilities were rounded up by
        // (f16 (7, 16, 2001, window 255) of 80 columns 47.1 us, each value cut by itself 47.9, neither 46.2)
        float top = 0.f;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
          for (int e = 0; e < 16; e += 2) top = max3(fabsf(o[t][e]), fabsf(o[t][e + 1]), top);
        const float past = top * inv;
        if (past > 65504.f && past < __builtin_huge_valf()) by_sum *= 65504.f / past;
      }
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          T v4[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v4[e] = static_cast<T>(o[t][4 * q + e] * by_sum);
          const int col = t * 32 + 8 * q + 4 * (lane >> 5);
          if (col < a.D)  // a.D % 8 == 0: the 4 columns are all in or all out
            *reinterpret_cast<u32x2*>(O + col) = __builtin_bit_cast(u32x2, v4);
        }
    }
  }
  wait_vmcnt<0>();  // no DMA may land after the workgroup ends
  const uint64_t bad = __ballot(in_rows && span_again(any, l));
  uint32_t rows = static_cast<uint32_t>(bad) | static_cast<uint32_t>(bad >> 32);
  while (rows != 0) {
    const int r = qw + __builtin_ctz(rows);
    rows &= rows - 1;
    const SpanRow y = span_row(a, mode, s, r);
    const int k0 = i0 * kKeys, k1 = min(k0 + nkv * kKeys, keys);
    span_row_again<T, DM / 16>(a, s, part, y, slice, min(k0, nf), min(k1, nf), max(0, k0 - nf), max(0, k1 - nf));
  }
}

}  // namespace span_tile
}  // namespace ntops
