// fp32 windowed and shared-prefix attention on the matrix cores: IEEE fp32 products
// (v_mfma_f32_16x16x4_f32) with fp32 sums.  Here for many rows; few ones further down.
//
// A block is 16 rows a wave of those that share a cache head, over the 32-key tiles of
// both spans or a slice of them.  The scores are computed transposed, S^T = K Q^T: lane
// l's accumulator r holds key 4 (l >> 4) + r of a 16-key block for row l & 15, which is
// the B operand of O^T += V^T P^T for MFMA step r when the keys of that step are taken as
// 4 (l >> 4) + r (a sum over keys does not depend on their order), so P never leaves the
// registers, and every accumulator of a lane belongs to one row.  The head dim is walked
// as d = 16 t + 4 g + e (g = l >> 4, e the step of four), so a lane reads four floats of K
// per four MFMAs; of V, whose rows stay as they are, the four columns side by side that
// four accumulators take, in an order in which the results lie side by side, too.  (With
// V transposed on its way into the LDS, whose stores then collide, long rows took 8 to 15 %
// more.)  Tiles are double-buffered; a tile's loads go to registers before the previous
// tile's products and are stored after them, one barrier a tile.  Two blocks a CU (over 128
// columns, whose tiles fill the LDS: one), 4 waves a SIMD.
//
// Bound by the fp32 matrix rate, a tenth of the 16-bit one here (154 against 1513
// TFLOP/s).  Measured: (1, 16 / 4, 4096 causal) of 128 638 us, 108 TFLOP/s -- nearly twice as
// long with blocks of one set after the other, which leave the longest two of a CU to end
// alone; (3, 12 / 4, 333 over up to 1501, window 500 and 8 sinks) of 96 47 us, the matrix
// cores half busy: 21 us of products, those of masked keys in edge tiles among them, the
// starts and ends of blocks of four tiles, and 8 us the merge of five slices; blocks of 64
// rows gained nothing.  Over 128 columns (1, 16 / 4, 500 behind 500) of 256 102 us, by the
// kernel of one wave per row 1151; (16, 16 / 4, 1 over 4100) of 256 216 against 319.
//
// What a row does not see: as in attn_spans_tile.h.
#include <algorithm>
#include <atomic>

#include "attn_spans.h"

namespace ntops {
namespace {

constexpr int kKeys = 32;
constexpr uint32_t kCus = 256;
constexpr int kFewWaves = 4;

template <int DP>
constexpr int kLdsBytes = 2 * kKeys * (DP + 4 + DP) * 4;

template <int DP, int NW>
__global__ __launch_bounds__(64 * NW, DP > 128 ? 2 : 4) void k_span_f32(SpanArgs a, int mode, int nqb, int slices, uint32_t total, SpanPart part) {
  constexpr int QB = 16 * NW;
  constexpr int KP = DP + 4;     // floats per K row in the LDS
  constexpr int VP = DP;         // per V row (those 4 apart, read side by side, start at the same bank)
  constexpr int kKTile = kKeys * KP, kBuf = kKTile + kKeys * VP;
  constexpr int NC = DP / 16;    // columns of V of a lane
  constexpr int kThreads = 64 * NW;
  constexpr int kF4 = kKeys * DP / 4;                   // 16-byte chunks per operand and tile
  constexpr int kLd = (kF4 + kThreads - 1) / kThreads;  // per thread
  extern __shared__ __attribute__((aligned(16))) float sm[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int64_t all = block_id();
  if (all >= total) return;  // the tail of a 2-D grid (the whole block)
  const uint32_t pid = static_cast<uint32_t>(all);
  // Long rows of keys first; up to two blocks a CU, which all start at once, the CUs with
  // the longest of the first half get the shortest of the second.
  const uint32_t sets = total / static_cast<uint32_t>(nqb * slices);
  const uint32_t order = total <= 2 * kCus && pid >= kCus ? total - 1 - (pid - kCus) : pid, in = order / sets, set = order - in * sets;
  const uint32_t back = in / static_cast<uint32_t>(slices);
  const int qb = nqb - 1 - static_cast<int>(back), slice = static_cast<int>(in - back * slices);
  const int group = a.group, ro = group * a.Sq;
  const bool front_only = mode == kFront;
  const auto token = [&](int row) { return static_cast<int>(static_cast<uint32_t>(row) / static_cast<uint32_t>(group)); };
  const int nrows = front_only ? ro * a.per : ro;
  const int r0 = qb * QB, r1 = min(r0 + QB, nrows);
  const Spans s = make_spans<4>(a, mode, set, front_only ? 0 : token(r0), front_only ? 0 : token(r1 - 1));

  const int qw = r0 + wave * 16;
  const bool active = qw < nrows;
  const bool in_rows = qw + r16 < nrows;
  const SpanRow x = span_row(a, mode, s, min(qw + r16, nrows - 1));
  const int tw0 = front_only ? 0 : token(min(qw, nrows - 1)), tw1 = front_only ? 0 : token(min(qw + 15, nrows - 1));
  f32x4 qf[DP / 16];
  {
    const float* Q = static_cast<const float*>(a.q) + x.b * a.qst[0] + x.h * a.qst[1] + x.t * a.qst[2];
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) {
      const int d = 16 * t + 4 * g;
      qf[t] = in_rows && d < a.D ? *reinterpret_cast<const f32x4*>(Q + d) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // the front's keys and the main ones behind them, as one sequence
  const int nf = s.n[0], keys = nf + s.n[1];
  const int sinks = nf + max(0, s.sinks);
  const int w_hi = nf + s.hi(tw1), w_lo = nf + s.lo(tw0), w_hi_all = nf + s.hi(tw0), w_lo_all = nf + s.lo(tw1);
  const int my_hi = nf + s.hi(x.t) - 4 * g, my_lo = nf + s.lo(x.t) - 4 * g;
  const int nt = (keys + kKeys - 1) / kKeys;
  const int share = (nt + slices - 1) / slices;
  const int i0 = min(slice * share, nt);
  const int nkv = min(i0 + share, nt) - i0;

  f32x4 kst[kLd], vst[kLd];
  const auto load_tile = [&](int t) __attribute__((always_inline)) {
    const int k0 = (i0 + t) * kKeys;
#pragma unroll
    for (int j = 0; j < kLd; ++j) {
      const int f = threadIdx.x + kThreads * j;
      const int key = k0 + f / (DP / 4), d = 4 * (f % (DP / 4));
      f32x4 kz = {0.f, 0.f, 0.f, 0.f}, vz = {0.f, 0.f, 0.f, 0.f};
      if (f < kF4 && key < keys && d < a.D) {
        const int sp = key < nf ? 0 : 1;
        const int64_t row = key < nf ? key : key - nf;
        kz = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(s.k[sp]) + row * s.kld[sp] + d);
        vz = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(s.v[sp]) + row * s.vld[sp] + d);
      }
      kst[j] = kz;
      vst[j] = vz;
    }
  };
  const auto store_tile = [&](int buf) __attribute__((always_inline)) {
    float* kt = sm + buf * kBuf;
    float* vt = kt + kKTile;
#pragma unroll
    for (int j = 0; j < kLd; ++j) {
      const int f = threadIdx.x + kThreads * j;
      if (f >= kF4) break;
      const int kl = f / (DP / 4), d = 4 * (f % (DP / 4));
      *reinterpret_cast<f32x4*>(kt + kl * KP + d) = kst[j];
      *reinterpret_cast<f32x4*>(vt + kl * VP + d) = vst[j];
    }
  };

  // Columns of V that lane r16 multiplies, in fours of 64 and in twos of the last 32 of 96:
  // what a lane gets of O then lies side by side in fours, and so do those of g = 0 .. 3.
  const int at4 = (r16 >> 2) + 4 * (r16 & 3), at2 = 2 * (r16 >> 2) + (r16 & 1) + 8 * (r16 >> 1 & 1);
  f32x4 o[DP / 16];
#pragma unroll
  for (int i = 0; i < DP / 16; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = neg_inf(), l = 0.f;
  if (nkv > 0) {
    load_tile(0);
    store_tile(0);
  }
  __syncthreads();
  for (int t = 0; t < nkv; ++t) {
    if (t + 1 < nkv) load_tile(t + 1);
    const float* kt = sm + (t & 1) * kBuf;
    const float* vt = kt + kKTile;
    const int k0 = (i0 + t) * kKeys;
    if (active && k0 < w_hi && (k0 + kKeys > w_lo || k0 < sinks)) {  // wave-uniform
      f32x4 sc[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) sc[kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int tt = 0; tt < DP / 16; ++tt) {
        f32x4 kf[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) kf[kb] = *reinterpret_cast<const f32x4*>(kt + (kb * 16 + r16) * KP + 16 * tt + 4 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) sc[kb] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[kb][e], qf[tt][e], sc[kb], 0, 0, 0);
      }
      const bool whole = k0 + kKeys <= w_hi_all && (k0 >= w_lo_all || k0 + kKeys <= sinks);
      const int up = my_hi - k0, sink = sinks - 4 * g - k0;
      const uint32_t hidden = static_cast<uint32_t>(max(0, my_lo - k0 - sink));  // [sinks, my_lo)
      float mx = neg_inf();
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int k = kb * 16 + r;
          float v = product(sc[kb][r], a.scale_log2);
          if (!whole) v = k < up && static_cast<uint32_t>(k - sink) >= hidden ? v : neg_inf();
          sc[kb][r] = v;
          mx = fmaxf(mx, v);
        }
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float m_new = fmaxf(m, mx);
      const float m_use = m_new == neg_inf() ? 0.f : m_new;  // nothing seen so far: P = 0
      const float alpha = fast_exp2(m - m_use);
      float ps = 0.f;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = fast_exp2(sc[kb][r] - m_use);
          sc[kb][r] = p;
          ps += p;
        }
      l = l * alpha + ps;  // (this lane's part of the row's sum)
      m = m_new;
#pragma unroll
      for (int u = 0; u < DP / 16; ++u) o[u] *= alpha;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float* row = vt + (kb * 16 + 4 * g + e) * VP;
          float v[NC];
#pragma unroll
          for (int u = 0; u + 4 <= NC; u += 4) {
            const f32x4 y = *reinterpret_cast<const f32x4*>(row + 16 * u + 4 * at4);
#pragma unroll
            for (int c = 0; c < 4; ++c) v[u + c] = y[c];
          }
          if constexpr (NC % 4 == 2) {
            const f32x2 y = *reinterpret_cast<const f32x2*>(row + 64 + 2 * at2);
            v[4] = y.x;
            v[5] = y.y;
          }
#pragma unroll
          for (int u = 0; u < NC; ++u) o[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[u], sc[kb][e], o[u], 0, 0, 0);
        }
    }
    if (t + 1 < nkv) store_tile((t + 1) & 1);  // read last in tile t - 1, before the barrier that ended it
    __syncthreads();
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  const bool none = m == neg_inf();
  const float inv = l == 0.f ? 0.f : 1.f / l;  // (a NaN sum passes through)
  // runs of four columns: `first(i)` and the accumulators
  const auto first = [&](int i) { return i < NC / 4 * 4 ? i / 4 * 64 + i % 4 * 16 + 4 * g : 64 + 16 * (i - 4) + 4 * g; };
  const auto run = [&](int i) {
    if (i < NC / 4 * 4) {
      const int u = i / 4 * 4, r = i % 4;
      return f32x4{o[u][r], o[u + 1][r], o[u + 2][r], o[u + 3][r]};
    }
    const int r = 2 * (i - 4);
    return f32x4{o[NC - 2][r], o[NC - 1][r], o[NC - 2][r + 1], o[NC - 1][r + 1]};
  };
  float any = 0.f;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const f32x4 y = run(i);
    any += first(i) < a.D ? (y[0] + y[1]) + (y[2] + y[3]) : 0.f;
  }
  if (in_rows) {
    const int64_t at = part.p ? part.at(a, x, slice) : 0;
    if (part.p && g == 0) {
      float* ml = part.ml(a, at);
      ml[0] = m;
      ml[1] = l;
    }
    float* O = part.p ? part.row(at) : static_cast<float*>(a.o) + x.b * a.ost[0] + x.h * a.ost[1] + x.t * a.ost[2];
    const float f = part.p ? 1.f : inv;
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (first(i) < a.D) *reinterpret_cast<f32x4*>(O + first(i)) = (none ? f32x4{0.f, 0.f, 0.f, 0.f} : run(i)) * f;
  }
  const uint64_t bad = __ballot(in_rows && !none && span_again(any, l));
  uint32_t rows = static_cast<uint32_t>(bad | bad >> 16 | bad >> 32 | bad >> 48) & 0xffffu;
  if (rows != 0) wait_vmcnt<0>();  // what has been written of these rows is written before what follows
  while (rows != 0) {
    const int r = qw + __builtin_ctz(rows);
    rows &= rows - 1;
    const SpanRow y = span_row(a, mode, s, r);
    const int k0 = i0 * kKeys, k1 = min(k0 + nkv * kKeys, keys);
    span_row_again<float, DP / 16>(a, s, part, y, slice, min(k0, nf), min(k1, nf), max(0, k0 - nf), max(0, k1 - nf));
  }
}

// Up to 16 rows of a set, head dims up to DP: each wave streams tiles of 16 keys of its own,
// global -> registers, one tile ahead, without the LDS: lane (g, r16) reads of K what the
// first product takes, key r16's columns 16 t + 4 g .. + 3, and of V columns 64 w + 4 r16 ..
// + 3 of the keys 4 g + e, the operand of O^T rows 4 r16 + c (an order of O's columns
// that the result undoes).  The waves are joined through the LDS at the end.
//
// Bound by the loads: (32, 32 / 8, 1 over 4096) of 128 164 us, 6.5 TB/s, where blocks of 128
// rows, of whose eight waves one has rows, took 311; (8, 32 / 8, 1 over 4096) 49 against 89,
// (1, 32 / 8, 1 over 1024) 12.0 against 17.8, a row alone at its head (32, 8, 1 over 4096) 164,
// by the kernel of one wave per row 199.
template <int DP>
__global__ __launch_bounds__(64 * kFewWaves, 2) void k_span_f32_few(SpanArgs a, int mode, int slices, uint32_t total, SpanPart part) {
  constexpr int NW = kFewWaves, KT = DP / 16, VW = DP / 64, LD = DP + 4;
  __shared__ __attribute__((aligned(16))) float so[NW * 16 * LD];
  __shared__ float sm[2 * NW * 16];
  __shared__ uint32_t again;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int64_t all = block_id();
  if (all >= total) return;  // the tail of a 2-D grid (the whole block)
  const uint32_t pid = static_cast<uint32_t>(all);
  const uint32_t set = pid / static_cast<uint32_t>(slices);
  const int slice = static_cast<int>(pid - set * slices);
  const bool front_only = mode == kFront;
  const int rows = a.group * a.Sq * (front_only ? a.per : 1), t1 = front_only ? 0 : a.Sq - 1;
  const Spans s = make_spans<4>(a, mode, set, 0, t1);
  const bool in_rows = r16 < rows;
  const SpanRow x = span_row(a, mode, s, min(r16, rows - 1));

  f32x4 qf[KT];
  {
    const float* Q = static_cast<const float*>(a.q) + x.b * a.qst[0] + x.h * a.qst[1] + x.t * a.qst[2];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      const int d = 16 * t + 4 * g;
      qf[t] = in_rows && d < a.D ? *reinterpret_cast<const f32x4*>(Q + d) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // the front's keys and the main ones behind them, as one sequence
  const int nf = s.n[0], keys = nf + s.n[1];
  const int sinks = nf + max(0, s.sinks);
  const int hi_all = nf + s.hi(0), lo_all = nf + s.lo(t1);
  const int my_hi = nf + s.hi(x.t) - 4 * g, my_lo = nf + s.lo(x.t) - 4 * g;
  const int nt = (keys + 15) / 16, share = (nt + slices - 1) / slices;
  const int i0 = min(slice * share, nt), i1 = min(i0 + share, nt);

  // (past the last key: that key again, and past the last column the first ones, whose
  // scores are masked, whose queries are 0 and which are not stored)
  const auto row_of = [&](int key, int which) __attribute__((always_inline)) {
    const int k = min(key, keys - 1), sp = k < nf ? 0 : 1;
    const int64_t row = sp ? k - nf : k;
    return which ? reinterpret_cast<const float*>(s.v[sp]) + row * s.vld[sp] : reinterpret_cast<const float*>(s.k[sp]) + row * s.kld[sp];
  };
  struct Tile {
    f32x4 k[KT], v[4][VW];
  };
  const auto load = [&](int i, Tile& t) __attribute__((always_inline)) {
    const float* K = row_of(16 * i + r16, 0);
#pragma unroll
    for (int u = 0; u < KT; ++u) {
      const int d = 16 * u + 4 * g;
      t.k[u] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(K + (d < a.D ? d : 0)));
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float* V = row_of(16 * i + 4 * g + e, 1);
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        const int d = 64 * w + 4 * r16;
        t.v[e][w] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(V + (d < a.D ? d : 0)));
      }
    }
  };

  f32x4 o[VW][4];
#pragma unroll
  for (int w = 0; w < VW; ++w)
#pragma unroll
    for (int c = 0; c < 4; ++c) o[w][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = neg_inf(), l = 0.f;  // of row r16; this lane's part of its sum
  const auto attend = [&](int i, Tile& t) __attribute__((always_inline)) {
    if (a.D < DP) {
#pragma unroll
      for (int u = 0; u < KT; ++u)
        if (16 * u + 4 * g >= a.D) t.k[u] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    f32x4 sc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int u = 0; u < KT; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[e & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(t.k[u][e], qf[u][e], sc[e & 1], 0, 0, 0);
    const int k0 = 16 * i;
    const bool whole = k0 + 16 <= hi_all && (k0 >= lo_all || k0 + 16 <= sinks);
    const int up = my_hi - k0, sink = sinks - 4 * g - k0;
    const uint32_t hidden = static_cast<uint32_t>(max(0, my_lo - k0 - sink));  // [sinks, my_lo)
    float p[4], mx = neg_inf();
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      p[r] = product(sc[0][r] + sc[1][r], a.scale_log2);
      if (!whole) p[r] = r < up && static_cast<uint32_t>(r - sink) >= hidden ? p[r] : neg_inf();
      mx = fmaxf(mx, p[r]);
    }
    if (__any(mx > m)) {
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float m_new = fmaxf(m, mx);
      const float alpha = m_new == neg_inf() ? 1.f : fast_exp2(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int w = 0; w < VW; ++w)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[w][c] *= alpha;
    }
    const float m_use = m == neg_inf() ? 0.f : m;  // nothing seen so far: P = 0
#pragma unroll
    for (int r = 0; r < 4; ++r) p[r] = fast_exp2(p[r] - m_use);
    l += (p[0] + p[1]) + (p[2] + p[3]);
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int w = 0; w < VW; ++w)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[w][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(t.v[e][w][c], p[e], o[w][c], 0, 0, 0);
  };
  Tile ta, tb;
  int i = i0 + wave;
  if (i < i1) load(i, ta);
  for (; i < i1; i += 2 * NW) {
    if (i + NW < i1) load(i + NW, tb);
    attend(i, ta);
    if (i + NW >= i1) break;
    if (i + 2 * NW < i1) load(i + 2 * NW, ta);
    attend(i + NW, tb);
  }

  // join the waves
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (threadIdx.x == 0) again = 0;
  if (g == 0) {
    sm[wave * 16 + r16] = m;
    sm[(NW + wave) * 16 + r16] = l;
  }
#pragma unroll
  for (int w = 0; w < VW; ++w)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *reinterpret_cast<f32x4*>(so + (wave * 16 + r16) * LD + 64 * w + 16 * g + 4 * r) = f32x4{o[w][0][r], o[w][1][r], o[w][2][r], o[w][3][r]};
  __syncthreads();
  for (int it = threadIdx.x; it < 16 * (DP / 4); it += 64 * NW) {
    const int row = it / (DP / 4), d = (it - row * (DP / 4)) * 4;
    if (row >= rows || d >= a.D) continue;
    float mm = sm[row];
#pragma unroll
    for (int w = 1; w < NW; ++w) mm = fmaxf(mm, sm[w * 16 + row]);
    float sum = 0.f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float mw = sm[w * 16 + row];
      // (a wave of which the row has seen nothing but NaN scores: its sum alone)
      const float fw = mw == neg_inf() ? 0.f : fast_exp2(mw - mm);
      sum += sm[(NW + w) * 16 + row] * fw;
      const f32x4 ow = *reinterpret_cast<const f32x4*>(so + (w * 16 + row) * LD + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += mw == neg_inf() ? 0.f : ow[e] * fw;
    }
    const float any = (v[0] + v[1]) + (v[2] + v[3]);
    if (span_again(any, sum)) atomicOr(&again, 1u << row);
    const SpanRow y = span_row(a, mode, s, row);
    if (part.p) {
      const int64_t at = part.at(a, y, slice);
      if (d == 0) {
        float* ml = part.ml(a, at);
        ml[0] = mm;
        ml[1] = sum;
      }
      *reinterpret_cast<f32x4*>(part.row(at) + d) = v;
    } else {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;  // (a NaN sum passes through)
      *reinterpret_cast<f32x4*>(static_cast<float*>(a.o) + y.b * a.ost[0] + y.h * a.ost[1] + y.t * a.ost[2] + d) = v * inv;
    }
  }
  __syncthreads();
  uint32_t bad = __builtin_amdgcn_readfirstlane(again);
  if (bad == 0) return;  // (the same for every wave)
  wait_vmcnt<0>();       // what has been written of these rows is written before what follows
  __syncthreads();
  while (bad != 0) {
    const int row = __builtin_ctz(bad);
    bad &= bad - 1;
    if (row % NW != wave) continue;
    const SpanRow y = span_row(a, mode, s, row);
    span_row_again<float, KT>(a, s, part, y, slice, min(16 * i0, nf), min(16 * i1, nf), max(0, 16 * i0 - nf), max(0, min(16 * i1, keys) - nf));
  }
}

template <int DP>
int launch_f32_few(const SpanArgs& a, int mode, int slices, const SpanPart& part, hipStream_t st) {
  const int64_t total = span_sets(a, mode) * slices;
  note_kernel("%s f32 few d%d mode%d split%d", a.pk ? "shared_prefix" : "sliding_window", DP, mode, slices);
  hipLaunchKernelGGL((k_span_f32_few<DP>), blocks_2d(total), dim3(64 * kFewWaves), 0, st, a, mode, slices, static_cast<uint32_t>(total), part);
  return check_launch("attention");
}

template <int DP, int NW>
int launch_f32(const SpanArgs& a, int mode, int slices, const SpanPart& part, hipStream_t st) {
  auto kern = k_span_f32<DP, NW>;
  if constexpr (kLdsBytes<DP> > 65536) {
    static std::atomic<uint64_t> done{0};
    if (int e = reserve_lds(reinterpret_cast<const void*>(kern), kLdsBytes<DP>, done, "attention")) return e;
  }
  const int64_t nqb = ceil_div(span_rows(a, mode), 16 * NW);
  const int64_t total = span_sets(a, mode) * nqb * slices;
  note_kernel("%s f32 d%d waves%d mode%d split%d", a.pk ? "shared_prefix" : "sliding_window", DP, NW, mode, slices);
  hipLaunchKernelGGL(kern, blocks_2d(total), dim3(64 * NW), kLdsBytes<DP>, st, a, mode, static_cast<int>(nqb), slices, static_cast<uint32_t>(total), part);
  return check_launch("attention");
}

// Over 128 columns all 256 are multiplied: (1, 16 / 4, 4096 causal) of 136 / 192 / 256 1578 /
// 1584 / 1592 us, (1, 16 / 4, 500 behind 500) 90 / 95 / 102.  A form of 192 is not built.
template <int DP>
int run_f32(const SpanArgs& a, int mode, int slices, const SpanPart& part, hipStream_t st) {
  return launch_f32<DP, 8>(a, mode, slices, part, st);
}

}  // namespace

int span_f32_run(const SpanArgs& a, int mode, int slices, const SpanPart& part, hipStream_t st) {
  if (a.D <= 128 && span_rows(a, mode) <= kF32FewRows)
    return a.D <= 64 ? launch_f32_few<64>(a, mode, slices, part, st) : launch_f32_few<128>(a, mode, slices, part, st);
  if (a.D <= 64) return run_f32<64>(a, mode, slices, part, st);
  if (a.D <= 96) return run_f32<96>(a, mode, slices, part, st);
  if (a.D <= 128) return run_f32<128>(a, mode, slices, part, st);
  return run_f32<256>(a, mode, slices, part, st);
}

}  // namespace ntops
