// Few query rows a cache head (single tokens, drafted ones): windowed and
// shared-prefix attention bound by streaming keys and values once.
//
// The rows that share a cache head fill the 16 columns of v_mfma_f32_16x16x32, up to
// four such groups of them, so that a key that has reached the LDS serves up to 64
// rows (S^T = K Q^T: a lane's scores all belong to one row, and P^T feeds
// O^T += V^T P^T from registers).  Every wave owns tiles of 8 KiB of keys and 8 KiB
// of values in its own part of the LDS, loaded by direct DMA two tiles ahead and
// refilled as soon as they are read: no barrier before the waves are joined.  Tiles
// never mix the two spans: those of the front come first.
//
// A launch holds two kinds of blocks, one behind the other: those of the rows of
// all sequences of a group over their shared prefix, and those of each sequence's
// rows over its own keys, so that neither waits for the other's tail.
//
// What a row does not see: masked scores are -inf whatever their key holds.  A
// value that is not finite times P = 0 is NaN, though; a row whose result is NaN under
// a sum that is none is computed again by itself, from the keys that it sees.
#include <algorithm>
#include <atomic>

#include "attn_spans.h"

namespace ntops {
namespace {

// v_mfma_f32_16x16x32: lane l holds row / column l & 15 at k = 8 (l >> 4) .. + 7 of
// A / B, and column l & 15, rows 4 (l >> 4) .. + 3 of the result.
template <typename T>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (std::is_same<T, __bf16>::value)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}

template <int D>
constexpr int kTileKeys = 4096 / D;  // keys of a wave's tile
// A row's reference, which its exponents are taken from, follows its maximum when that
// is past it by more than this (base 2): the largest probability is then at most 2^8,
// in fp32 sums and in 16-bit products as good as 1, and O is rescaled on few tiles.
constexpr float kSlack = 8.f;
constexpr int kAhead = 4;  // fragments of V read ahead of the MFMAs that use them

// The copy of a 16-byte chunk a lane with the non-temporal hint (mfma.h: dma16): each
// byte is read once.
__device__ __forceinline__ void dma16_once(u32x4 rsrc, uint32_t lds_dst, uint32_t voffset) {
  asm volatile("buffer_load_dwordx4 %0, %1, 0 offen nt lds"
               :
               : "v"(voffset), "s"(rsrc), "{m0}"(lds_dst)
               : "memory");
}

// Loads of one tile's K (or V) rows: 8 instructions of 1 KiB, the swizzle on the global
// side.  Instruction i brings rows kRows i and on: lane l's row is lane / cpr past them,
// its chunk that of instruction 0, for K with 4 (i & 3) (D = 64: 4 (i & 1)) flipped.
template <int D, bool IS_V>
struct TileDma {
  static constexpr int kInst = 8;
  static constexpr int kRows = 512 / D;  // rows per instruction
  u32x4 rsrc;
  uint32_t ld2;    // bytes from row to row
  uint32_t row, col;  // bytes of the lane's row and chunk

  __device__ __forceinline__ void init(const void* base, int64_t ld, int n, int lane, int dt) {
    rsrc = make_rsrc(base, n > 0 ? ((n - 1) * ld + dt) * 2 : 0);
    ld2 = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(ld * 2));
    constexpr int cpr = D / 8;
    const int r = lane / cpr, slot = lane % cpr;
    row = r * ld2;
    col = (IS_V ? vslot<D>(r, slot) : kslot<D>(r, slot)) * 16;
  }
  // rows `row0` and on into LDS at `dst`; !valid: loads of nothing, which still count in
  // vmcnt.  Columns past the head dim: of K zeros; of V whatever follows, which reaches
  // nothing but the columns of O past the head dim.
  __device__ __forceinline__ void issue(uint32_t dst, int row0, bool valid, int dt) const {
    u32x4 r = rsrc;
    r.z = valid ? r.z : 0u;
    const uint32_t off = row0 * ld2;
    if (IS_V || dt == D) {
#pragma unroll
      for (int i = 0; i < kInst; ++i)
        dma16_once(r, dst + i * 1024, (IS_V ? col : col ^ flip(i)) + (row + (off + i * kRows * ld2)));
    } else {
#pragma unroll
      for (int i = 0; i < kInst; ++i) {
        const uint32_t c = col ^ flip(i);
        dma16_once(r, dst + i * 1024, c < static_cast<uint32_t>(dt * 2) ? c + (row + (off + i * kRows * ld2)) : kOOB);
      }
    }
  }
  static constexpr uint32_t flip(int i) { return 64 * (i & (D == 128 ? 3 : 1)); }
};

// Reads of LDS filled by DMA must not move across the wait that orders them.
template <int N>
__device__ __forceinline__ void wait_dma() {
  __builtin_amdgcn_sched_barrier(0);
  wait_vmcnt<N>();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// One kind of blocks of a launch.
struct FewBlocks {
  int mode;       // SpanMode
  int row_blocks;  // of a set
  int slices;
  int first;       // slice of the rows that slice 0 is
  uint32_t sets, blocks;
};

// Where the queries lie: up to two groups of rows go to registers, through the LDS of a
// tile that has not been loaded yet; more stay in the LDS behind the waves' tiles, as
// fragments, shared by the block.
template <int D, int RG>
constexpr int kQueryLds = RG > 2 ? RG * (D / 32) * 1024 : 0;

// RG: groups of 16 rows a block has room for.
template <typename T, int D, int NW, int RG>
__device__ __forceinline__ void few_block(const SpanArgs& a, const FewBlocks& f, SpanPart part, uint32_t id, char* smem) {
  constexpr int NK = kTileKeys<D>;
  constexpr int KB = NK / 16;  // 16-key blocks of a tile
  constexpr int KS = D / 32;   // k-steps of S^T = K Q^T
  constexpr int DT = D / 16;   // 16-row tiles of O^T
  constexpr bool kShared = RG > 2;
  static_assert(kShared || RG * KS * 1024 <= 8192, "the queries go through a tile's values");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c16 = lane & 15;
  // Blocks of the same keys and other rows run on one XCD (workgroups go round the 8),
  // whose L2 then brings the keys in once.
  uint32_t at = id;
  int rb = 0;
  if (f.row_blocks > 1) {
    const uint32_t t = id >> 3, of = t / static_cast<uint32_t>(f.row_blocks);
    rb = static_cast<int>(t - of * f.row_blocks);
    at = of * 8 + (id & 7);
  }
  const uint32_t set = at / static_cast<uint32_t>(f.slices);
  const int slice = static_cast<int>(at - set * f.slices);
  if (set >= f.sets) return;  // (the whole block: the last eight)
  const int r0 = rb * (16 * RG);
  const int ro = a.group * a.Sq;
  const int set_rows = f.mode == kFront ? ro * a.per : ro;
  const int rows = min(16 * RG, set_rows - r0);
  int t0 = 0, t1 = 0;
  if (f.mode != kFront) {
    t0 = static_cast<int>(static_cast<uint32_t>(r0) / static_cast<uint32_t>(a.group));
    t1 = static_cast<int>(static_cast<uint32_t>(r0 + rows - 1) / static_cast<uint32_t>(a.group));
  }
  part.first = f.first;

  // The queries are on their way before the lengths are known.
  char* mine = smem + wave * 32768;
  const uint32_t mine_addr = lds_addr(mine);
  char* sq = kShared ? smem + NW * 32768 : mine + 16384 + 8192;  // [rg][ks][lane]
  int token[RG];
  {
    const SpanSet w = span_set(a, f.mode, set);
    const T* Q = static_cast<const T*>(a.q) + w.b0 * a.qst[0] + static_cast<int64_t>(w.hk) * a.group * a.qst[1];
    const u32x4 rq = make_rsrc(Q, 0x7ffffff0);
    const uint32_t sq_addr = lds_addr(sq);
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
      const int r = rg * 16 + c16;
      const SpanRow x = span_row(a, f.mode, w, r0 + min(r, rows - 1));
      token[rg] = x.t;
      const uint32_t off = static_cast<uint32_t>(((x.b - w.b0) * a.qst[0] + (x.h - w.hk * a.group) * a.qst[1] + x.t * a.qst[2]) * 2);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int d0 = ks * 32 + 8 * g;
        if (!kShared || (rg * KS + ks) % NW == wave)
          dma16(rq, __builtin_amdgcn_readfirstlane(sq_addr + (rg * KS + ks) * 1024), r < rows && d0 < a.D ? off + d0 * 2 : kOOB);
      }
    }
  }
  const Spans s = make_spans<2>(a, f.mode, set, t0, t1);
  int hi[RG], lo[RG];
#pragma unroll
  for (int rg = 0; rg < RG; ++rg) {
    hi[rg] = s.hi(token[rg]);
    lo[rg] = s.lo(token[rg]);
  }
  // at least the least factor there is, so that a masked score stays -inf under a zero scale
  const float c = fabsf(a.scale_log2) < 0x1p-126f ? 0x1p-126f : fabsf(a.scale_log2);
  const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;  // a negative scale: -Q
  const int hi_min = s.hi(t0), lo_max = s.lo(t1);  // a main tile between them is seen whole by every row

  const int nft = (s.n[0] + NK - 1) / NK, nt = nft + (s.n[1] + NK - 1) / NK;
  const int per = (nt + f.slices - 1) / f.slices;
  const int i0 = min(slice * per, nt), i1 = min(i0 + per, nt);
  const int n = i1 - i0 > wave ? (i1 - i0 - wave + NW - 1) / NW : 0;  // tiles of this wave: i0 + wave, + NW, ...
  TileDma<D, false> kd;
  TileDma<D, true> vd;
  const auto tile_at = [&](int j) { return i0 + wave + j * NW; };
  // (a wave's tiles of the front come first, so each DMA turns to the main span once)
  int kspan = tile_at(0) < nft ? 0 : 1, vspan = kspan;
  kd.init(s.k[kspan], s.kld[kspan], s.n[kspan], lane, a.D);
  vd.init(s.v[vspan], s.vld[vspan], s.n[vspan], lane, a.D);
  const auto issue_k = [&](int j) __attribute__((always_inline)) {
    const int i = tile_at(j);
    if (j < n && kspan == 0 && i >= nft) {
      kspan = 1;
      kd.init(s.k[1], s.kld[1], s.n[1], lane, a.D);
    }
    kd.issue(mine_addr + (j & 1) * 16384, (i < nft ? i : i - nft) * NK, j < n, a.D);
  };
  const auto issue_v = [&](int j) __attribute__((always_inline)) {
    const int i = tile_at(j);
    if (j < n && vspan == 0 && i >= nft) {
      vspan = 1;
      vd.init(s.v[1], s.vld[1], s.n[1], lane, a.D);
    }
    vd.issue(mine_addr + (j & 1) * 16384 + 8192, (i < nft ? i : i - nft) * NK, j < n, a.D);
  };

  f32x4 o[RG][DT];
  float m[RG], l[RG];  // reference (base 2) of the lane's row; this lane's part of its sum
#pragma unroll
  for (int rg = 0; rg < RG; ++rg) {
    m[rg] = neg_inf();
    l[rg] = 0.f;
#pragma unroll
    for (int t = 0; t < DT; ++t) o[rg][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const auto query = [&](int rg, int ks) __attribute__((always_inline)) {
    return *reinterpret_cast<const u32x4*>(sq + (rg * KS + ks) * 1024 + lane * 16);
  };
  u32x4 qf[kShared ? 1 : RG][KS];
  issue_k(0);
  issue_v(0);
  issue_k(1);
  if constexpr (kShared) {
    issue_v(1);
    wait_dma<32>();  // the wave's part of the queries is in
    if (flip) {
#pragma unroll
      for (int i = 0; i < RG * KS; ++i)
        if (i % NW == wave) *reinterpret_cast<u32x4*>(sq + i * 1024 + lane * 16) ^= flip;
      wait_lgkmcnt0();
    }
    block_barrier();
  } else {
    wait_dma<24>();
#pragma unroll
    for (int rg = 0; rg < RG; ++rg)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[rg][ks] = query(rg, ks) ^ flip;
    wait_lgkmcnt0();
    issue_v(1);
  }
  for (int j = 0; j < n; ++j) {
    const char* sk = mine + (j & 1) * 16384;
    const char* sv = sk + 8192;
    wait_dma<24>();  // K of tile j is in; its V and tile j + 1 may be in flight
    // scores of keys kt + 16 kb + 4 g + e of the tile's span
    const int i = tile_at(j);
    const bool front = i < nft;
    const int kt = (front ? i : i - nft) * NK;
    const bool whole = front ? kt + NK <= s.n[0] : kt + NK <= hi_min && (kt >= lo_max || kt + NK <= s.sinks);
    u32x4 pf[RG][KB / 2];
    // Two groups of rows side by side, which hide each other's latencies: a SIMD has this
    // wave alone.  (The keys' fragments are read again for each pair: there are registers
    // for O alone.)
    constexpr int PG = RG > 1 ? 2 : 1;
#pragma unroll
    for (int rg0 = 0; rg0 < RG; rg0 += PG) {
      if constexpr (RG > 1) __builtin_amdgcn_sched_barrier(0);
      f32x4 sc[PG][KB];
#pragma unroll
      for (int u = 0; u < PG; ++u)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) sc[u][kb] = f32x4{0.f, 0.f, 0.f, 0.f};
      // the fragments of k-step ks + 1 are read while the MFMAs of ks run
      u32x4 q[2][PG], kf[2][KB];
      const auto read = [&](int ks) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < PG; ++u) q[ks & 1][u] = kShared ? query(rg0 + u, ks) : qf[kShared ? 0 : rg0 + u][ks];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const int row = kb * 16 + c16;
          kf[ks & 1][kb] = *reinterpret_cast<const u32x4*>(sk + row * (D * 2) + kslot<D>(row, ks * 4 + g) * 16);
        }
      };
      read(0);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (ks + 1 < KS) read(ks + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int u = 0; u < PG; ++u) sc[u][kb] = mfma16<T>(kf[ks & 1][kb], q[ks & 1][u], sc[u][kb]);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (rg0 + PG == RG) {
        wait_lgkmcnt0();
        issue_k(j + 2);
      }
      if (!whole) {
#pragma unroll
        for (int u = 0; u < PG; ++u) {
          const int rg = rg0 + u;
          const int up = (front ? s.n[0] : hi[rg]) - kt - 4 * g;
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[u][kb][e] = kb * 16 + e < up ? sc[u][kb][e] : neg_inf();
          if (!front && kt < lo_max) {  // hidden: [sinks, lo)
            const int sink = max(0, s.sinks) - kt - 4 * g;
            const uint32_t hidden = static_cast<uint32_t>(max(0, lo[rg] - kt - 4 * g - sink));
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                sc[u][kb][e] = static_cast<uint32_t>(kb * 16 + e - sink) < hidden ? neg_inf() : sc[u][kb][e];
          }
        }
      }
      float mx[PG];
      bool raise = false;
#pragma unroll
      for (int u = 0; u < PG; ++u) {
        float top[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          top[kb] = max3(sc[u][kb][0], sc[u][kb][1], sc[u][kb][2]);
          top[kb] = max3(top[kb], sc[u][kb][3], kb > 0 ? top[kb - 1] : top[kb]);
        }
        mx[u] = top[KB - 1] * c;
        raise = raise || mx[u] > m[rg0 + u] + kSlack;
      }
      if (__any(raise)) {
#pragma unroll
        for (int u = 0; u < PG; ++u) {
          const int rg = rg0 + u;
          mx[u] = fmaxf(mx[u], __shfl_xor(mx[u], 16, 64));
          mx[u] = fmaxf(mx[u], __shfl_xor(mx[u], 32, 64));
          const bool up = mx[u] > m[rg] + kSlack;
          const float alpha = up ? fast_exp2(m[rg] - mx[u]) : 1.f;
          m[rg] = up ? mx[u] : m[rg];
          l[rg] *= alpha;
#pragma unroll
          for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[rg][t][e] *= alpha;
        }
      }
#pragma unroll
      for (int u = 0; u < PG; ++u) {
        const int rg = rg0 + u;
        const float mb = m[rg] == neg_inf() ? 0.f : m[rg];  // nothing seen so far: P = 0
#pragma unroll
        for (int p = 0; p < KB / 2; ++p) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = fast_exp2(fmaf(sc[u][2 * p + (e >> 2)][e & 3], c, -mb));
          l[rg] += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
          pf[rg][p] = pack8<T>(x);  // keys 32 p + 4 g + 0..3 and 32 p + 16 + 4 g + 0..3
        }
      }
    }

    wait_dma<24>();  // V of tile j is in
    // V^T: lane row 16 t + (l & 15) at the keys of pf[p]; fragment i + kAhead is read
    // while the MFMAs of i run
    const auto read_v = [&](int i) __attribute__((always_inline)) {
      const int col = (i % DT) * 16 + (c16 & 3) * 4;
      s16x4 w[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int row = (i / DT) * 32 + u * 16 + g * 4 + (c16 >> 2);
        w[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_s16x4_t*)(sv + row * (D * 2) + vslot<D>(row, col >> 3) * 16 + ((col >> 2) & 1) * 8));
      }
      const u32x2 lw = __builtin_bit_cast(u32x2, w[0]), hw = __builtin_bit_cast(u32x2, w[1]);
      return u32x4{lw.x, lw.y, hw.x, hw.y};
    };
    constexpr int nv = KB / 2 * DT;
    u32x4 vf[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) vf[i] = read_v(i);
#pragma unroll
    for (int i = 0; i < nv; ++i) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int rg = 0; rg < RG; ++rg) o[rg][i % DT] = mfma16<T>(vf[i % kAhead], pf[rg][i / DT], o[rg][i % DT]);
      if (i + kAhead < nv) vf[i % kAhead] = read_v(i + kAhead);
    }
    __builtin_amdgcn_sched_barrier(0);
    wait_lgkmcnt0();
    issue_v(j + 2);
  }
  wait_dma<0>();  // no DMA may land in the LDS that the joining reuses

  // join the waves, a group of rows after the other: [wave][16] maxima, [wave][16]
  // sums, a bit per row that has to be computed again, the rows' places, then
  // [wave][16][D + 4] O
  float* sm = reinterpret_cast<float*>(smem);
  uint32_t* again = reinterpret_cast<uint32_t*>(sm + 2 * NW * 16);
  int64_t* to = reinterpret_cast<int64_t*>(sm + 2 * NW * 16 + 4);  // where each row goes
  float* so = sm + 2 * NW * 16 + 36;
  constexpr int LD = D + 4;
#pragma unroll
  for (int rg = 0; rg < RG; ++rg) {
    if (rg > 0 && rg * 16 >= rows) continue;
    __syncthreads();
    l[rg] += __shfl_xor(l[rg], 16, 64);
    l[rg] += __shfl_xor(l[rg], 32, 64);
    if (rg == 0 && threadIdx.x < 2) again[threadIdx.x] = 0;
    if (g == 0) {
      sm[wave * 16 + c16] = m[rg];
      sm[(NW + wave) * 16 + c16] = l[rg];
      if (rg % NW == wave) {
        const SpanRow x = span_row(a, f.mode, s, r0 + min(rg * 16 + c16, rows - 1));
        to[c16] = part.p ? part.at(a, x, slice) : x.b * a.ost[0] + x.h * a.ost[1] + x.t * a.ost[2];
      }
    }
#pragma unroll
    for (int t = 0; t < DT; ++t) *reinterpret_cast<f32x4*>(so + (wave * 16 + c16) * LD + t * 16 + 4 * g) = o[rg][t];
    __syncthreads();
    for (int it = threadIdx.x; it < 16 * (D / 4); it += 64 * NW) {
      const int row = it / (D / 4), d = (it - row * (D / 4)) * 4;
      if (rg * 16 + row >= rows || d >= a.D) continue;
      float mm = sm[row];
#pragma unroll
      for (int w = 1; w < NW; ++w) mm = fmaxf(mm, sm[w * 16 + row]);
      float sum = 0.f;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float mw = sm[w * 16 + row];
        // (a wave of which the row has seen nothing: 0 whatever it met)
        const float fw = mw == neg_inf() ? 0.f : fast_exp2(mw - mm);
        sum += sm[(NW + w) * 16 + row] * fw;
        const f32x4 ow = *reinterpret_cast<const f32x4*>(so + (w * 16 + row) * LD + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += mw == neg_inf() ? 0.f : ow[e] * fw;
      }
      const float any = (v[0] + v[1]) + (v[2] + v[3]);
      if (!(any == any) && sum == sum) atomicOr(&again[rg >> 1], 1u << ((rg & 1) * 16 + row));
      if (part.p) {
        const int64_t pa = to[row];
        if (d == 0) {
          float* ml = part.ml(a, pa);
          ml[0] = mm;
          ml[1] = sum;
        }
        *reinterpret_cast<f32x4*>(part.row(pa) + d) = v;
      } else {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;  // (a NaN sum passes through)
        T w4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w4[e] = static_cast<T>(v[e] * inv);
        *reinterpret_cast<u32x2*>(static_cast<T*>(a.o) + to[row] + d) =
            __builtin_bit_cast(u32x2, w4);
      }
    }
  }
  __syncthreads();
  const uint32_t bad0 = __builtin_amdgcn_readfirstlane(again[0]), bad1 = __builtin_amdgcn_readfirstlane(again[1]);
  uint64_t bad = static_cast<uint64_t>(bad1) << 32 | bad0;
  if (bad == 0) return;  // (the same for every wave)
  wait_vmcnt<0>();       // what has been written of these rows is written before what follows
  __syncthreads();
  while (bad != 0) {
    const int row = __builtin_ctzll(bad);
    bad &= bad - 1;
    if (row % NW != wave) continue;
    const SpanRow x = span_row(a, f.mode, s, r0 + row);
    float ro_[D / 16], rm, rl;
    span_attend_row<T, D / 16, 1>(a, s, x, min(i0 * NK, s.n[0]), min(i1 * NK, s.n[0]), max(0, min((i0 - nft) * NK, s.n[1])),
                               max(0, min((i1 - nft) * NK, s.n[1])), ro_, rm, rl);
    span_write_row<T, D / 16>(a, part, x, slice, ro_, rm, rl);
  }
}

// RGF, RGM: groups of rows of the blocks over shared prefixes (0: there are none) and
// of the others.
template <typename T, int D, int NW, int RGF, int RGM>
__global__ __launch_bounds__(64 * NW, 2) void k_span_few(SpanArgs a, FewBlocks front, FewBlocks main, SpanPart part) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];  // [wave][2 stages][K, V], queries
  const int64_t all = block_id();
  if (all >= static_cast<int64_t>(front.blocks) + main.blocks) return;  // the tail of a 2-D grid (the whole block)
  const uint32_t id = static_cast<uint32_t>(all);
  if constexpr (RGF > 0) {
    if (id < front.blocks) {
      few_block<T, D, NW, RGF>(a, front, part, id, smem);
      return;
    }
  }
  few_block<T, D, NW, RGM>(a, main, part, id - front.blocks, smem);
}

template <typename T, int D, int NW, int RGF, int RGM>
int launch_few(const SpanArgs& a, const FewBlocks& front, const FewBlocks& main, const SpanPart& part, hipStream_t st) {
  constexpr int kLds = NW * 32768 + kQueryLds<D, RGF>;
  static_assert((2 * NW * 16 + 36 + NW * 16 * (D + 4)) * 4 <= NW * 32768, "LDS");
  auto kern = k_span_few<T, D, NW, RGF, RGM>;
  if constexpr (kLds > 65536) {
    static std::atomic<uint64_t> done{0};
    if (int e = reserve_lds(reinterpret_cast<const void*>(kern), kLds, done, "attention")) return e;
  }
  note_kernel("%s few d%d waves%d rows%d+%d split%d+%d", a.pk ? "shared_prefix" : "sliding_window", D, NW, 16 * RGF, 16 * RGM, front.slices,
              main.slices);
  hipLaunchKernelGGL(kern, blocks_2d(static_cast<int64_t>(front.blocks) + main.blocks), dim3(64 * NW), kLds, st, a, front, main, part);
  return check_launch("attention");
}

template <typename T, int D, int NW, int RGF>
int launch_few(const SpanArgs& a, const FewBlocks& front, const FewBlocks& main, int rows, const SpanPart& part, hipStream_t st) {
  if constexpr (RGF != 1 && RGF != 2)  // (a group has more rows than a sequence)
    if (rows > 16) return launch_few<T, D, NW, RGF, 2>(a, front, main, part, st);
  return launch_few<T, D, NW, RGF, 1>(a, front, main, part, st);
}

template <typename T, int D>
int run_few(const SpanArgs& a, const FewPlan& p, const SpanPart& part, hipStream_t st) {
  FewBlocks front{}, main{};
  main.mode = p.mode;
  const int rows = static_cast<int>(span_rows(a, main.mode));  // <= kFewRows: one block of rows a set
  main.row_blocks = 1;
  main.slices = p.slices;
  main.first = part.first;
  main.sets = static_cast<uint32_t>(span_sets(a, main.mode));
  main.blocks = main.sets * main.slices;
  if (p.front_slices > 0) {
    front.mode = kFront;
    const int64_t front_rows = span_rows(a, kFront);
    front.row_blocks = static_cast<int>(ceil_div(front_rows, 64));
    front.slices = p.front_slices;
    front.sets = static_cast<uint32_t>(span_sets(a, kFront));
    front.blocks = front.sets * front.slices;
    if (front.row_blocks > 1) front.blocks = (front.blocks + 7) / 8 * 8 * front.row_blocks;
    if (front_rows <= 16) return launch_few<T, D, 2, 1>(a, front, main, rows, part, st);
    if (front_rows <= 32) return launch_few<T, D, 2, 2>(a, front, main, rows, part, st);
    return launch_few<T, D, 2, 4>(a, front, main, rows, part, st);
  }
  return p.waves == 1 ? launch_few<T, D, 1, 0>(a, front, main, rows, part, st) : launch_few<T, D, 2, 0>(a, front, main, rows, part, st);
}

}  // namespace

int span_few_run(int dtype, const SpanArgs& a, const FewPlan& p, const SpanPart& part, hipStream_t st) {
  if (dtype == NTOPS_BF16) return a.D > 64 ? run_few<__bf16, 128>(a, p, part, st) : run_few<__bf16, 64>(a, p, part, st);
  return a.D > 64 ? run_few<_Float16, 128>(a, p, part, st) : run_few<_Float16, 64>(a, p, part, st);
}

}  // namespace ntops
