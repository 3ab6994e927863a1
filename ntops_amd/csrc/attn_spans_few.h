// Few query rows a cache head (single tokens, drafted ones): windowed and
// shared-prefix attention bound by streaming keys and values once.
//
// The rows that share a cache head fill the 16 columns of v_mfma_f32_16x16x32, one or
// two such groups of them, so that a key that has reached the LDS serves up to 32
// rows (S^T = K Q^T: a lane's scores all belong to one row, and P^T feeds
// O^T += V^T P^T from registers).  Every wave owns tiles of 8 KiB of keys and 8 KiB
// of values in its own part of the LDS, loaded by direct DMA two tiles ahead and
// refilled as soon as they are read: no barrier before the waves are joined.  Tiles
// never mix the two spans: those of the front come first.  A SIMD has one or two of
// these waves, so fragments are read ahead of the MFMAs that use them (without, 2 %
// more).
//
// Bound by the HBM where there are keys for every CU: bf16 (64, 32 / 8, 1 over up to 8192,
// window 4096) of 128 columns 150 to 154 us, 6.4 TB/s; few keys by latency: (1, 32 / 8, 1 over 4096,
// window 1024) 9.2 us and 3.5 the merge, of which the start, the lengths, the addresses
// that follow from them and the first tile take most, one after the other.
//
// What a row does not see: masked scores are -inf whatever their key holds.  A
// value that is not finite times P = 0 is NaN, though; a row whose result is NaN, or past
// fp32's range, under a sum that is a number is computed again by itself, from the keys
// that it sees.
#pragma once

#include "attn_spans.h"

namespace ntops {
namespace span_few {

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
  // nothing but the columns of O past the head dim.  That is the next key, which is read
  // anyway, where a head's keys lie side by side, but another head's where a token's heads do:
  // (64, 32 / 8, 1 over 8192, window 4096) of 80 columns 101 / 189 us, of 128 160 / 169.
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
  int mode;  // SpanMode
  int slices;
  int first;  // slice of the rows that slice 0 is
  uint32_t blocks;
};

inline FewBlocks few_blocks(const SpanArgs& a, int mode, int slices, int first) {
  return {mode, slices, first, static_cast<uint32_t>(span_sets(a, mode)) * static_cast<uint32_t>(slices)};
}

// RG: groups of 16 rows a block has room for.
template <typename T, int D, int NW, int RG>
__device__ __forceinline__ void few_block(const SpanArgs& a, const FewBlocks& f, SpanPart part, uint32_t id, char* smem) {
  constexpr int NK = kTileKeys<D>;
  constexpr int KB = NK / 16;  // 16-key blocks of a tile
  constexpr int KS = D / 32;   // k-steps of S^T = K Q^T
  constexpr int DT = D / 16;   // 16-row tiles of O^T
  static_assert((2 * NW * 16 + 36 + NW * 16 * (D + 4)) * 4 <= NW * 32768, "the joining's LDS");
  static_assert(RG * KS * 1024 <= 8192, "the queries go through the LDS of a tile's values, which are loaded after them");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c16 = lane & 15;
  const uint32_t set = id / static_cast<uint32_t>(f.slices);
  const int slice = static_cast<int>(id - set * f.slices);
  const int ro = a.group * a.Sq;
  const int rows = f.mode == kFront ? ro * a.per : ro;  // <= 16 RG
  const int t1 = f.mode == kFront ? 0 : static_cast<int>(static_cast<uint32_t>(rows - 1) / static_cast<uint32_t>(a.group));
  part.first = f.first;

  // The queries are on their way before the lengths are known.
  char* mine = smem + wave * 32768;
  const uint32_t mine_addr = lds_addr(mine);
  char* sq = mine + 16384 + 8192;  // [rg][ks][lane]
  int token[RG];
  {
    const SpanSet w = span_set(a, f.mode, set);
    const T* Q = static_cast<const T*>(a.q) + w.b0 * a.qst[0] + static_cast<int64_t>(w.hk) * a.group * a.qst[1];
    const u32x4 rq = make_rsrc(Q, 0x7ffffff0);
    const uint32_t sq_addr = lds_addr(sq);
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
      const int r = rg * 16 + c16;
      const SpanRow x = span_row(a, f.mode, w, min(r, rows - 1));
      token[rg] = x.t;
      const uint32_t off = static_cast<uint32_t>(((x.b - w.b0) * a.qst[0] + (x.h - w.hk * a.group) * a.qst[1] + x.t * a.qst[2]) * 2);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int d0 = ks * 32 + 8 * g;
        dma16(rq, __builtin_amdgcn_readfirstlane(sq_addr + (rg * KS + ks) * 1024), r < rows && d0 < a.D ? off + d0 * 2 : kOOB);
      }
    }
  }
  const Spans s = make_spans<2>(a, f.mode, set, 0, t1);
  int hi[RG], lo[RG];
#pragma unroll
  for (int rg = 0; rg < RG; ++rg) {
    hi[rg] = s.hi(token[rg]);
    lo[rg] = s.lo(token[rg]);
  }
  // (under a zero scale the least factor there is, so that a masked score stays -inf)
  const float c = a.scale_log2 == 0.f ? 0x1p-149f : fabsf(a.scale_log2);
  const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;  // a negative scale: -Q
  const int hi_min = s.hi(0), lo_max = s.lo(t1);  // a main tile between them is seen whole by every row

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
  // exponents are by * score - mb: of c and the reference (0: nothing seen so far, P = 0), or
  // where `far` (span_far of some row's reference, wave-uniform) of scores that are exponents
  float by = c, mb[RG];
  bool far = false;
#pragma unroll
  for (int rg = 0; rg < RG; ++rg) {
    m[rg] = neg_inf();
    mb[rg] = 0.f;
    l[rg] = 0.f;
#pragma unroll
    for (int t = 0; t < DT; ++t) o[rg][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const auto query = [&](int rg, int ks) __attribute__((always_inline)) {
    return *reinterpret_cast<const u32x4*>(sq + (rg * KS + ks) * 1024 + lane * 16);
  };
  u32x4 qf[RG][KS];
  issue_k(0);
  issue_v(0);
  issue_k(1);
  wait_dma<24>();
#pragma unroll
  for (int rg = 0; rg < RG; ++rg)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[rg][ks] = query(rg, ks) ^ flip;
  wait_lgkmcnt0();
  issue_v(1);
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
    f32x4 sc[RG][KB];
#pragma unroll
    for (int rg = 0; rg < RG; ++rg)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) sc[rg][kb] = f32x4{0.f, 0.f, 0.f, 0.f};
    // the fragments of k-step ks + 1 are read while the MFMAs of ks run
    u32x4 kf[2][KB];
    const auto read = [&](int ks) __attribute__((always_inline)) {
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
        for (int rg = 0; rg < RG; ++rg) sc[rg][kb] = mfma16<T>(kf[ks & 1][kb], qf[rg][ks], sc[rg][kb]);
      __builtin_amdgcn_sched_barrier(0);
    }
    wait_lgkmcnt0();
    issue_k(j + 2);
    if (!whole) {
#pragma unroll
      for (int rg = 0; rg < RG; ++rg) {
        const int up = (front ? s.n[0] : hi[rg]) - kt - 4 * g;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[rg][kb][e] = kb * 16 + e < up ? sc[rg][kb][e] : neg_inf();
        if (!front && kt < lo_max) {  // hidden: [sinks, lo)
          const int sink = max(0, s.sinks) - kt - 4 * g;
          const uint32_t hidden = static_cast<uint32_t>(max(0, lo[rg] - kt - 4 * g - sink));
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              sc[rg][kb][e] = static_cast<uint32_t>(kb * 16 + e - sink) < hidden ? neg_inf() : sc[rg][kb][e];
        }
      }
    }
    float mx[RG];
    bool raise = false;
    const uint32_t seen = read_of(sc[0][KB - 1][3], sc[RG - 1][KB - 1][3]);
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
      float top[KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        top[kb] = max3_after(sc[rg][kb][0], sc[rg][kb][1], sc[rg][kb][2], seen);
        top[kb] = max3(top[kb], sc[rg][kb][3], kb > 0 ? top[kb - 1] : top[kb]);
      }
      mx[rg] = top[KB - 1] * c;
      raise = raise || mx[rg] > m[rg] + kSlack;
    }
    raise = __any(raise);
    if (raise || far) {
      if (raise) {
#pragma unroll
        for (int rg = 0; rg < RG; ++rg) {
          mx[rg] = fmaxf(mx[rg], __shfl_xor(mx[rg], 16, 64));
          mx[rg] = fmaxf(mx[rg], __shfl_xor(mx[rg], 32, 64));
          const bool up = mx[rg] > m[rg] + kSlack;
          const float alpha = up ? fast_exp2(m[rg] - mx[rg]) : 1.f;
          m[rg] = up ? mx[rg] : m[rg];
          l[rg] *= alpha;
#pragma unroll
          for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[rg][t][e] *= alpha;
          mb[rg] = m[rg] == neg_inf() ? 0.f : m[rg];
          far = far || __any(span_far(m[rg]));
        }
      }
      if (far) {
#pragma unroll
        for (int rg = 0; rg < RG; ++rg) {
          const float ref = m[rg] == neg_inf() ? 0.f : m[rg];
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[rg][kb][e] = product(sc[rg][kb][e], c) - ref;
          mb[rg] = 0.f;
        }
        by = 1.f;
      }
    }
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
#pragma unroll
      for (int p = 0; p < KB / 2; ++p) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = fast_exp2(fmaf(sc[rg][2 * p + (e >> 2)][e & 3], by, -mb[rg]));
        l[rg] += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        // (rounded to the type for the second product, the sum above not: attn_spans_tile.h)
        pf[rg][p] = pack8<T>(x);  // keys 32 p + 4 g + 0..3 and 32 p + 16 + 4 g + 0..3
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
    if (rg == 0 && threadIdx.x == 0) *again = 0;
    if (g == 0) {
      sm[wave * 16 + c16] = m[rg];
      sm[(NW + wave) * 16 + c16] = l[rg];
      if (rg % NW == wave) {
        const SpanRow x = span_row(a, f.mode, s, min(rg * 16 + c16, rows - 1));
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
      if (span_again(any, sum)) atomicOr(again, 1u << (rg * 16 + row));
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
        for (int e = 0; e < 4; ++e) w4[e] = mean_as<T>(v[e] * inv);
        *reinterpret_cast<u32x2*>(static_cast<T*>(a.o) + to[row] + d) =
            __builtin_bit_cast(u32x2, w4);
      }
    }
  }
  __syncthreads();
  uint32_t bad = __builtin_amdgcn_readfirstlane(*again);
  if (bad == 0) return;  // (the same for every wave)
  wait_vmcnt<0>();       // what has been written of these rows is written before what follows
  __syncthreads();
  while (bad != 0) {
    const int row = __builtin_ctz(bad);
    bad &= bad - 1;
    if (row % NW != wave) continue;
    const SpanRow x = span_row(a, f.mode, s, row);
    span_row_again<T, D / 16>(a, s, part, x, slice, min(i0 * NK, s.n[0]), min(i1 * NK, s.n[0]), max(0, min((i0 - nft) * NK, s.n[1])),
                              max(0, min((i1 - nft) * NK, s.n[1])));
  }
}

}  // namespace span_few
}  // namespace ntops
