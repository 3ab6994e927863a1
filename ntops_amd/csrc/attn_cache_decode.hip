// A few query rows over an 8-bit cache (decode): Sq * (Hq / Hkv) <= 32 rows per
// cache head.
//
// Bound by streaming the cache once.  A work item is (batch, cache head, slice
// of the sequence's tokens); the rows that share the head fill the 16 columns
// of v_mfma_f32_16x16x32 (S^T = K Q^T, O^T += V^T P^T), or twice 16 (RB 2), for
// which the cache's fragments are read and widened once.  Every wave owns its own
// key tiles, 4 KiB of keys and of values each (32 keys at a head dim of 128), in
// its own part of the LDS: direct non-temporal DMA two tiles ahead, refilled as
// soon as the tile's keys, then its values, have been read, and no barrier
// before the waves' merge.  A byte is a value here, so that per byte there is
// twice the work of 16-bit caches; a wave alone on its SIMD issues a vector
// instruction every 8 to 9 clocks at best, and two waves a SIMD hide that: (16, 32
// / 8 heads, 1, 2048 .. 4096, 128) bf16 in two waves a block of 8 KiB tiles 32.4
// us, in four 26.5, in eight of 4 KiB tiles 25.6; (1, 32 / 8, 1, 131072, 128) f16
// 59.5, 53.4, 51.4 (5.2 TB/s).
//
// e4m3 becomes bf16 (f16 for the keys of f16 queries) in registers, exactly: a
// key fragment is a 16-byte read whose halves feed two instructions, a value
// fragment a transposing 8-byte read.  The scale of a key's block times the
// softmax scale multiplies its scores, that of a value's block its
// probabilities, which are then rounded to bf16 whatever the query's type: only
// bf16 holds them under scales of any size.  For f16 queries the rest of the
// rounding is a second operand of the same product (pack_p).
//
// A NaN value reaches the rows that see it and no others, though P = 0 times it is
// NaN: in a tile that not every row sees whole (several positions, causal), NaN codes
// are noted for the rows that see them and cleared before the product.
//
// Slices are parts of the sequence's own length, known on the device only, so
// the number of slices is set by the GPU's size and an empty slice leaves an
// empty partial result.
#include <algorithm>
#include <atomic>

#include "attn_cache.h"

namespace ntops {
namespace {

constexpr int kMaxSplit = 64;

template <typename T>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (std::is_same<T, __bf16>::value)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}

// 16-byte slot of chunk c of row r in the tiles (D / 16 chunks a row): the
// reads of a key fragment (16 rows at one chunk) and of a value fragment (rows
// 0 .. 7 and 16 .. 23, or 8 .. 15 and 24 .. 31 of 32 in half a wave) each
// touch every bank once.  Involutions.
template <int D>
__device__ __forceinline__ int kslot8(int r, int c) {
  return kslot<D / 2>(r, c);
}
template <int D>
__device__ __forceinline__ int vslot8(int r, int c) {
  return D == 128 ? c ^ (((r >> 1) & 3) | ((r >> 4) & 1) << 2) : c ^ (((r >> 2) & 1) | ((r >> 4) & 1) << 1);
}

__device__ __forceinline__ void dma16_nt(u32x4 rsrc, uint32_t lds_dst, uint32_t voffset) {
  asm volatile("buffer_load_dwordx4 %0, %1, 0 offen nt lds"
               :
               : "v"(voffset), "s"(rsrc), "{m0}"(lds_dst)
               : "memory");
}

constexpr int kTileBytes = 4096;                  // a tile's keys, or its values
constexpr int kStage = 2 * kTileBytes + 2 * 256;  // and the scales of each
constexpr int kTileInst = kTileBytes / 1024 + 1;  // instructions of one, with its scales

// Loads of a tile's key (or value) rows, 4 instructions of 1 KiB, and of the
// scales of its 16-token parts, one instruction.
template <int D, bool IS_V>
struct TileDma {
  static constexpr int kInst = kTileBytes / 1024;
  static constexpr int kRows = 1024 / D;  // rows per instruction
  u32x4 rows, scales;
  uint32_t voff[kInst];
  uint32_t part;  // this lane's 16-token part, in tokens
  int first_part, shift;

  // base: the slice's first row (token t0, a multiple of 16); n: tokens from there on
  __device__ __forceinline__ void init(const uint8_t* base, int64_t ld, const float* scale, int64_t t0, int n, int lane,
                                       int dt, int block_shift) {
    rows = make_rsrc(base, n > 0 ? static_cast<uint32_t>((n - 1) * ld + dt) : 0u);
    shift = block_shift;
    const int64_t b0 = t0 >> shift;
    first_part = static_cast<int>(t0 - (b0 << shift));
    scales = make_rsrc(scale + b0, n > 0 ? static_cast<uint32_t>(((first_part + n - 1) >> shift) * 4 + 4) : 0u);
    part = static_cast<uint32_t>(lane * 16);
    constexpr int cpr = D / 16;
#pragma unroll
    for (int i = 0; i < kInst; ++i) {
      const int row = i * kRows + lane / cpr;
      const int c = IS_V ? vslot8<D>(row, lane % cpr) : kslot8<D>(row, lane % cpr);
      voff[i] = c * 16 < dt ? static_cast<uint32_t>(row * ld + c * 16) : kOOB;
    }
  }
  // The tile at token t of the slice (byte offset off) to dst, its scales to sdst.
  __device__ __forceinline__ void issue(uint32_t dst, uint32_t sdst, uint32_t off, int t) const {
#pragma unroll
    for (int i = 0; i < kInst; ++i)
      dma16_nt(rows, dst + i * 1024, voff[i] == kOOB ? kOOB : voff[i] + off);
    const uint32_t at = static_cast<uint32_t>(first_part + t) + part;
    dma4(scales, sdst, (at >> shift) * 4);
  }
};

template <int N>
__device__ __forceinline__ void wait_dma() {
  __builtin_amdgcn_sched_barrier(0);
  wait_vmcnt<N>();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// 8 e4m3 values (two words) as an operand of 8 T.
template <typename T>
__device__ __forceinline__ u32x4 widen8(uint32_t lo, uint32_t hi) {
  if constexpr (std::is_same<T, __bf16>::value)
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true))};
  else
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true))};
}

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2_t;

// part: fp32, per query row and slice the unnormalised O row, then (max in base
// 2, sum) pairs; null: one slice, O normalised into a.o.
template <typename T, int D, int NW, int RB>
__global__ __launch_bounds__(64 * NW, 1) void k_cache_decode(CacheAttnArgs a, int nsplit, float* part) {
  constexpr int NK = kTileBytes / D;  // keys per tile
  constexpr int KB = NK / 16;   // 16-key parts of a tile
  constexpr int KC = D / 64;    // 16-byte key reads of a lane per part: two k-steps each
  constexpr int DT = D / 16;    // 16-row tiles of O^T
  extern __shared__ __attribute__((aligned(1024))) char smem[];  // [wave][2 stages]

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4;
  const int64_t blk = block_id();
  if (blk >= static_cast<int64_t>(nsplit) * a.B * a.Hkv) return;  // the tail of a 2-D grid (the whole block)
  const int bh = static_cast<int>(blk / nsplit);
  const int sp = static_cast<int>(blk - static_cast<int64_t>(bh) * nsplit);
  const int b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int group = a.Hq / a.Hkv;
  constexpr int ROWS = 16 * RB;
  const int rows = group * a.Sq;  // <= ROWS
  const int64_t n_all = length_of(a, b);
  // this slice: whole rounds of the waves' tiles
  const int64_t step = NK * NW;
  const int64_t chunk = (n_all + nsplit * step - 1) / (nsplit * step) * step;
  const int64_t t0 = sp * chunk;
  const int n = __builtin_amdgcn_readfirstlane(static_cast<int>(max(int64_t(0), min(n_all - t0, chunk))));
  // query row of this lane's column, in each 16 rows: head hk * group + r / Sq, position r % Sq
  const int r = lane & 15;
  // keys of the slice that the rows see, and that every row sees
  int lim[RB];
#pragma unroll
  for (int x = 0; x < RB; ++x)
    lim[x] = a.causal ? static_cast<int>(max(int64_t(-1), min(int64_t(n), n_all - a.Sq + (16 * x + r) % a.Sq + 1 - t0))) : n;
  const int lim_min = a.causal ? static_cast<int>(max(int64_t(-1), min(int64_t(n), n_all - a.Sq + 1 - t0))) : n;

  // The query rows ahead of the first tiles, by DMA too (rows of D values, chunk c
  // of row r at slot c ^ r): as loads of their own they would be waited for first.
  // Every wave brings them all, to one place.
  constexpr int kQInst = ROWS * D / 512;  // instructions of 1 KiB
  constexpr int kQRows = 512 / D;         // rows of one
  const uint32_t q_lds = lds_addr(smem) + NW * 2 * kStage;
  {
    const T* Q = static_cast<const T*>(a.q) + b * a.qst[0] + static_cast<int64_t>(hk) * group * a.qst[1];
    const u32x4 rq = make_rsrc(Q, static_cast<uint32_t>(((group - 1) * a.qst[1] + (a.Sq - 1) * a.qst[2] + a.D) * 2));
#pragma unroll
    for (int i = 0; i < kQInst; ++i) {
      const int row = i * kQRows + lane / (D / 8);
      const int c = (lane % (D / 8)) ^ (row & (D / 8 - 1));
      const uint32_t at = static_cast<uint32_t>((row / a.Sq * a.qst[1] + row % a.Sq * a.qst[2]) * 2 + c * 16);
      dma16(rq, q_lds + i * 1024, row < rows && c * 8 < a.D ? at : kOOB);
    }
  }

  TileDma<D, false> kd;
  TileDma<D, true> vd;
  kd.init(a.k + b * a.kst[0] + hk * a.kst[1] + t0 * a.kst[2], a.kst[2], a.ks + b * a.kss[0] + hk * a.kss[1], t0, n, lane,
          a.D, a.shift);
  vd.init(a.v + b * a.vst[0] + hk * a.vst[1] + t0 * a.vst[2], a.vst[2], a.vs + b * a.vss[0] + hk * a.vss[1], t0, n, lane,
          a.D, a.shift);
  const int nt = (n + NK - 1) / NK;
  const int mine_n = nt > wave ? (nt - wave + NW - 1) / NW : 0;  // tiles wave, wave + NW, ..
  char* mine = smem + wave * (2 * kStage);
  const uint32_t mine_addr = lds_addr(mine);
  auto issue_k = [&](int j) {
    if (j >= mine_n) return;
    const int t = (wave + j * NW) * NK;
    const uint32_t st = mine_addr + (j & 1) * kStage;
    kd.issue(st, st + 2 * kTileBytes, static_cast<uint32_t>(t * a.kst[2]), t);
  };
  auto issue_v = [&](int j) {
    if (j >= mine_n) return;
    const int t = (wave + j * NW) * NK;
    const uint32_t st = mine_addr + (j & 1) * kStage;
    vd.issue(st + kTileBytes, st + 2 * kTileBytes + 256, static_cast<uint32_t>(t * a.vst[2]), t);
  };

  f32x4 o[RB][DT];
  float m[RB], l[RB];  // running max (base 2) of each row; this lane's part of its sum
#pragma unroll
  for (int x = 0; x < RB; ++x) {
#pragma unroll
    for (int t = 0; t < DT; ++t) o[x][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    m[x] = neg_inf();
    l[x] = 0.f;
  }

  issue_k(0);
  issue_v(0);
  issue_k(1);
  issue_v(1);
  // all but what was issued behind tile j's keys: its values, and the tile after it
  const auto wait_keys = [&](int j) {
    if (j + 1 < mine_n)
      wait_dma<3 * kTileInst>();
    else if (j < mine_n)
      wait_dma<kTileInst>();
    else
      wait_dma<0>();
  };
  wait_keys(0);  // and the queries
  u32x4 qf[RB][2 * KC];
#pragma unroll
  for (int x = 0; x < RB; ++x)
#pragma unroll
    for (int s = 0; s < 2 * KC; ++s) {
      const int c = ((s >> 1) * 4 + g) * 2 + (s & 1), row = 16 * x + r;  // the key bytes of k-step s in this lane
      qf[x][s] = *reinterpret_cast<const u32x4*>(smem + NW * 2 * kStage + row * (D * 2) + (c ^ (row & (D / 8 - 1))) * 16);
    }
  for (int j = 0; j < mine_n; ++j) {
    const char* sk = mine + (j & 1) * kStage;
    const char* sv = sk + kTileBytes;
    wait_keys(j);
    f32x4 s[RB][KB];
    float ks[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int x = 0; x < RB; ++x) s[x][kb] = f32x4{0.f, 0.f, 0.f, 0.f};
      ks[kb] = *reinterpret_cast<const float*>(sk + 2 * kTileBytes + kb * 4);
    }
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const int row = kb * 16 + (lane & 15);
        const u32x4 w = *reinterpret_cast<const u32x4*>(sk + row * D + kslot8<D>(row, c * 4 + g) * 16);
        const u32x4 k0 = widen8<T>(w.x, w.y), k1 = widen8<T>(w.z, w.w);
#pragma unroll
        for (int x = 0; x < RB; ++x) {
          s[x][kb] = mfma16<T>(k0, qf[x][2 * c], s[x][kb]);
          s[x][kb] = mfma16<T>(k1, qf[x][2 * c + 1], s[x][kb]);
        }
      }
    wait_lgkmcnt0();
    issue_k(j + 2);

    // scores of the slice's keys kt + 16 kb + 4 g + e
    const int kt = (wave + j * NW) * NK;
#pragma unroll
    for (int x = 0; x < RB; ++x) {
      float mx = neg_inf();
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[x][kb][e] *= ks[kb] * a.scale_log2;
      if (kt + NK > lim_min) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[x][kb][e] = kt + kb * 16 + 4 * g + e < lim[x] ? s[x][kb][e] : neg_inf();
      }
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[x][kb][e]);
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float m_new = fmaxf(m[x], mx);
      const float m_use = m_new == neg_inf() ? 0.f : m_new;  // nothing seen so far: P = 0
      if (__any(m_new > m[x])) {
        const float alpha = fast_exp2(m[x] - m_use);
        l[x] *= alpha;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[x][t][e] *= alpha;
        m[x] = m_new;
      }
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[x][kb][e] = fast_exp2(s[x][kb][e] - m_use);
          l[x] += s[x][kb][e];
        }
    }
    // values of tile j are in; behind them came tile j + 1, and the keys of j + 2
    if (j + 2 < mine_n)
      wait_dma<3 * kTileInst>();
    else if (j + 1 < mine_n)
      wait_dma<2 * kTileInst>();
    else
      wait_dma<0>();
    uint32_t nan[RB] = {};  // columns 16 t + 4 g + e (bit 4 t + e) that a NaN value reaches
    if (lim_min < n && kt + NK > lim_min) {
      char* own = const_cast<char*>(sv) + lane * 16;
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < kTileBytes / 1024; ++i) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(own + i * 1024);
#pragma unroll
        for (int e = 0; e < 4; ++e) any |= nan_bytes(w[e]);
      }
      if (__any(any != 0)) {
        for (int k = 0; k < NK; ++k) {
          uint32_t bits = 0;
#pragma unroll
          for (int t = 0; t < DT; ++t)
            bits |= byte_bits(nan_bytes(*reinterpret_cast<const uint32_t*>(sv + k * D + vslot8<D>(k, t) * 16 + 4 * g))) << (4 * t);
#pragma unroll
          for (int x = 0; x < RB; ++x) nan[x] |= kt + k < lim[x] ? bits : 0;
        }
        for (int i = 0; i < kTileBytes / 1024; ++i) {
          u32x4 w = *reinterpret_cast<const u32x4*>(own + i * 1024);
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] &= ~(nan_bytes(w[e]) * 0xffu);
          *reinterpret_cast<u32x4*>(own + i * 1024) = w;
        }
        asm volatile("" ::: "memory");  // a wave's LDS operations run in order: written, then read by other lanes
      }
    }
    constexpr bool LO = std::is_same<T, _Float16>::value;
    u32x4 pf[RB][KB / 2], pl[RB][KB / 2];
#pragma unroll
    for (int p = 0; p < KB / 2; ++p) {
      float v[RB][8];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float vs = *reinterpret_cast<const float*>(sk + 2 * kTileBytes + 256 + (2 * p + u) * 4);
#pragma unroll
        for (int x = 0; x < RB; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[x][4 * u + e] = s[x][2 * p + u][e] * vs;
      }
#pragma unroll
      for (int x = 0; x < RB; ++x) pack_p<LO>(v[x], pf[x][p], pl[x][p]);  // keys 32 p + 4 g + 0..3 and 32 p + 16 + 4 g + 0..3
    }
#pragma unroll
    for (int p = 0; p < KB / 2; ++p)
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        // V^T: lane row 16 t + (l & 15) at the keys of pf[p]: of the 16 lanes
        // of a read, two hold 8 columns each of one of its 8 rows
        const int i = lane & 15;
        const int row = p * 32 + ((i >> 3) & 1) * 16 + g * 4 + ((i >> 1) & 3);
        const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            (lds_i32x2_t*)(sv + row * D + vslot8<D>(row, t) * 16 + (i & 1) * 8));
        const u32x4 vf = widen8<__bf16>(w.x, w.y);
#pragma unroll
        for (int x = 0; x < RB; ++x) {
          o[x][t] = mfma16<__bf16>(vf, pf[x][p], o[x][t]);
          if constexpr (LO) o[x][t] = mfma16<__bf16>(vf, pl[x][p], o[x][t]);
        }
      }
    if (lim_min < n && kt + NK > lim_min)
#pragma unroll
      for (int x = 0; x < RB; ++x)
        if (__any(nan[x] != 0))
#pragma unroll
          for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (nan[x] >> (4 * t + e) & 1) o[x][t][e] = __builtin_nanf("");
    wait_lgkmcnt0();
    issue_v(j + 2);
  }
#pragma unroll
  for (int x = 0; x < RB; ++x) {
    l[x] += __shfl_xor(l[x], 16, 64);
    l[x] += __shfl_xor(l[x], 32, 64);
  }
  wait_dma<0>();  // no DMA may land in the LDS the merge reuses
  __syncthreads();

  // merge the waves: per-wave (max, sum) of every row, then O scaled to the
  // block's max
  float* sm = reinterpret_cast<float*>(smem);  // [wave][ROWS] max, [wave][ROWS] sum, then [wave][ROWS][D + 4] O
  float* so = sm + 2 * NW * ROWS;
  constexpr int LD = D + 4;
  if (g == 0)
#pragma unroll
    for (int x = 0; x < RB; ++x) {
      sm[wave * ROWS + 16 * x + r] = m[x];
      sm[(NW + wave) * ROWS + 16 * x + r] = l[x];
    }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < RB; ++x) {
    const int row = 16 * x + r;
    float mb = sm[row];
#pragma unroll
    for (int w = 1; w < NW; ++w) mb = fmaxf(mb, sm[w * ROWS + row]);
    // A row that sees none of the wave's keys has no max, and 0 whatever it met of
    // the values.  (One whose scores are all NaN has a NaN sum.)
    const bool none = m[x] == neg_inf();
    const float f = fast_exp2(m[x] - mb);
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) so[(wave * ROWS + row) * LD + t * 16 + 4 * g + e] = none ? 0.f : o[x][t][e] * f;
  }
  __syncthreads();
  const int64_t nrow = static_cast<int64_t>(a.B) * a.Hq * a.Sq;
  float* part_ml = part + nrow * nsplit * a.D;
  for (int i = threadIdx.x; i < rows * (D / 4); i += 64 * NW) {
    const int row = i / (D / 4), d = (i - row * (D / 4)) * 4;
    if (d >= a.D) continue;
    float mm = sm[row];
#pragma unroll
    for (int w = 1; w < NW; ++w) mm = fmaxf(mm, sm[w * ROWS + row]);
    float sum = 0.f;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float mw = sm[w * ROWS + row], lw = sm[(NW + w) * ROWS + row];
      sum += mw == neg_inf() ? lw : lw * fast_exp2(mw - mm);  // (no max: 0, or NaN)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += so[(w * ROWS + row) * LD + d + e];
    }
    const int hh = hk * group + row / a.Sq, qq = row % a.Sq;
    if (part) {
      const int64_t at = ((static_cast<int64_t>(b) * a.Hq + hh) * a.Sq + qq) * nsplit + sp;
      if (d == 0) {
        part_ml[2 * at] = mm;
        part_ml[2 * at + 1] = sum;
      }
      *reinterpret_cast<f32x4*>(part + at * a.D + d) = f32x4{v[0], v[1], v[2], v[3]};
    } else {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      T w4[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w4[e] = static_cast<T>(v[e] * inv);
      *reinterpret_cast<u32x2*>(static_cast<T*>(a.o) + b * a.ost[0] + hh * a.ost[1] + qq * a.ost[2] + d) =
          __builtin_bit_cast(u32x2, w4);
    }
  }
}

// Combines the slices of every query row in slice order: one wave per row.
template <typename T>
__global__ __launch_bounds__(256) void k_cache_merge(CacheAttnArgs a, int nsplit, const float* part) {
  const int lane = threadIdx.x & 63;
  const int64_t nrow = static_cast<int64_t>(a.B) * a.Hq * a.Sq;
  const int64_t row = block_id() * 4 + (threadIdx.x >> 6);
  if (row >= nrow) return;
  const float* po = part + row * nsplit * a.D;
  const float* ml = part + nrow * nsplit * a.D + 2 * row * nsplit;
  const int d = lane * 2;
  constexpr int kAtOnce = 16;
  const auto load = [&](int s0, float2 (&v)[kAtOnce]) {
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u)
      v[u] = s0 + u < nsplit && d < a.D ? *reinterpret_cast<const float2*>(po + static_cast<int64_t>(s0 + u) * a.D + d)
                                        : float2{0.f, 0.f};
  };
  float2 v[kAtOnce];
  load(0, v);  // in flight while the weights are formed
  float m = neg_inf(), l = 0.f;
  if (lane < nsplit) {
    m = ml[2 * lane];
    l = ml[2 * lane + 1];
  }
  const float mm = wave_max(m);
  const float w = m == neg_inf() ? 0.f : fast_exp2(m - mm);
  const float sum = wave_sum(m == neg_inf() ? l : l * w);  // (no max: 0, or NaN)
  float x = 0.f, y = 0.f;
  for (int s0 = 0; s0 < nsplit; s0 += kAtOnce) {
    if (s0 > 0) load(s0, v);
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const float ws = s0 + u < nsplit ? lane_read(w, s0 + u) : 0.f;
      x += ws * v[u].x;
      y += ws * v[u].y;
    }
  }
  if (d < a.D) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int q = static_cast<int>(row % a.Sq);
    const int64_t bh = row / a.Sq;
    T* O = static_cast<T*>(a.o) + (bh / a.Hq) * a.ost[0] + (bh % a.Hq) * a.ost[1] + q * a.ost[2];
    T v2[2] = {static_cast<T>(x * inv), static_cast<T>(y * inv)};
    *reinterpret_cast<uint32_t*>(O + d) = __builtin_bit_cast(uint32_t, v2);
  }
}

// Waves of a block and slices of a sequence.  The sequences' lengths are not
// known here: as many slices as leave about one eight-wave block per CU, none
// shorter than two tiles a wave at full length (twice the slices: (16, 32 / 8, 1,
// 2048 .. 4096, 128) 26.5 -> 30.3 us with four-wave blocks).  From one head per CU
// on four-wave blocks, two to a CU, hide each other's start ((64, 32 / 32, 1, 512 ..
// 1024, 128): eight-wave ones 85.1 us, four 68.7, two 73.8; (100, 32 / 8, 1, 2048 ..
// 4096, 128): four 114, two 124; (33, 32 / 8, 1, 500 .. 1000, 128): eight 19.7, four
// 17.9; 448 heads over 2048 .. 4096: 66.1, 67.3).  Up to one and a half heads per CU
// that leaves half the CUs idle at the end, and a long sequence goes in three
// slices: 264 heads over 4096 67.5 -> 59.8 us, over 2048 .. 4096 48.9 -> 46.5, 320
// 70.6 -> 61.3 and 55.9 -> 51.8, 384 73.9 -> 73.2, but 448 78.7 -> 85.0.
void decode_split(int64_t heads, int64_t C, int64_t D, int& waves, int& nsplit) {
  const int64_t cus = cu_count_cached();
  waves = heads > cus ? 4 : 8;
  const int64_t step = (D > 64 ? 32 : 64) * waves;
  int64_t n = std::min({static_cast<int64_t>(kMaxSplit), cus / heads, ceil_div(C, 2 * step)});
  if (n <= 2 && C <= 8 * step) n = 1;  // two short slices gain what the merge's launch costs
  if (heads > cus && 2 * heads <= 3 * cus && C > 2048) n = 3;
  nsplit = static_cast<int>(std::max<int64_t>(n, 1));
}

template <typename T, int D, int NW, int RB>
int launch_decode(const CacheAttnArgs& a, int nsplit, float* part, hipStream_t st) {
  constexpr int kLds = NW * 2 * kStage + 32 * D * RB;
  static_assert((2 * NW + NW * (D + 4)) * 16 * RB * 4 <= kLds && kLds * 8 / NW <= 163840, "LDS");
  auto kern = k_cache_decode<T, D, NW, RB>;
  static std::atomic<uint64_t> reserved{0};
  if (const int rc = reserve_lds(reinterpret_cast<const void*>(kern), kLds, reserved, "kv_cache_attention"); rc != NTOPS_OK) return rc;
  const int64_t blocks = static_cast<int64_t>(nsplit) * a.B * a.Hkv;
  note_kernel("kv_cache_decode d%d rows%d waves%d split%d", D, 16 * RB, NW, nsplit);
  hipLaunchKernelGGL(kern, blocks_2d(blocks), dim3(64 * NW), kLds, st, a, nsplit, part);
  if (part) cache_merge(std::is_same<T, __bf16>::value ? NTOPS_BF16 : NTOPS_F16, a, nsplit, part, st);
  return check_launch("kv_cache_attention");
}

template <typename T>
int run_decode(const CacheAttnArgs& a, void* ws, int64_t ws_bytes, hipStream_t st) {
  int waves, nsplit;
  decode_split(static_cast<int64_t>(a.B) * a.Hkv, a.C, a.D, waves, nsplit);
  const int64_t need = cache_decode_workspace(a.B, a.Hq, a.Hkv, a.Sq, a.C, a.D);
  if (need == 0 || ws == nullptr || ws_bytes < need) {
    nsplit = 1;
    ws = nullptr;
  }
  float* part = static_cast<float*>(ws);
  const auto go = [&](auto rb) {
    constexpr int RB = decltype(rb)::value;
    if (waves == 8) return a.D > 64 ? launch_decode<T, 128, 8, RB>(a, nsplit, part, st) : launch_decode<T, 64, 8, RB>(a, nsplit, part, st);
    return a.D > 64 ? launch_decode<T, 128, 4, RB>(a, nsplit, part, st) : launch_decode<T, 64, 4, RB>(a, nsplit, part, st);
  };
  return a.Sq * (a.Hq / a.Hkv) <= 16 ? go(std::integral_constant<int, 1>{}) : go(std::integral_constant<int, 2>{});
}

}  // namespace

void cache_merge(int dtype, const CacheAttnArgs& a, int nsplit, const float* part, hipStream_t st) {
  const int64_t rows = static_cast<int64_t>(a.B) * a.Hq * a.Sq;
  const auto kern = dtype == NTOPS_BF16 ? &k_cache_merge<__bf16> : &k_cache_merge<_Float16>;
  hipLaunchKernelGGL(kern, blocks_2d(ceil_div(rows, 4)), dim3(256), 0, st, a, nsplit, part);
}

bool cache_matrix_layout(const CacheAttnArgs& a, int dtype) {
  const auto q8 = [](const int64_t* s) { return s[2] % 8 == 0 && s[1] % 8 == 0 && s[0] % 8 == 0; };
  const auto c16 = [](const int64_t* s) { return s[2] % 16 == 0 && s[1] % 16 == 0 && s[0] % 16 == 0; };
  const int64_t ld = std::max(a.kst[2], a.vst[2]);
  return (dtype == NTOPS_BF16 || dtype == NTOPS_F16) && a.C > 0 && a.D % 16 == 0 && a.D <= 128 && q8(a.qst) &&
         a.ost[2] % 4 == 0 && a.ost[1] % 4 == 0 && a.ost[0] % 4 == 0 && c16(a.kst) && c16(a.vst) && aligned16(a.q) &&
         aligned16(a.k) && aligned16(a.v) && (reinterpret_cast<uintptr_t>(a.o) & 7u) == 0 && a.qst[1] >= 0 && a.qst[2] >= 0 &&
         (a.Hq / a.Hkv) * a.qst[1] + static_cast<int64_t>(a.Sq) * a.qst[2] < (int64_t(1) << 29) && a.kst[2] >= a.D &&
         a.vst[2] >= a.D && (a.C + 1024) * ld < 0x7fffffffLL && a.C < (int64_t(1) << 30);
}

bool cache_decode_serves(const CacheAttnArgs& a, int dtype) {
  return cache_matrix_layout(a, dtype) && static_cast<int64_t>(a.Sq) * (a.Hq / a.Hkv) <= kDecodeRows &&
         static_cast<int64_t>(a.B) * a.Hkv <= 0x7fffffffLL / kMaxSplit;
}

int64_t cache_decode_workspace(int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t C, int64_t D) {
  if (Sq * (Hq / Hkv) > kDecodeRows || D % 16 != 0 || D > 128 || C == 0) return 0;
  int waves, nsplit;
  decode_split(B * Hkv, C, D, waves, nsplit);
  return nsplit > 1 ? B * Hq * Sq * nsplit * (D + 2) * 4 : 0;
}

int cache_decode(int dtype, const CacheAttnArgs& a, void* workspace, int64_t workspace_bytes, hipStream_t st) {
  return dtype == NTOPS_BF16 ? run_decode<__bf16>(a, workspace, workspace_bytes, st)
                             : run_decode<_Float16>(a, workspace, workspace_bytes, st);
}

}  // namespace ntops
