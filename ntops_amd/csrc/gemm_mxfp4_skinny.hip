// MXFP4 products of up to 32 rows (decode projections): bound by streaming B,
// (16 + 1) / 32 bytes a value, once.
//
// A block covers 16 J columns; its four waves each own K steps of their own and
// stream them through their own part of the LDS by direct DMA, as many steps ahead
// as half a CU's LDS holds (one to three), with no barrier before their fp32 sums are
// merged.  Two blocks share a CU, so that one streams while the other starts or
// merges: 1 row, 100000 x 4096 took 52.2 us with one block of twice the ring a CU and
// 38.7 with two (now 36.1, 6.0 TB/s), 28672 x 4096 17.8 and 15.1.  A step is 4 or (J 4) 8 KiB of B (16 J
// rows of 256 or 128 bytes, non-temporal, whole lines), the same columns of A's
// rows, and the scales; steps of 8 KiB for J 1 left the ring one step shorter, 8.2 us
// -> 10.4 at 1 row, 4096 x 14336.  Up to 4 rows (MR 4) A's part of a step is a
// quarter, and the ring longer; the instruction's other rows read the four again.  From
// 17 rows on (MR 32) two sixteens use B's fragments: 17 rows, 4096 x 4096 6.2 us (in
// 64 x 64 tiles 8.8), 32 rows, 14336 x 4096 11.5 (12.6), 4096 x 14336 13.7 (15.8), 1000
// x 2000 4.5 (6.9).
//
// The scales are loaded as the dwords that the step's CPR bytes of a row lie in (one
// more than they fill, as a row may start inside one) and read as single bytes;
// bytes behind the row's last block count as 0, as they may be another row's 255.
// Such a dword may reach up to 3 bytes past the scales' end or before their start;
// being aligned it lies within what the memory's page holds.
//
// Activations that are still 16-bit (X) are quantized here, up to 4 rows: a step's
// A is then its raw values, a lane rounds whole blocks of them (mxfp4.h), and the
// codes go to the LDS, where the fragments are read as ever.  Every block rounds the
// same rows again, which pays for up to 4 of them: a kernel before this one and then
// this one, against this one alone, in a captured graph, took 1 row of 4096 values
// 5.5 against 4.2 us for 640 columns and 10.9 against 9.5 for 14336; 4 rows 5.6
// against 4.5 and 11.0 against 9.9, and 4 rows of 14336 values, the most a wave has
// to round, 10.7 against 10.2 for 4096 columns.
#include <algorithm>
#include <atomic>

#include "gemm_mxfp4.h"
#include "mxfp4.h"

namespace ntops {
namespace {

constexpr int kWaves = 4;

// 16-byte slot of chunk c of row r, CPR chunks a row: the 16 rows of a fragment
// read touch 16 different slots of the LDS's 256 bytes.
template <int CPR>
__device__ __forceinline__ int sk_slot(int r, int c) {
  return CPR == 8 ? kslot<64>(r, c) : c ^ (r & 15);
}

template <bool NT>
__device__ __forceinline__ void sk_dma(u32x4 rsrc, uint32_t dst, uint32_t off) {
  if constexpr (NT)
    asm volatile("buffer_load_dwordx4 %0, %1, 0 offen nt lds" : : "v"(off), "s"(rsrc), "{m0}"(dst) : "memory");
  else
    dma16(rsrc, dst, off);
}

// One operand's steps: ROWS rows of CPR blocks, and their scales.
template <int ROWS, int CPR, bool NT>
struct Loader {
  static constexpr int kInst = (ROWS * CPR + 63) / 64;
  static constexpr int kRpi = 64 / CPR;  // rows per instruction
  static constexpr int ND = CPR / 4 + 1;  // dwords of a row's scales
  static constexpr int kScaleInst = (ROWS * ND + 63) / 64;
  static constexpr int kBytes = kInst * 1024, kScaleBytes = kScaleInst * 256;
  u32x4 codes, scales;
  uint32_t voff[kInst], soff[kScaleInst];
  int kb;

  // the step's block that this lane brings with instruction i
  __device__ __forceinline__ static int chunk(int lane, int i) {
    return sk_slot<CPR>(i * kRpi + lane / CPR, lane % CPR);
  }
  // rows: valid ones
  __device__ __forceinline__ void init(const uint8_t* c, int64_t ld, const uint8_t* s, int64_t lds, int rows, int blocks,
                                       int lane) {
    kb = blocks;
    codes = make_rsrc(c, (rows - 1) * ld + blocks * 16ll);
    const int o = static_cast<int>(reinterpret_cast<uintptr_t>(s) & 3u);
    scales = make_rsrc(s - o, (o + (rows - 1) * lds + blocks + 3) & ~3ll);
#pragma unroll
    for (int i = 0; i < kInst; ++i) {
      const int r = i * kRpi + lane / CPR;
      voff[i] = r < rows && r < ROWS ? static_cast<uint32_t>(r * ld + chunk(lane, i) * 16) : kOOB;
    }
#pragma unroll
    for (int i = 0; i < kScaleInst; ++i) {
      const int id = i * 64 + lane, r = id / ND;
      soff[i] = r < rows && r < ROWS ? (static_cast<uint32_t>(o + r * lds) & ~3u) + (id - r * ND) * 4 : kOOB;
    }
  }
  __device__ __forceinline__ void issue(uint32_t dst, int b0, int lane) const {
#pragma unroll
    for (int i = 0; i < kInst; ++i)
      sk_dma<NT>(codes, dst + i * 1024,
                 voff[i] != kOOB && b0 + chunk(lane, i) < kb ? voff[i] + static_cast<uint32_t>(b0) * 16 : kOOB);
#pragma unroll
    for (int i = 0; i < kScaleInst; ++i)
      dma4(scales, dst + kBytes + i * 256, soff[i] != kOOB ? soff[i] + static_cast<uint32_t>(b0) : kOOB);
  }
};

// Raw rows of 32 CPR 16-bit values: 16-byte piece p of block c at piece p ^ (c & 3),
// for reads of whole blocks by neighbouring lanes.
template <int ROWS, int CPR>
struct RawLoader {
  static constexpr int kInst = ROWS * CPR / 16;
  static constexpr int kBytes = kInst * 1024, kScaleBytes = 0, kScaleInst = 0;
  u32x4 rows;
  uint32_t voff[kInst];
  int row_bytes;
  __device__ __forceinline__ static int in_row(int lane, int i) {  // the lane's byte of its row of the step
    const int at = (i * 1024 + lane * 16) % (CPR * 64);
    return (at & ~63) + (((at >> 4) ^ (at >> 6)) & 3) * 16;
  }
  __device__ __forceinline__ void init(const void* x, int64_t ld, int n, int K, int lane) {
    row_bytes = K * 2;
    rows = make_rsrc(x, (n - 1) * ld * 2 + row_bytes);
#pragma unroll
    for (int i = 0; i < kInst; ++i) {
      const int r = (i * 1024 + lane * 16) / (CPR * 64);
      voff[i] = r < n ? static_cast<uint32_t>(r * ld * 2 + in_row(lane, i)) : kOOB;
    }
  }
  __device__ __forceinline__ void issue(uint32_t dst, int b0, int lane) const {
#pragma unroll
    for (int i = 0; i < kInst; ++i)
      dma16(rows, dst + i * 1024,
            voff[i] != kOOB && b0 * 64 + in_row(lane, i) < row_bytes ? voff[i] + static_cast<uint32_t>(b0) * 64 : kOOB);
  }
  // block c of row r
  __device__ __forceinline__ static void block(const char* t, int r, int c, u32x4 (&x)[4]) {
#pragma unroll
    for (int p = 0; p < 4; ++p) x[p] = *reinterpret_cast<const u32x4*>(t + (r * CPR + c) * 64 + (p ^ (c & 3)) * 16);
  }
};

// Steps in the ring: what fits into a CU's LDS.  X: A is raw, and a wave keeps the
// codes and scales of one step.
template <typename X, int J, int MR>
struct Ring {
  static constexpr bool kRaw = !std::is_same<X, void>::value;
  static constexpr int CPR = J == 1 ? 16 : 8;  // blocks of a row per step
  using LC = Loader<MR, CPR, false>;
  using LA = std::conditional_t<kRaw, RawLoader<MR, CPR>, LC>;
  using LB = Loader<16 * J, CPR, true>;
  static constexpr int kStepB = LB::kBytes + LB::kScaleBytes;
  static constexpr int kStep = kStepB + LA::kBytes + LA::kScaleBytes;
  static constexpr int kOwn = kRaw ? LC::kBytes + LC::kScaleBytes : 0;
  static constexpr int S = (163840 / 2 / kWaves - kOwn) / kStep;  // two blocks a CU
  static constexpr int kLds = kWaves * (S * kStep + kOwn);
  static_assert(S >= 1 && S <= 3 && kLds >= kWaves * J * (MR > 16 ? MR / 16 : 1) * 1024, "a step, and the sums to merge");
};

template <typename T, typename X, int J, int MR>
__global__ __launch_bounds__(64 * kWaves, 2) void k_mx4_skinny(Mx4Args g, int whole) {
  using R = Ring<X, J, MR>;
  using LA = typename R::LA;
  using LC = typename R::LC;
  using LB = typename R::LB;
  constexpr int CPR = R::CPR, S = R::S, kStep = R::kStep, kStepB = R::kStepB;
  constexpr int NB = CPR / 4;  // instructions of a step: block 4 u + q in lane group q
  constexpr int kInst = LA::kInst + LA::kScaleInst + LB::kInst + LB::kScaleInst;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * (16 * J);
  const int nv = min(16 * J, g.N - n0);
  const int i16 = lane & 15, q = lane >> 4;

  LA la;
  LB lb;
  if constexpr (R::kRaw)
    la.init(g.x, g.ldx, g.M, g.K, lane);
  else
    la.init(g.a, g.lda, g.as, g.ldas, g.M, g.kb, lane);
  lb.init(g.b + n0 * g.ldb, g.ldb, g.bs + n0 * g.ldbs, g.ldbs, nv, g.kb, lane);
  const int steps = (g.kb + CPR - 1) / CPR;
  const int n = steps > wave ? (steps - wave + kWaves - 1) / kWaves : 0;  // this wave's: wave, wave + kWaves, ..
  char* mine = smem + wave * (S * kStep + R::kOwn);
  char* own = mine + S * kStep;  // X: the step's codes and scales
  const uint32_t mine_addr = lds_addr(mine);
  int slot_in = 0;
  // step j of this wave into ring slot j % S
  auto issue = [&](int j) {
    if (j >= n) return;
    const int b0 = (wave + j * kWaves) * CPR;
    const uint32_t dst = mine_addr + slot_in * kStep;
    lb.issue(dst, b0, lane);
    la.issue(dst + kStepB, b0, lane);
    slot_in = slot_in + 1 == S ? 0 : slot_in + 1;
  };
  // this lane's first scale byte in a step's dwords: of its rows of A, of its columns
  constexpr int RB = MR > 16 ? MR / 16 : 1;
  int ar[RB], sat[RB];
#pragma unroll
  for (int x = 0; x < RB; ++x) {
    ar[x] = 16 * x + (i16 & (MR - 1));
    sat[x] = LC::kBytes + ar[x] * (LC::ND * 4) + q +
             (R::kRaw ? 0 : static_cast<int>((reinterpret_cast<uintptr_t>(g.as) + ar[x] * g.ldas) & 3u));
  }
  int sbt[J];
#pragma unroll
  for (int j = 0; j < J; ++j)
    sbt[j] = LB::kBytes + (j * 16 + i16) * (LB::ND * 4) +
             static_cast<int>((reinterpret_cast<uintptr_t>(g.bs) + (n0 + j * 16 + i16) * g.ldbs) & 3u) + q;
  f32x4 acc[RB][J];
#pragma unroll
  for (int x = 0; x < RB; ++x)
#pragma unroll
    for (int j = 0; j < J; ++j) acc[x][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < S; ++s) issue(s);
  int slot = 0;
  for (int i = 0; i < n; ++i) {
    __builtin_amdgcn_sched_barrier(0);
    // step i is in: all but the steps behind it, S - 1 until the last ones
    const int behind = n - 1 - i;
    if (behind >= S - 1)
      wait_vmcnt<(S - 1) * kInst>();
    else if (S > 2 && behind == 1)
      wait_vmcnt<kInst>();
    else
      wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    const char* tb = mine + slot * kStep;
    const char* ta = tb + kStepB;
    if constexpr (R::kRaw) {
      // (the step's blocks by lanes; rows that all lie past M are left as they are:
      // what they give is never stored)
#pragma unroll
      for (int id0 = 0; id0 < MR * CPR; id0 += 64) {
        const int id = id0 + lane, r = id / CPR, c = id - r * CPR;
        if (id0 / CPR < g.M && id < MR * CPR) {
          u32x4 x[4];
          LA::block(ta, r, c, x);
          uint32_t s;
          const u32x4 codes = quantize32<X>(x, s);
          *reinterpret_cast<u32x4*>(own + r * (CPR * 16) + sk_slot<CPR>(r, c) * 16) = codes;
          *reinterpret_cast<uint8_t*>(own + LC::kBytes + r * (LC::ND * 4) + c) = static_cast<uint8_t>(s);
        }
      }
      asm volatile("" ::: "memory");  // a wave's LDS operations run in order: written, then read by other lanes
      ta = own;
    }
    const int left = g.kb - (wave + i * kWaves) * CPR;  // blocks of the row from the step's first on
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      const int c = 4 * u + q;
      u32x4 a[RB];
      uint32_t sa[RB];
#pragma unroll
      for (int x = 0; x < RB; ++x) {
        a[x] = *reinterpret_cast<const u32x4*>(ta + ar[x] * (CPR * 16) + sk_slot<CPR>(ar[x], c) * 16);
        sa[x] = *reinterpret_cast<const uint8_t*>(ta + sat[x] + 4 * u);
        if (left < CPR) sa[x] = c < left ? sa[x] : 0;
      }
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int r = j * 16 + i16;
        const u32x4 b = *reinterpret_cast<const u32x4*>(tb + r * (CPR * 16) + sk_slot<CPR>(r, c) * 16);
        uint32_t sb = *reinterpret_cast<const uint8_t*>(tb + sbt[j] + 4 * u);
        if (left < CPR) sb = c < left ? sb : 0;
#pragma unroll
        for (int x = 0; x < RB; ++x) acc[x][j] = mfma_mx4<0, 0>(b, sb, a[x], sa[x], acc[x][j]);
      }
    }
    wait_lgkmcnt0();
    issue(i + S);
    slot = slot + 1 == S ? 0 : slot + 1;
  }
  wait_vmcnt<0>();  // no DMA may land in the LDS the merge reuses
  __syncthreads();
  // lane l holds rows 16 x + l & 15, columns 16 j + 4 (l >> 4) .. + 3
  f32x4* red = reinterpret_cast<f32x4*>(smem);  // [wave][x][j][lane]
#pragma unroll
  for (int x = 0; x < RB; ++x)
#pragma unroll
    for (int j = 0; j < J; ++j) red[((wave * RB + x) * J + j) * 64 + lane] = acc[x][j];
  __syncthreads();
  for (int i = wave; i < RB * J; i += kWaves) {
    f32x4 v = red[i * 64 + lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
      const f32x4 y = red[(w * (RB * J) + i) * 64 + lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += y[e];
    }
    store4<T>(static_cast<T*>(g.d), g.ldd, i / J * 16 + i16, n0 + i % J * 16 + 4 * q, g.M, g.N, v, static_cast<const T*>(g.bias), whole != 0);
  }
}

template <typename T, typename X, int J, int MR>
int launch_skinny(const Mx4Args& g, hipStream_t st) {
  constexpr int kLds = Ring<X, J, MR>::kLds;
  auto kern = k_mx4_skinny<T, X, J, MR>;
  static std::atomic<uint64_t> reserved{0};
  if (const int rc = reserve_lds(reinterpret_cast<const void*>(kern), kLds, reserved, "mxfp4_mm"); rc != NTOPS_OK) return rc;
  const int whole = (g.ldd & 3) == 0 && (reinterpret_cast<uintptr_t>(g.d) & (4 * sizeof(T) - 1)) == 0;
  note_kernel("mxfp4_skinny j%d m%d%s", J, MR, Ring<X, J, MR>::kRaw ? " fused" : "");
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>((g.N + 16 * J - 1) / (16 * J))), dim3(64 * kWaves), kLds, st, g, whole);
  return check_launch("mxfp4_mm");
}

template <typename T, typename X, int MR>
int run_skinny(const Mx4Args& g, int j, hipStream_t st) {
  if constexpr (MR <= 16)
    if (j == 4) return launch_skinny<T, X, 4, MR>(g, st);
  return j == 2 ? launch_skinny<T, X, 2, MR>(g, st) : launch_skinny<T, X, 1, MR>(g, st);
}

// Columns of a block, in 16s.  A CU's blocks, counted in halves as two run at once
// and one alone has the CU's bandwidth, cost their bytes and their starts, as much
// as 20 KiB of B each.  A ring of one step (lone) needs the CU's other block to
// cover its waits; two columns give the same sums as four.  From 17 rows on only two
// have a ring of more than one step, and are taken wherever a CU would get a second
// block of one.  Measured with 1, 2 and 4 in one graph over weights from memory (us):
//                    1 row, rounded here  1 row             16 rows           32 rows
//   4096 x 4096       5.2,  6.0,  9.5      4.4,  4.8,  6.6   4.8,  5.4,  8.4   5.9,  6.3,  9.5
//   4096 x 14336      9.0, 12.3, 22.7      7.6,  9.6, 17.3   9.2, 12.7, 22.5  12.5, 16.0, 26.6
//   6144 x 4096       6.3,  6.2,  9.7      5.3,  5.0,  6.9   6.1,  5.7,  8.6   7.8,  6.7,  9.8
//   14336 x 4096     10.4,  9.3, 11.3      8.9,  7.8,  8.3  10.3,  9.0,  9.9  13.3, 10.8, 11.1
//   14336 x 14336    24.0, 22.7, 27.0     21.4, 21.3, 22.7  26.6, 26.4, 26.7  36.5, 32.3, 30.8
//   24000 x 2048     10.3,  8.8,  8.7      9.2,  7.9,  7.7   9.8,  8.2,  8.7  11.8,  9.5,  9.9
//   28672 x 4096     16.9, 15.3, 14.6     14.9, 13.4, 13.1  17.6, 15.4, 15.4  23.4, 18.2, 17.5
//   100000 x 4096    54.0, 42.3, 40.9     46.0, 37.1, 37.5  55.2, 43.8, 46.5  70.7, 53.1, 52.9
// Starts of 44 KiB would take two columns in the third and fifth row, and four at
// 18944 x 3584, which lose up to 14 % there; without four from 5 rows on 49152 x 1536
// of 16 rows took 11.9 instead of 10.3.
int columns(int64_t M, int64_t N, int64_t kb, bool lone) {
  int best = 1;
  int64_t least = 0;
  const int64_t cus = cu_count_cached();
  if (M > 16) return ceil_div(N, 16) <= cus ? 1 : 2;
  for (int j = 1; j <= 4; j *= 2) {
    const int64_t halves = std::max<int64_t>(2, ceil_div(2 * ceil_div(N, 16 * j), cus));
    const int64_t cost = halves * (20 * 1024 + 16 * j * kb * 17);
    if (j == 1 || cost <= least) {
      least = cost;
      best = j;
    }
  }
  return best == 4 && lone && ceil_div(N, 64) <= cus ? 2 : best;
}

}  // namespace

int mx4_skinny(int out_dtype, const Mx4Args& g, hipStream_t st) {
  const int j = columns(g.M, g.N, g.kb, g.M > 4);
  return dispatch_float16_32(out_dtype, "mxfp4_mm", [&](auto tag) {
    using T = decltype(tag);
    return g.M <= 4 ? run_skinny<T, void, 4>(g, j, st) : g.M <= 16 ? run_skinny<T, void, 16>(g, j, st) : run_skinny<T, void, 32>(g, j, st);
  });
}

int mx4_skinny_fused(int x_dtype, int out_dtype, const Mx4Args& g, hipStream_t st) {
  const int j = columns(g.M, g.N, g.kb, true);
  return dispatch_float16_32(out_dtype, "mxfp4_mm", [&](auto tag) {
    using T = decltype(tag);
    return x_dtype == NTOPS_BF16 ? run_skinny<T, __bf16, kFusedRows>(g, j, st) : run_skinny<T, _Float16, kFusedRows>(g, j, st);
  });
}

}  // namespace ntops
