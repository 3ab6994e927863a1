// The MXFP4 product's tile kernel, its split over K, and the C entry points.
//
// BT x BT output tiles, four waves of BT / 2 x BT / 2, K tiles of 256 values (128
// bytes a row, whole lines) through a ring of four stages filled by direct DMA
// three tiles ahead; one barrier per K tile.
//
// Scales come as dwords.  Where a row's scales do not start on one, or K tiles
// end inside a dword (FIT false), a lane loads the three dwords that its row's 8
// bytes lie in and reads single bytes; bytes behind the row's last block, which
// may belong to another row and be 255 (NaN), become 0 there.  Such a dword may
// reach up to 3 bytes past the scales' end or before their start; being aligned
// it lies within what the memory's page holds.
#include <algorithm>
#include <atomic>

#include "gemm_mxfp4.h"

namespace ntops {
namespace {

constexpr int kStages = 4;

template <int BT, bool FIT>
struct TileShape {
  static constexpr int kRowsPerWave = BT / 4;                  // rows of an operand that a wave loads
  static constexpr int kCodes = BT * 128;                      // bytes of an operand's codes per stage
  static constexpr int kDwords = FIT ? 2 : 3;                  // of a row's scales
  static constexpr int kScaleInst = (kRowsPerWave * kDwords + 63) / 64;
  static constexpr int kScales = 4 * kScaleInst * 256;         // bytes of an operand's scales
  static constexpr int kStage = 2 * (kCodes + kScales);
  static constexpr int kLds = kStages * kStage;
  static constexpr int kLoads = 2 * (kRowsPerWave / 8 + kScaleInst);  // DMA instructions per wave and stage
};

// whole: the output's rows are runs that 4 elements at a time can be stored to.
template <typename T, int BT, bool FIT>
__global__ __launch_bounds__(256, BT == 64 ? 2 : 1) void k_mx4_tile(Mx4Args g, int tm_count, int tn_count, int whole) {
  using S = TileShape<BT, FIT>;
  constexpr int TW = BT / 32;  // 16-row (and column) pieces of a wave's tile
  constexpr int ND = S::kDwords;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int q = lane >> 4, i16 = lane & 15;
  // tiles by columns of up to 8 row tiles, so that neighbouring blocks share operands
  const int t = blockIdx.x;
  const int band = t / (8 * tn_count);
  const int rows_here = min(8, tm_count - band * 8);
  const int in = t - band * 8 * tn_count;
  const int m0 = (band * 8 + in % rows_here) * BT, n0 = in / rows_here * BT;
  const int slice = blockIdx.y;
  const int kb0 = slice * g.kchunk, kb1 = min(g.kb, kb0 + g.kchunk);
  const int nt = (kb1 - kb0 + 7) / 8;

  const int mv = min(BT, g.M - m0), nv = min(BT, g.N - n0);
  const u32x4 ra = make_rsrc(g.a + m0 * g.lda, (mv - 1) * g.lda + g.kb * 16);
  const u32x4 rb = make_rsrc(g.b + n0 * g.ldb, (nv - 1) * g.ldb + g.kb * 16);
  // scales from the dword on that holds the tile's first byte
  const uint8_t* sa0 = g.as + m0 * g.ldas;
  const uint8_t* sb0 = g.bs + n0 * g.ldbs;
  const int oa = FIT ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(sa0) & 3u);
  const int ob = FIT ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(sb0) & 3u);
  const u32x4 rsa = make_rsrc(sa0 - oa, (oa + (mv - 1) * g.ldas + g.kb + 3) & ~3ll);
  const u32x4 rsb = make_rsrc(sb0 - ob, (ob + (nv - 1) * g.ldbs + g.kb + 3) & ~3ll);
  const uint32_t smem_addr = lds_addr(smem);

  // this wave's loads of K tile j: BT / 4 rows of A and of B (8 rows an
  // instruction), and their scales (row l / ND, dword l % ND)
  auto issue = [&](int j) {
    const uint32_t st = smem_addr + static_cast<uint32_t>((j & (kStages - 1)) * S::kStage);
    const int b0 = kb0 + j * 8;
#pragma unroll
    for (int u = 0; u < S::kRowsPerWave / 8; ++u) {
      const int row = wave * S::kRowsPerWave + u * 8 + (lane >> 3);
      const int blk = b0 + kslot<64>(row, lane & 7);
      const uint32_t dst = st + static_cast<uint32_t>((wave * S::kRowsPerWave + u * 8) * 128);
      dma16(ra, dst, blk < kb1 && row < mv ? static_cast<uint32_t>(row * g.lda + blk * 16) : kOOB);
      dma16(rb, dst + S::kCodes, blk < kb1 && row < nv ? static_cast<uint32_t>(row * g.ldb + blk * 16) : kOOB);
    }
#pragma unroll
    for (int u = 0; u < S::kScaleInst; ++u) {
      const int id = u * 64 + lane;
      const int in_wave = id / ND, row = wave * S::kRowsPerWave + in_wave;
      const int blk = b0 + (id - in_wave * ND) * 4;
      const bool ok = in_wave < S::kRowsPerWave && b0 < kb1;
      const uint32_t dst = st + 2 * S::kCodes + static_cast<uint32_t>((wave * S::kScaleInst + u) * 256);
      // (past the row's last dword: the next row's, masked below; past the last row's: zeros)
      dma4(rsa, dst, ok && row < mv ? static_cast<uint32_t>(oa + row * g.ldas + blk) & ~3u : kOOB);
      dma4(rsb, dst + S::kScales, ok && row < nv ? static_cast<uint32_t>(ob + row * g.ldbs + blk) & ~3u : kOOB);
    }
  };
  // LDS offset of row r's scales of a K tile (not FIT: of the byte of block q)
  auto scale_at = [&](int r, int o, int64_t ld) {
    const int w = r / S::kRowsPerWave, in_wave = r - w * S::kRowsPerWave;
    return w * S::kScaleInst * 256 + in_wave * ND * 4 + (FIT ? 0 : static_cast<int>((o + r * ld) & 3) + q);
  };
  int sat[TW], sbt[TW];
#pragma unroll
  for (int i = 0; i < TW; ++i) {
    sat[i] = 2 * S::kCodes + scale_at(wm * (BT / 2) + i * 16 + i16, oa, g.ldas);
    sbt[i] = 2 * S::kCodes + S::kScales + scale_at(wn * (BT / 2) + i * 16 + i16, ob, g.ldbs);
  }

  f32x4 acc[TW][TW];
#pragma unroll
  for (int i = 0; i < TW; ++i)
#pragma unroll
    for (int j = 0; j < TW; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  issue(0);
  issue(1);
  issue(2);
  for (int j = 0; j < nt; ++j) {
    __builtin_amdgcn_sched_barrier(0);
    wait_vmcnt<2 * S::kLoads>();  // K tile j is in (past the last tile the loads are empty, but count)
    block_barrier();              // for every wave; and tile j - 1's stage is free
    asm volatile("" ::: "memory");
    issue(j + 3);
    const char* st = smem + (j & (kStages - 1)) * S::kStage;
    uint32_t sa[TW], sb[TW];
    // the scales of blocks q and q + 4 of each row, in bytes 0 and 1
    if constexpr (FIT) {
      const uint32_t sel = 0x0400u + q * 0x0101u;
      const auto two = [&](int at) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(st + at);
        return __builtin_amdgcn_perm(w.y, w.x, sel);
      };
#pragma unroll
      for (int i = 0; i < TW; ++i) {
        sa[i] = two(sat[i]);
        sb[i] = two(sbt[i]);
      }
    } else {
      const int left = kb1 - kb0 - j * 8 - q;  // blocks from this lane's first on
      const uint32_t mask = left > 4 ? 0xffffu : left > 0 ? 0xffu : 0u;
#pragma unroll
      for (int i = 0; i < TW; ++i) {
        const uint8_t* pa = reinterpret_cast<const uint8_t*>(st + sat[i]);
        const uint8_t* pb = reinterpret_cast<const uint8_t*>(st + sbt[i]);
        sa[i] = (pa[0] | static_cast<uint32_t>(pa[4]) << 8) & mask;
        sb[i] = (pb[0] | static_cast<uint32_t>(pb[4]) << 8) & mask;
      }
    }
    const auto frag = [&](int area, int r, int ks) {
      return *reinterpret_cast<const u32x4*>(st + area * S::kCodes + r * 128 + kslot<64>(r, 4 * ks + q) * 16);
    };
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      u32x4 fa[TW], fb[TW];
#pragma unroll
      for (int i = 0; i < TW; ++i) {
        fa[i] = frag(0, wm * (BT / 2) + i * 16 + i16, ks);
        fb[i] = frag(1, wn * (BT / 2) + i * 16 + i16, ks);
      }
#pragma unroll
      for (int i = 0; i < TW; ++i)
#pragma unroll
        for (int k = 0; k < TW; ++k)
          acc[i][k] = ks == 0 ? mfma_mx4<0, 0>(fb[k], sb[k], fa[i], sa[i], acc[i][k])
                              : mfma_mx4<1, 1>(fb[k], sb[k], fa[i], sa[i], acc[i][k]);
    }
    wait_lgkmcnt0();  // this stage's reads are over before the next barrier frees it
  }
  wait_vmcnt<0>();  // no DMA may land after the workgroup ends
#pragma unroll
  for (int i = 0; i < TW; ++i)
#pragma unroll
    for (int k = 0; k < TW; ++k) {
      const int m = m0 + wm * (BT / 2) + i * 16 + i16, n = n0 + wn * (BT / 2) + k * 16 + 4 * q;
      if (g.split > 1)
        store4<float>(g.part + static_cast<int64_t>(slice) * g.M * g.N, g.N, m, n, g.M, g.N, acc[i][k], nullptr, (g.N & 3) == 0);
      else
        store4<T>(static_cast<T*>(g.d), g.ldd, m, n, g.M, g.N, acc[i][k], static_cast<const T*>(g.bias), whole != 0);
    }
}

// The slices' partial products summed in their order, and the bias.
template <typename T>
__global__ __launch_bounds__(256) void k_mx4_reduce(Mx4Args g) {
  const int64_t i = block_id() * 256 + threadIdx.x;
  const int64_t mn = static_cast<int64_t>(g.M) * g.N;
  if (i >= mn) return;
  float v = 0.f;
  for (int s = 0; s < g.split; ++s) v += g.part[s * mn + i];
  const int64_t m = i / g.N, n = i - m * g.N;
  if (g.bias != nullptr) v += static_cast<float>(static_cast<const T*>(g.bias)[n]);
  static_cast<T*>(g.d)[m * g.ldd + n] = static_cast<T>(v);
}

constexpr int64_t kMaxSize = int64_t(1) << 30;   // bytes of a tile's rows, or of a row
constexpr int64_t kMaxCount = int64_t(1) << 29;  // rows

// Whether K tiles of 8 blocks are whole dwords of these scale rows.
bool scales_fit(int64_t kb, const void* s, int64_t ld) {
  return kb % 8 == 0 && ld % 4 == 0 && (reinterpret_cast<uintptr_t>(s) & 3u) == 0;
}

// 256 x 256 tiles for about a round of the GPU or more.
bool large_suits(int64_t M, int64_t N) { return ceil_div(M, 256) * ceil_div(N, 256) >= cu_count_cached() / 2; }

// The tile's size: 128 from a tile per CU on ((1024, 4096, 4096) bf16 25.2 us, on 64
// x 64 tiles 30.9; (512, 4096, 4096), 128 large tiles, 23.6 and 17.8).  Slices of K:
// as many as bring the blocks near the number of CUs (twice as many: (256, 4096,
// 4096) 11.2 -> 16.1), none under eight K tiles, whose time a reduction's launch
// takes ((500, 1001, 2080) in slices of four 12.3 us, whole 9.1; (64, 4096, 14336) in
// slices of eight or more 17.6, of sixteen or more 19.1).
void plan(int64_t M, int64_t N, int64_t kb, int& bt, int& split, int& kchunk) {
  const int64_t cus = cu_count_cached();
  const auto tiles = [&](int64_t t) { return ceil_div(M, t) * ceil_div(N, t); };
  bt = tiles(128) >= cus ? 128 : 64;
  const int64_t kt = ceil_div(kb, 8);
  int64_t s = std::max<int64_t>(1, std::min<int64_t>({cus / tiles(bt), kt / 8, 16}));
  const int64_t per = ceil_div(kt, s);
  kchunk = static_cast<int>(per * 8);
  split = static_cast<int>(ceil_div(kt, per));
}

template <typename T, int BT, bool FIT>
int launch_tile(const Mx4Args& g, hipStream_t st) {
  auto kern = k_mx4_tile<T, BT, FIT>;
  constexpr int kLds = TileShape<BT, FIT>::kLds;
  static std::atomic<uint64_t> reserved{0};
  if (const int rc = reserve_lds(reinterpret_cast<const void*>(kern), kLds, reserved, "mxfp4_mm"); rc != NTOPS_OK) return rc;
  const int tm = static_cast<int>(ceil_div(g.M, BT)), tn = static_cast<int>(ceil_div(g.N, BT));
  const int whole = (g.ldd & 3) == 0 && (reinterpret_cast<uintptr_t>(g.d) & (4 * sizeof(T) - 1)) == 0;
  note_kernel("mxfp4_tile%d split%d%s", BT, g.split, FIT ? "" : " bytes");
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(tm * tn), static_cast<unsigned>(g.split)), dim3(256), kLds, st, g,
                     tm, tn, whole);
  if (g.split > 1)
    hipLaunchKernelGGL((k_mx4_reduce<T>), blocks_2d(ceil_div(static_cast<int64_t>(g.M) * g.N, 256)), dim3(256), 0, st, g);
  return check_launch("mxfp4_mm");
}

template <typename T>
int run_tile(const Mx4Args& g, int bt, hipStream_t st) {
  const bool fit = scales_fit(g.kb, g.as, g.ldas) && scales_fit(g.kb, g.bs, g.ldbs);
  if (bt == 128) return fit ? launch_tile<T, 128, true>(g, st) : launch_tile<T, 128, false>(g, st);
  return fit ? launch_tile<T, 64, true>(g, st) : launch_tile<T, 64, false>(g, st);
}

}  // namespace
}  // namespace ntops

using namespace ntops;

extern "C" int64_t ntops_mxfp4_mm_workspace(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || M > kMaxCount || N > kMaxCount || K > kMaxSize) return 0;
  if (M <= kSkinnyRows) return 0;
  if (large_suits(M, N)) return mx4_large_workspace(M, N, ceil_div(K, 32));
  int bt, split, kchunk;
  plan(M, N, ceil_div(K, 32), bt, split, kchunk);
  return split > 1 ? split * M * N * 4 : 0;
}

namespace ntops {
namespace {

// The arguments of ntops_mxfp4_mm, checked (M, N > 0), in g.
int mx4_args(int out_dtype, int64_t M, int64_t N, int64_t K, const void* a, int64_t a_row_stride, const void* a_scales,
             int64_t as_row_stride, const void* b, int64_t b_row_stride, const void* b_scales, int64_t bs_row_stride,
             const void* bias, void* out, int64_t out_row_stride, const void* workspace, int64_t workspace_bytes, Mx4Args& g) {
  if (M < 0 || N < 0 || K < 0) return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: negative size");
  if (out_dtype != NTOPS_F32 && out_dtype != NTOPS_F16 && out_dtype != NTOPS_BF16)
    return set_error(NTOPS_ERR_UNSUPPORTED, "mxfp4_mm: unsupported output dtype %d (F32/F16/BF16 only)", out_dtype);
  if (!out || (K > 0 && (!a || !a_scales || !b || !b_scales))) return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: null pointer");
  const int64_t kb = ceil_div(K, 32);
  if (K == 0) a_row_stride = b_row_stride = as_row_stride = bs_row_stride = 0;  // no rows to read
  if (K > 0 && (!aligned16(a) || !aligned16(b) || a_row_stride % 16 != 0 || b_row_stride % 16 != 0))
    return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: code rows not aligned to 16 bytes");
  if (a_row_stride < 0 || b_row_stride < 0 || as_row_stride < 0 || bs_row_stride < 0)
    return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: negative row stride");
  const int64_t lim = kMaxSize;
  const auto span = [&](int64_t ld, int64_t row) { return 256 * ld + row; };  // bytes that one tile's rows cover
  if (M > kMaxCount || N > kMaxCount || kb * 16 > lim || span(a_row_stride, kb * 16) > lim || span(b_row_stride, kb * 16) > lim ||
      span(as_row_stride, kb) > lim || span(bs_row_stride, kb) > lim ||
      ceil_div(M, 64) * ceil_div(N, 64) > 0x7fffff)
    return set_error(NTOPS_ERR_UNSUPPORTED, "mxfp4_mm: operands too large");
  g.a = static_cast<const uint8_t*>(a);
  g.as = static_cast<const uint8_t*>(a_scales);
  g.b = static_cast<const uint8_t*>(b);
  g.bs = static_cast<const uint8_t*>(b_scales);
  g.bias = bias;
  g.d = out;
  g.lda = a_row_stride;
  g.ldas = as_row_stride;
  g.ldb = b_row_stride;
  g.ldbs = bs_row_stride;
  g.ldd = out_row_stride;
  g.M = static_cast<int>(M);
  g.N = static_cast<int>(N);
  g.kb = static_cast<int>(kb);
  if (workspace_bytes < 0 || (workspace != nullptr && !aligned16(workspace)))
    return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: workspace not aligned to 16 bytes");
  return NTOPS_OK;
}

}  // namespace
}  // namespace ntops

extern "C" int ntops_mxfp4_mm(int out_dtype, int64_t M, int64_t N, int64_t K, const void* a, int64_t a_row_stride,
                              const void* a_scales, int64_t as_row_stride, const void* b, int64_t b_row_stride,
                              const void* b_scales, int64_t bs_row_stride, const void* bias, void* out,
                              int64_t out_row_stride, void* workspace, int64_t workspace_bytes, void* stream) {
  if ((M == 0 || N == 0) && M >= 0 && N >= 0 && K >= 0 &&
      (out_dtype == NTOPS_F32 || out_dtype == NTOPS_F16 || out_dtype == NTOPS_BF16))
    return NTOPS_OK;
  Mx4Args g{};
  if (const int rc = mx4_args(out_dtype, M, N, K, a, a_row_stride, a_scales, as_row_stride, b, b_row_stride, b_scales, bs_row_stride,
                              bias, out, out_row_stride, workspace, workspace_bytes, g);
      rc != NTOPS_OK)
    return rc;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t kb = g.kb;
  return dispatch_float16_32(out_dtype, "mxfp4_mm", [&](auto tag) -> int {
    using T = decltype(tag);
    if (M <= kSkinnyRows && kb > 0) return mx4_skinny(out_dtype, g, st);
    if (large_suits(M, N) && mx4_large_serves(out_dtype, g) && workspace != nullptr &&
        workspace_bytes >= mx4_large_workspace(M, N, kb))
      return mx4_large(out_dtype, g, workspace, st);
    int bt;
    plan(M, N, std::max<int64_t>(kb, 1), bt, g.split, g.kchunk);
    if (g.split > 1 && (workspace == nullptr || workspace_bytes < g.split * M * N * 4)) {
      g.split = 1;
      g.kchunk = (g.kb + 7) / 8 * 8;
    }
    g.part = static_cast<float*>(workspace);
    return run_tile<T>(g, bt, st);
  });
}

namespace ntops {
namespace {

// Whether a product's blocks quantize these activations themselves.
bool fused(int x_dtype, int64_t M, int64_t K, const void* x, int64_t x_row_stride) {
  return (x_dtype == NTOPS_BF16 || x_dtype == NTOPS_F16) && M <= kFusedRows && K % 8 == 0 && aligned16(x) &&
         (M == 1 || (x_row_stride % 8 == 0 && x_row_stride >= 0 && x_row_stride < kMaxSize / (2 * kFusedRows) - K));
}

int64_t round16(int64_t n) { return (n + 15) & ~int64_t(15); }

}  // namespace
}  // namespace ntops

extern "C" int64_t ntops_mxfp4_linear_workspace(int x_dtype, int64_t M, int64_t N, int64_t K, const void* x,
                                                int64_t x_row_stride) {
  if (M <= 0 || N <= 0 || K <= 0 || M > kMaxCount || N > kMaxCount || K > kMaxSize || fused(x_dtype, M, K, x, x_row_stride)) return 0;
  const int64_t kb = ceil_div(K, 32);
  return round16(M * kb * 16) + round16(M * kb) + ntops_mxfp4_mm_workspace(M, N, K);
}

extern "C" int ntops_mxfp4_linear(int x_dtype, int out_dtype, int64_t M, int64_t N, int64_t K, const void* x,
                                  int64_t x_row_stride, const void* b, int64_t b_row_stride, const void* b_scales,
                                  int64_t bs_row_stride, const void* bias, void* out, int64_t out_row_stride, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  if (M < 0 || N < 0 || K < 0) return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: negative size");
  if (x_dtype != NTOPS_F32 && x_dtype != NTOPS_F16 && x_dtype != NTOPS_BF16)
    return set_error(NTOPS_ERR_UNSUPPORTED, "mxfp4_mm: unsupported input dtype %d (F32/F16/BF16 only)", x_dtype);
  if (M > kMaxCount || N > kMaxCount || K > kMaxSize) return set_error(NTOPS_ERR_UNSUPPORTED, "mxfp4_mm: operands too large");
  if (K > 0 && M > 0 && !x) return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: null pointer");
  const int64_t kb = ceil_div(K, 32);
  if (M == 0 || N == 0 || K == 0)
    return ntops_mxfp4_mm(out_dtype, M, N, 0, nullptr, 0, nullptr, 0, nullptr, 0, nullptr, 0, bias, out, out_row_stride, nullptr, 0, stream);
  // (all but x checked before a kernel starts; A stands in for the codes to come)
  Mx4Args g{};
  if (const int rc = mx4_args(out_dtype, M, N, K, b, kb * 16, b_scales, kb, b, b_row_stride, b_scales, bs_row_stride, bias, out,
                              out_row_stride, nullptr, 0, g);
      rc != NTOPS_OK)
    return rc;
  if (fused(x_dtype, M, K, x, x_row_stride)) {
    g.x = x;
    g.ldx = M == 1 ? 0 : x_row_stride;
    g.K = static_cast<int>(K);
    return mx4_skinny_fused(x_dtype, out_dtype, g, static_cast<hipStream_t>(stream));
  }
  const int64_t codes = round16(M * kb * 16), scales = round16(M * kb);
  if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < codes + scales)
    return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: needs %lld bytes of workspace, aligned to 16",
                     static_cast<long long>(codes + scales));
  uint8_t* at = static_cast<uint8_t*>(workspace);
  if (const int rc = ntops_quantize_mxfp4(x_dtype, M, K, x, x_row_stride, at, at + codes, stream); rc != NTOPS_OK) return rc;
  return ntops_mxfp4_mm(out_dtype, M, N, K, at, kb * 16, at + codes, kb, b, b_row_stride, b_scales, bs_row_stride, bias, out,
                        out_row_stride, at + codes + scales, workspace_bytes - codes - scales, stream);
}
