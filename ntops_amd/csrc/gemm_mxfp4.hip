// The MXFP4 product's tile kernel, its split over K, and the C entry points.
//
// 128 x 128 output tiles, four waves of 64 x 64, K tiles of 256 values (128
// bytes a row, whole lines) through a ring of four stages filled by direct DMA
// three tiles ahead; one barrier per K tile.  A stage is 32 KiB of codes and 2
// KiB of scales.
#include <algorithm>
#include <atomic>

#include "gemm_mxfp4.h"

namespace ntops {
namespace {

constexpr int kTile = 128;                  // rows and columns of an output tile
constexpr int kStages = 4;
constexpr int kCodes = 2 * kTile * 128;     // A's rows, then B's
constexpr int kScales = 2 * kTile * 8;
constexpr int kStage = kCodes + kScales;
constexpr int kLds = kStages * kStage;
constexpr int kLoads = 8 + 2;               // DMA instructions per wave and stage

// out rows m0 .. of one lane's 4 consecutive columns n .. n + 3.
template <typename T>
__device__ __forceinline__ void store4(T* d, int64_t ldd, int m, int n, int M, int N, f32x4 v, const T* bias, bool whole) {
  if (m >= M) return;
  T* at = d + static_cast<int64_t>(m) * ldd + n;
  T o[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float b = bias != nullptr && n + e < N ? static_cast<float>(bias[n + e]) : 0.f;
    o[e] = static_cast<T>(v[e] + b);
  }
  if (whole && n + 4 <= N) {
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<u32x2*>(at) = __builtin_bit_cast(u32x2, o);
    else
      *reinterpret_cast<u32x4*>(at) = __builtin_bit_cast(u32x4, o);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < N) at[e] = o[e];
  }
}

// whole: the output's rows are runs that 4 elements at a time can be stored to.
template <typename T>
__global__ __launch_bounds__(256, 1) void k_mx4_tile(Mx4Args g, int tm_count, int tn_count, int whole) {
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
  const int m0 = (band * 8 + in % rows_here) * kTile, n0 = in / rows_here * kTile;
  const int slice = blockIdx.y;
  const int kb0 = slice * g.kchunk, kb1 = min(g.kb, kb0 + g.kchunk);
  const int nt = (kb1 - kb0 + 7) / 8;

  const int mv = min(kTile, g.M - m0), nv = min(kTile, g.N - n0);
  const u32x4 ra = mx4_rsrc(g.a + m0 * g.lda, (mv - 1) * g.lda + g.kb * 16);
  const u32x4 rb = mx4_rsrc(g.b + n0 * g.ldb, (nv - 1) * g.ldb + g.kb * 16);
  const int kb4 = (g.kb + 3) & ~3;  // (padded rows: zeros behind their blocks)
  const u32x4 rsa = mx4_rsrc(g.as + m0 * g.ldas, (mv - 1) * g.ldas + kb4);
  const u32x4 rsb = mx4_rsrc(g.bs + n0 * g.ldbs, (nv - 1) * g.ldbs + kb4);
  const uint32_t smem_addr = lds_addr(smem);

  // this wave's loads of K tile j: rows 32 wave .. + 31 of A and of B (8 rows
  // an instruction), their scales in one instruction each (row l / 2, dword l % 2)
  auto issue = [&](int j) {
    const uint32_t st = smem_addr + static_cast<uint32_t>((j & (kStages - 1)) * kStage);
    const int b0 = kb0 + j * 8;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int row = wave * 32 + u * 8 + (lane >> 3);
      const int blk = b0 + kslot<64>(row, lane & 7);
      const uint32_t dst = st + static_cast<uint32_t>((wave * 32 + u * 8) * 128);
      dma16(ra, dst, blk < kb1 && row < mv ? static_cast<uint32_t>(row * g.lda + blk * 16) : kOOB);
      dma16(rb, dst + kTile * 128, blk < kb1 && row < nv ? static_cast<uint32_t>(row * g.ldb + blk * 16) : kOOB);
    }
    const int row = wave * 32 + (lane >> 1), blk = b0 + (lane & 1) * 4;
    const uint32_t dst = st + kCodes + static_cast<uint32_t>(wave * 256);
    dma4(rsa, dst, blk < kb1 && row < mv ? static_cast<uint32_t>(row * g.ldas + blk) : kOOB);
    dma4(rsb, dst + kTile * 8, blk < kb1 && row < nv ? static_cast<uint32_t>(row * g.ldbs + blk) : kOOB);
  };

  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  issue(0);
  issue(1);
  issue(2);
  for (int j = 0; j < nt; ++j) {
    __builtin_amdgcn_sched_barrier(0);
    wait_vmcnt<2 * kLoads>();  // K tile j is in (past the last tile the loads are empty, but count)
    block_barrier();           // for every wave; and tile j - 1's stage is free
    asm volatile("" ::: "memory");
    issue(j + 3);
    const char* st = smem + (j & (kStages - 1)) * kStage;
    uint32_t sa[4], sb[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sa[i] = *reinterpret_cast<const uint16_t*>(st + kCodes + (wm * 64 + i * 16 + i16) * 8 + q * 2);
      sb[i] = *reinterpret_cast<const uint16_t*>(st + kCodes + (kTile + wn * 64 + i * 16 + i16) * 8 + q * 2);
    }
    const auto frag = [&](int area, int r, int ks) {
      return *reinterpret_cast<const u32x4*>(st + area * (kTile * 128) + r * 128 + kslot<64>(r, 2 * q + ks) * 16);
    };
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      u32x4 fa[4], fb[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        fa[i] = frag(0, wm * 64 + i * 16 + i16, ks);
        fb[i] = frag(1, wn * 64 + i * 16 + i16, ks);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          acc[i][k] = ks == 0 ? mfma_mx4<0, 0>(fb[k], sb[k], fa[i], sa[i], acc[i][k])
                              : mfma_mx4<1, 1>(fb[k], sb[k], fa[i], sa[i], acc[i][k]);
    }
    wait_lgkmcnt0();  // this stage's reads are over before the next barrier frees it
  }
  wait_vmcnt<0>();  // no DMA may land after the workgroup ends
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int m = m0 + wm * 64 + i * 16 + i16, n = n0 + wn * 64 + k * 16 + 4 * q;
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

// Scale rows copied to rows of `to_ld` bytes, a multiple of 16, zeros behind
// their `kb` bytes: blockIdx.y 0 the a rows, 1 the b rows.
__global__ __launch_bounds__(256) void k_mx4_pad_scales(Mx4Args g, uint8_t* a, uint8_t* b, int to_ld) {
  const bool second = blockIdx.y != 0;
  const int rows = second ? g.N : g.M;
  uint8_t* to = second ? b : a;
  if (to == nullptr) return;
  const uint8_t* from = second ? g.bs : g.as;
  const int64_t ld = second ? g.ldbs : g.ldas;
  const int words = to_ld / 4;
  const int64_t total = static_cast<int64_t>(rows) * words;
  for (int64_t i = blockIdx.x * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = i / words;
    const int c = static_cast<int>(i - row * words) * 4;
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < g.kb) w |= static_cast<uint32_t>(from[row * ld + c + e]) << (8 * e);
    *reinterpret_cast<uint32_t*>(to + row * to_ld + c) = w;
  }
}

int64_t round16(int64_t n) { return (n + 15) & ~int64_t(15); }

// Whether the kernels can read these scale rows as they are: whole groups of 8
// blocks (what follows a row's last block would count as a scale, and 255 is
// NaN), dwords aligned.
bool scales_fit(int64_t kb, const void* s, int64_t ld) {
  return kb % 8 == 0 && ld % 4 == 0 && (reinterpret_cast<uintptr_t>(s) & 3u) == 0;
}

// Slices of K: as many as bring the blocks near the number of CUs, none under
// four K tiles.
void split_k(int64_t M, int64_t N, int64_t kb, int& split, int& kchunk) {
  const int64_t tiles = ceil_div(M, kTile) * ceil_div(N, kTile);
  const int64_t kt = ceil_div(kb, 8);
  int64_t s = std::max<int64_t>(1, std::min<int64_t>({cu_count_cached() / tiles, kt / 4, 16}));
  const int64_t per = ceil_div(kt, s);
  kchunk = static_cast<int>(per * 8);
  split = static_cast<int>(ceil_div(kt, per));
}

template <typename T>
int run_tile(const Mx4Args& g, hipStream_t st) {
  auto kern = k_mx4_tile<T>;
  static std::atomic<bool> attr_set{false};  // (threads may get here together)
  if (!attr_set.load(std::memory_order_relaxed)) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, kLds) !=
        hipSuccess)
      return set_error(NTOPS_ERR_HIP, "mxfp4_mm: cannot reserve %d bytes of LDS", kLds);
    attr_set.store(true, std::memory_order_relaxed);
  }
  const int tm = static_cast<int>(ceil_div(g.M, kTile)), tn = static_cast<int>(ceil_div(g.N, kTile));
  const int whole = (g.ldd & 3) == 0 && (reinterpret_cast<uintptr_t>(g.d) & (4 * sizeof(T) - 1)) == 0;
  note_kernel("mxfp4_tile split%d", g.split);
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(tm * tn), static_cast<unsigned>(g.split)), dim3(256), kLds, st, g,
                     tm, tn, whole);
  if (g.split > 1)
    hipLaunchKernelGGL((k_mx4_reduce<T>), blocks_2d(ceil_div(static_cast<int64_t>(g.M) * g.N, 256)), dim3(256), 0, st, g);
  return check_launch("mxfp4_mm");
}

}  // namespace
}  // namespace ntops

using namespace ntops;

extern "C" int64_t ntops_mxfp4_mm_workspace(int64_t M, int64_t N, int64_t K, const void* a_scales, int64_t as_row_stride,
                                            const void* b_scales, int64_t bs_row_stride) {
  if (M <= 0 || N <= 0 || K <= 0 || M > 0x7fffffff || N > 0x7fffffff || K > 0x7fffffff) return 0;
  const int64_t kb = ceil_div(K, 32);
  int split, kchunk;
  split_k(M, N, kb, split, kchunk);
  int64_t bytes = split > 1 ? split * M * N * 4 : 0;
  bytes = round16(bytes);
  if (!scales_fit(kb, a_scales, as_row_stride)) bytes += M * round16(kb);
  if (!scales_fit(kb, b_scales, bs_row_stride)) bytes += N * round16(kb);
  return bytes;
}

extern "C" int ntops_mxfp4_mm(int out_dtype, int64_t M, int64_t N, int64_t K, const void* a, int64_t a_row_stride,
                              const void* a_scales, int64_t as_row_stride, const void* b, int64_t b_row_stride,
                              const void* b_scales, int64_t bs_row_stride, const void* bias, void* out,
                              int64_t out_row_stride, void* workspace, int64_t workspace_bytes, void* stream) {
  if (M < 0 || N < 0 || K < 0) return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: negative size");
  if (out_dtype != NTOPS_F32 && out_dtype != NTOPS_F16 && out_dtype != NTOPS_BF16)
    return set_error(NTOPS_ERR_UNSUPPORTED, "mxfp4_mm: unsupported output dtype %d (F32/F16/BF16 only)", out_dtype);
  if (M == 0 || N == 0) return NTOPS_OK;
  if (!out || (K > 0 && (!a || !a_scales || !b || !b_scales))) return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: null pointer");
  const int64_t kb = ceil_div(K, 32);
  if (K == 0) a_row_stride = b_row_stride = as_row_stride = bs_row_stride = 0;  // no rows to read
  if (K > 0 && (!aligned16(a) || !aligned16(b) || a_row_stride % 16 != 0 || b_row_stride % 16 != 0))
    return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: code rows not aligned to 16 bytes");
  if (a_row_stride < 0 || b_row_stride < 0 || as_row_stride < 0 || bs_row_stride < 0)
    return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: negative row stride");
  const int64_t lim = int64_t(1) << 30;
  const auto span = [&](int64_t ld, int64_t row) { return 256 * ld + row; };  // bytes that one tile's rows cover
  if (M > lim || N > lim || kb * 16 > lim || span(a_row_stride, kb * 16) > lim || span(b_row_stride, kb * 16) > lim ||
      span(as_row_stride, kb) > lim || span(bs_row_stride, kb) > lim ||
      ceil_div(M, kTile) * ceil_div(N, kTile) > 0x7fffff)
    return set_error(NTOPS_ERR_UNSUPPORTED, "mxfp4_mm: operands too large");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  Mx4Args g{};
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
  const bool pad_a = kb > 0 && !scales_fit(kb, a_scales, as_row_stride);
  const bool pad_b = kb > 0 && !scales_fit(kb, b_scales, bs_row_stride);
  split_k(M, N, std::max<int64_t>(kb, 1), g.split, g.kchunk);
  const int64_t part_bytes = g.split > 1 ? round16(g.split * M * N * 4) : 0;
  const int64_t ld = round16(kb);
  const int64_t pad_bytes = (pad_a ? M * ld : 0) + (pad_b ? N * ld : 0);
  if (workspace_bytes < 0 || (workspace != nullptr && !aligned16(workspace)))
    return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: workspace not aligned to 16 bytes");
  if (pad_bytes > 0 && (workspace == nullptr || workspace_bytes < pad_bytes))
    return set_error(NTOPS_ERR_INVALID, "mxfp4_mm: these scale rows need %lld bytes of workspace",
                     static_cast<long long>(pad_bytes));
  if (g.split > 1 && (workspace == nullptr || workspace_bytes < part_bytes + pad_bytes)) {
    g.split = 1;
    g.kchunk = std::max(8, g.kb);
  } else if (g.split > 1) {
    g.part = static_cast<float*>(workspace);
  }
  if (pad_bytes > 0) {
    uint8_t* at = static_cast<uint8_t*>(workspace) + (g.split > 1 ? part_bytes : 0);
    uint8_t* pa = pad_a ? at : nullptr;
    uint8_t* pb = pad_b ? at + (pad_a ? M * ld : 0) : nullptr;
    const int64_t words = std::max(pad_a ? M : 0, pad_b ? N : 0) * (ld / 4);
    const int64_t blocks = std::min<int64_t>(ceil_div(words, 256), 4096);
    hipLaunchKernelGGL(k_mx4_pad_scales, dim3(static_cast<unsigned>(blocks), 2), dim3(256), 0, st, g, pa, pb,
                       static_cast<int>(ld));
    if (pad_a) {
      g.as = pa;
      g.ldas = ld;
    }
    if (pad_b) {
      g.bs = pb;
      g.ldbs = ld;
    }
  }
  return dispatch_float16_32(out_dtype, "mxfp4_mm", [&](auto tag) { return run_tile<decltype(tag)>(g, st); });
}
