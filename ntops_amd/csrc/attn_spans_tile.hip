// Windowed and shared-prefix attention of many rows (attn_spans_tile.h): launches.
#include <atomic>

#include "attn_spans_tile.h"

namespace ntops {
namespace {

using namespace span_tile;

template <typename T, int D, int DM>
__global__ __launch_bounds__(64 * kWaves, D > 128 ? 1 : D > 96 ? 2 : 3) void k_span_tile(SpanArgs a, int mode, int nqb, int slices, uint32_t total, SpanPart part) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int64_t all = block_id();
  if (all >= total) return;  // the tail of a 2-D grid (the whole block)
  tile_block<T, D, DM>(a, mode, nqb, slices, total, part, static_cast<uint32_t>(all), smem);
}

template <typename T, int D, int DM>
int launch_tile(const SpanArgs& a, int mode, int slices, const SpanPart& part, hipStream_t st) {
  auto kern = k_span_tile<T, D, DM>;
  if constexpr (kTileLds<D> > 65536) {
    static std::atomic<uint64_t> done{0};
    if (int e = reserve_lds(reinterpret_cast<const void*>(kern), kTileLds<D>, done, "attention")) return e;
  }
  const int64_t nqb = ceil_div(span_rows(a, mode), kRowsBlock);
  const int64_t total = span_sets(a, mode) * nqb * slices;
  note_kernel("%s tile d%d mode%d split%d", a.pk ? "shared_prefix" : "sliding_window", DM, mode, slices);
  hipLaunchKernelGGL(kern, blocks_2d(total), dim3(64 * kWaves), kTileLds<D>, st, a, mode, static_cast<int>(nqb), slices, static_cast<uint32_t>(total), part);
  return check_launch("attention");
}

template <typename T>
int run_tile(const SpanArgs& a, int mode, int slices, const SpanPart& part, hipStream_t st) {
  if (a.D <= 64) return launch_tile<T, 64, 64>(a, mode, slices, part, st);
  if (a.D <= 96) return launch_tile<T, 96, 96>(a, mode, slices, part, st);
  if (a.D <= 128) return launch_tile<T, 128, 128>(a, mode, slices, part, st);
  if (a.D <= 192) return launch_tile<T, 256, 192>(a, mode, slices, part, st);
  return launch_tile<T, 256, 256>(a, mode, slices, part, st);
}

}  // namespace

int span_tile_run(int dtype, const SpanArgs& a, int mode, int slices, const SpanPart& part, hipStream_t st) {
  return dtype == NTOPS_BF16 ? run_tile<__bf16>(a, mode, slices, part, st) : run_tile<_Float16>(a, mode, slices, part, st);
}

}  // namespace ntops
