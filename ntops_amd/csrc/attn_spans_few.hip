// Windowed and shared-prefix attention of few rows (attn_spans_few.h): launches.
#include "attn_spans_few.h"

namespace ntops {
namespace {

using namespace span_few;

// RG: groups of 16 rows of a sequence; FRONT: blocks over shared prefixes (of up to 16
// rows) come first.
template <typename T, int D, int NW, bool FRONT, int RG>
__global__ __launch_bounds__(64 * NW, 2) void k_span_few(SpanArgs a, FewBlocks front, FewBlocks main, SpanPart part) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];  // [wave][2 stages][K, V]
  const int64_t all = block_id();
  if (all >= static_cast<int64_t>(front.blocks) + main.blocks) return;  // the tail of a 2-D grid (the whole block)
  const uint32_t id = static_cast<uint32_t>(all);
  if constexpr (FRONT) {
    if (id < front.blocks) {
      few_block<T, D, NW, 1>(a, front, part, id, smem);
      return;
    }
  }
  few_block<T, D, NW, RG>(a, main, part, id - front.blocks, smem);
}

template <typename T, int D, int NW, bool FRONT, int RG>
int launch_few(const SpanArgs& a, const FewPlan& p, const SpanPart& part, hipStream_t st) {
  constexpr int kLds = NW * 32768;
  const FewBlocks front = FRONT ? few_blocks(a, kFront, p.front_slices, 0) : FewBlocks{};
  const FewBlocks main = few_blocks(a, p.mode, p.slices, part.first);
  note_kernel("%s few d%d waves%d rows%d+%d split%d+%d", a.pk ? "shared_prefix" : "sliding_window", D, NW, FRONT ? 16 : 0, 16 * RG, front.slices,
              main.slices);
  hipLaunchKernelGGL((k_span_few<T, D, NW, FRONT, RG>), blocks_2d(static_cast<int64_t>(front.blocks) + main.blocks), dim3(64 * NW), kLds, st, a,
                     front, main, part);
  return check_launch("attention");
}

template <typename T, int D>
int run_few(const SpanArgs& a, const FewPlan& p, const SpanPart& part, hipStream_t st) {
  const bool more = span_rows(a, p.mode) > 16;
  if (p.front_slices > 0) return launch_few<T, D, 2, true, 1>(a, p, part, st);  // (a group has more rows than a sequence)
  if (p.waves == 1) return more ? launch_few<T, D, 1, false, 2>(a, p, part, st) : launch_few<T, D, 1, false, 1>(a, p, part, st);
  return more ? launch_few<T, D, 2, false, 2>(a, p, part, st) : launch_few<T, D, 2, false, 1>(a, p, part, st);
}

}  // namespace

int span_few_run(int dtype, const SpanArgs& a, const FewPlan& p, const SpanPart& part, hipStream_t st) {
  if (dtype == NTOPS_BF16) return a.D > 64 ? run_few<__bf16, 128>(a, p, part, st) : run_few<__bf16, 64>(a, p, part, st);
  return a.D > 64 ? run_few<_Float16, 128>(a, p, part, st) : run_few<_Float16, 64>(a, p, part, st);
}

}  // namespace ntops
