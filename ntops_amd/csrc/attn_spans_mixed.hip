// Shared-prefix attention of many sequences with few rows each (decoding a batch behind
// one prompt): blocks of attn_spans_tile.h take the rows of all sequences of a group over
// their prefix, blocks of attn_spans_few.h each sequence's rows over its own keys, in one
// launch, so that the first, bound by the matrix cores and vector instructions, run beside
// the second, bound by streaming.  bf16, 32 / 8 heads of 128, 64 sequences of one token
// over a shared 8192 and up to 1024 of their own: 50 us, of which 4.5 the merge (168 MB of
// own keys and 34 of the prefix: 41 at 4.95 TB/s), 53 with the prefix by blocks of few rows,
// 63 by a launch of its own; 16 sequences 25 against 36.
#include "attn_spans_few.h"
#include "attn_spans_tile.h"

namespace ntops {
namespace {

constexpr int kFewWaves = 2;

// D, DT: columns of a row in the LDS, of few rows and of tiles; RGM: groups of 16 rows of a
// sequence.  A block of few rows has two waves.  Its others end at once, by a scalar branch
// that no mask of lanes can turn into code they walk through: every wave that is left
// meets the block's barriers.  (As a condition on the lanes 2 to 3 % less time.)
template <typename T, int D, int DT, int RGM>
__global__ __launch_bounds__(64 * span_tile::kWaves, 2) void k_span_mixed(SpanArgs a, int nqb, int slices, uint32_t front, span_few::FewBlocks main, SpanPart part) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int64_t all = block_id();
  if (all >= static_cast<int64_t>(front) + main.blocks) return;  // the tail of a 2-D grid (the whole block)
  const uint32_t id = static_cast<uint32_t>(all);
  if (id >= front && __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) >= kFewWaves) return;
  if (id < front) {
    part.first = 0;
    span_tile::tile_block<T, DT, DT>(a, kFront, nqb, slices, front, part, id, smem);
    return;
  }
  span_few::few_block<T, D, kFewWaves, RGM>(a, main, part, id - front, smem);
}

template <typename T, int D, int DT, int RGM>
int launch_mixed(const SpanArgs& a, int front_slices, const span_few::FewBlocks& main, const SpanPart& part, hipStream_t st) {
  constexpr int kLds = span_tile::kTileLds<DT> > kFewWaves * 32768 ? span_tile::kTileLds<DT> : kFewWaves * 32768;
  static_assert(kLds <= 65536, "LDS");
  const int64_t nqb = ceil_div(span_rows(a, kFront), kTileRows);
  const int64_t front = span_sets(a, kFront) * nqb * front_slices;
  note_kernel("%s mixed d%d rows%d split%d+%d", a.pk ? "shared_prefix" : "sliding_window", DT, 16 * RGM, front_slices, main.slices);
  hipLaunchKernelGGL((k_span_mixed<T, D, DT, RGM>), blocks_2d(front + main.blocks), dim3(64 * span_tile::kWaves), kLds, st, a, static_cast<int>(nqb),
                     front_slices, static_cast<uint32_t>(front), main, part);
  return check_launch("attention");
}

template <typename T, int D, int DT>
int launch_mixed(const SpanArgs& a, const FewPlan& p, const SpanPart& part, hipStream_t st) {
  const span_few::FewBlocks main = span_few::few_blocks(a, p.mode, p.slices, part.first);
  return span_rows(a, kMain) > 16 ? launch_mixed<T, D, DT, 2>(a, p.front_slices, main, part, st) : launch_mixed<T, D, DT, 1>(a, p.front_slices, main, part, st);
}

template <typename T>
int run_mixed(const SpanArgs& a, const FewPlan& p, const SpanPart& part, hipStream_t st) {
  if (a.D <= 64) return launch_mixed<T, 64, 64>(a, p, part, st);
  if (a.D <= 96) return launch_mixed<T, 128, 96>(a, p, part, st);
  return launch_mixed<T, 128, 128>(a, p, part, st);
}

}  // namespace

int span_mixed_run(int dtype, const SpanArgs& a, const FewPlan& p, const SpanPart& part, hipStream_t st) {
  return dtype == NTOPS_BF16 ? run_mixed<__bf16>(a, p, part, st) : run_mixed<_Float16>(a, p, part, st);
}

}  // namespace ntops
