// sliding_window_attention and shared_prefix_attention: the kernel for any head
// dim and layout, the merge of partial results, and the C entry points.
//
//   O = softmax(scale Q K^T) V over the keys that a row sees.  Row t of a sequence
//   of n tokens is its token p = n - Sq + t.
//     window: keys j <= p with j > p - window or j < sinks
//     prefix: every key of the prefix, and its own sequence's keys j <= p
//   A row that sees no key is 0.
#include <algorithm>

#include "attn_spans.h"

namespace ntops {
namespace {

constexpr int kMaxDim = 256;
constexpr int kMaxSlices = 64;
constexpr int64_t kMaxCount = 0x7fffffff;

// One wave per query row and slice of what it sees (front and main keys in equal
// parts of both).
template <typename T, int EL>
__global__ __launch_bounds__(256) void k_span_rows(SpanArgs a, int mode, int slices, SpanPart part, int64_t total) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t at = block_id() * 4 + wave;
  if (at >= total) return;
  const uint32_t id = static_cast<uint32_t>(at), rows = static_cast<uint32_t>(a.group * a.Sq * (mode == kFront ? a.per : 1));
  const uint32_t row = id / static_cast<uint32_t>(slices), set = row / rows;
  const int slice = static_cast<int>(id - row * slices), r = static_cast<int>(row - set * rows);
  const int t = static_cast<int>(static_cast<uint32_t>(r) / static_cast<uint32_t>(a.group) % static_cast<uint32_t>(a.Sq));
  const Spans s = make_spans<sizeof(T)>(a, mode, set, t, t);
  const SpanRow x = span_row(a, mode, s, r);
  const int fc = (s.n[0] + slices - 1) / slices, mc = (s.n[1] + slices - 1) / slices;
  const int f0 = min(slice * fc, s.n[0]), f1 = min(slice * fc + fc, s.n[0]), m0 = min(slice * mc, s.n[1]), m1 = min(slice * mc + mc, s.n[1]);
  float o[EL], m, l;
  span_attend_row<T, EL, (EL > 8 ? 2 : 4), false>(a, s, x, f0, f1, m0, m1, o, m, l);
  float any = 0.f;
#pragma unroll
  for (int u = 0; u < EL; ++u) any += o[u];
  if (__any(span_again(any, l)))
    span_row_again<T, EL>(a, s, part, x, slice, f0, f1, m0, m1);
  else
    span_write_row<T, EL, false>(a, part, x, slice, o, m, l);
}

// Combines the slices of every query row in slice order: one wave per row, W lanes
// a slice and 64 / W slices side by side, AHEAD times as many in flight.
template <typename T, int W, int AHEAD>
__global__ __launch_bounds__(256) void k_span_merge(SpanArgs a, SpanPart part) {
  const int lane = threadIdx.x & 63;
  const int64_t row = block_id() * 4 + (threadIdx.x >> 6);
  if (row >= static_cast<int64_t>(a.B) * a.Hq * a.Sq) return;
  constexpr int NS = 64 / W;
  const int d = (lane % W) * 4, g = lane / W;
  const auto load = [&](int s) {
    return s < part.slices && d < part.ld ? *reinterpret_cast<const f32x4*>(part.row(row * part.slices + s) + d) : f32x4{0.f, 0.f, 0.f, 0.f};
  };
  f32x4 v[AHEAD];  // in flight while the weights are formed
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) v[u] = load(u * NS + g);
  float m = neg_inf(), l = 0.f;
  if (lane < part.slices) {
    const float* ml = part.ml(a, row * part.slices + lane);
    m = ml[0];
    l = ml[1];
  }
  const float mm = wave_max(m);
  float w = m == neg_inf() ? 0.f : fast_exp2(m - mm);
  const float sum = wave_sum(l * w);
  // (divided first: sums of slices may pass fp32's range where the result does not)
  w *= sum == 0.f ? 0.f : 1.f / sum;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  const auto add = [&](int s, f32x4 x) {
    const float ws = __shfl(w, s & 63, 64);
    // (a slice of weight 0 holds nothing that the row has seen, or nothing beside the others)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += ws != 0.f ? ws * x[e] : 0.f;
  };
  for (int s0 = 0; s0 < part.slices; s0 += AHEAD * NS) {
    if (s0 > 0) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) v[u] = load(s0 + u * NS + g);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (s0 + u * NS < part.slices) add(s0 + u * NS + g, v[u]);
  }
#pragma unroll
  for (int step = W; step < 64; step <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], step, 64);
  if (g != 0) return;
  const uint32_t id = static_cast<uint32_t>(row), bh = id / static_cast<uint32_t>(a.Sq), b = bh / static_cast<uint32_t>(a.Hq);
  T* O = static_cast<T*>(a.o) + b * a.ost[0] + (bh - b * a.Hq) * a.ost[1] + (id - bh * a.Sq) * a.ost[2];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (d + e < a.D) O[(d + e) * a.ost[3]] = mean_as<T>(o[e]);
}

template <typename T, int W>
int launch_merge(const SpanArgs& a, const SpanPart& part, hipStream_t st) {
  const dim3 grid = blocks_2d(ceil_div(static_cast<int64_t>(a.B) * a.Hq * a.Sq, 4)), block(256);
  // (33 slices of 128 columns, 8 or 4 times 2 in flight: (1, 32 / 8, 1 over 32768) 29.5 / 31.5 us)
  if (part.slices > 4 * (64 / W))
    hipLaunchKernelGGL((k_span_merge<T, W, 8>), grid, block, 0, st, a, part);
  else
    hipLaunchKernelGGL((k_span_merge<T, W, 4>), grid, block, 0, st, a, part);
  return check_launch("attention");
}

int merge(int dtype, const SpanArgs& a, const SpanPart& part, hipStream_t st) {
  return dispatch_float16_32(dtype, "attention", [&](auto tag) {
    using T = decltype(tag);
    if (part.ld <= 64) return launch_merge<T, 16>(a, part, st);
    if (part.ld <= 128) return launch_merge<T, 32>(a, part, st);
    return launch_merge<T, 64>(a, part, st);
  });
}

template <typename T, int EL>
int launch_rows(const SpanArgs& a, int mode, int slices, const SpanPart& part, hipStream_t st) {
  const int64_t total = static_cast<int64_t>(a.B) * a.Hq * a.Sq * slices;
  hipLaunchKernelGGL((k_span_rows<T, EL>), blocks_2d(ceil_div(total, 4)), dim3(256), 0, st, a, mode, slices, part, total);
  return check_launch("attention");
}

// Most keys of the main span that a row sees.
int64_t main_keys(const SpanArgs& a) { return std::min<int64_t>(a.C, static_cast<int64_t>(a.window) + a.sinks); }

// How a problem is served.  With front_slices the rows of all sequences of a group go
// over their prefix together, in that many slices, and each sequence's rows over its own
// keys in `slices`; without, each sequence's rows go over both spans.
enum Path { kRows, kFew, kTile, kF32 };
struct Plan {
  Path front, main;  // (in one launch where the main one is kFew)
  int front_slices, slices;
  int waves;  // of a block of kFew
};

// Eight waves a CU, none of less than 32 keys: fp32 (1, 8, 1 over 200) of 128 11.6 us, of 128
// keys at least 26.8, (1, 8, 1 over 1000) 16.7 / 23.9, (1, 8, 1 over 2048) 19.8 / 23.3.
Plan rows_plan(const SpanArgs& a) {
  const int64_t rows = static_cast<int64_t>(a.B) * a.Hq * a.Sq;
  const int64_t n = std::min({static_cast<int64_t>(kMaxSlices), cu_count_cached() * 8 / rows, (a.P + main_keys(a)) / 32});
  return {kRows, kRows, 0, static_cast<int>(std::max<int64_t>(1, n)), 0};
}

// Blocks of `rows` rows.
int64_t row_blocks(const SpanArgs& a, int mode, int rows) { return span_sets(a, mode) * ceil_div(span_rows(a, mode), rows); }

// Slices of few rows for `heads` sets of them over `keys` keys, in tiles of `tile` keys a
// wave: a block a CU, none of less than two tiles a wave, past sixteen slices of four,
// below which the partial results and the merge cost what the slices gain.  bf16, 128
// columns, 4100 keys, 1 / 2 / 4 / 8 / 16 / 32 slices: 8 heads of 8 rows - / - / - / 17.0 / 16.0 /
// 16.3 us, 64 heads - / 33.4 / 29.7 / 33.9, 256 heads 91.2 / 98.6; two / four tiles a wave: 8
// heads over 1024 9.6 / 10.8, over 500 9.3 / 10.7, of 64 columns over 1024 9.1 / 10.8, one head
// over 8192 21.6 / 18.6.  fp32 (whose tiles are half as large) one / two tiles: 8 heads over
// 1024 12.1 / 13.0, over 4096 22.6 / 18.2; 64 heads over 4096, 4 / 8 / 16 slices 47.8 / 50.1 / 52.2.
int few_slices(int64_t heads, int64_t keys, int waves, int tile) {
  const int64_t step = static_cast<int64_t>(tile) * waves;
  const int64_t most = std::max(std::min<int64_t>(16, ceil_div(keys, 2 * step)), ceil_div(keys, 4 * step));
  int64_t n = std::min({static_cast<int64_t>(kMaxSlices), cu_count_cached() / heads, most});
  if (n <= 2 && keys <= 8 * step) n = 1;  // two short slices gain what the merge's launch costs
  return static_cast<int>(std::max<int64_t>(n, 1));
}

// fp32: few rows as few_slices has them; blocks of kF32Rows rows, two a CU, in slices of no
// less than two tiles (one / two / four: (1, 12 / 4, 30 over 200) of 96 13.3 / 16.6 / 23.6 us, (2, 12
// / 4, 100 over 600) of 96 27.2 / 24.0 / 29.2, (4, 12 / 4, 30 over 1200) of 64 26.3 / 24.0 / 22.2).
Plan f32_plan(const SpanArgs& a, bool joined) {
  const int64_t blocks = 2 * cu_count_cached();
  const auto slices = [&](int64_t items, int64_t keys, int most) {
    const int64_t n = std::min({static_cast<int64_t>(most), blocks / items, ceil_div(keys, 64)});
    return static_cast<int>(std::max<int64_t>(n, 1));
  };
  const int64_t main = row_blocks(a, kMain, kF32Rows);
  const bool few = a.D <= 128 && span_rows(a, kMain) <= kF32FewRows;
  if (!joined && a.P > 0 && a.B > a.G) {
    const int64_t front = row_blocks(a, kFront, kF32Rows);
    // few rows: by the bytes read again, as in read_again below: (4, 32 / 8, 1 over 2048) of 128
    // (50 MB) joined / apart 21.0 / 25.9 us, 16 over 1024 (126 MB) 31.7 / 35.3, 4 over 8192 (201
    // MB) 44.7 / 35.0, 4 over 32768 137 / 62, 64 over 2048 144 / 82
    const double again = static_cast<double>(a.B - a.G) * a.Hkv * a.P * a.D * 8;
    if (few ? again > (128 << 20) : main * a.P > front * a.P + (front * a.P + main * a.C) / 4)
      return {kF32, kF32, slices(front, a.P, kMaxSlices / 2), slices(main, a.C, kMaxSlices / 2), 0};
  }
  if (few) return {kF32, kF32, 0, few_slices(main, a.P + std::min<int64_t>(a.C, main_keys(a) + a.Sq), 4, 8), 0};
  // (a row alone at its cache head needs no keys kept for others: (8, 8, 1 over 8192) of 256
  // by kF32 381 us, by kRows 212; (64, 8, 1 over 1000) 381 / 201)
  if (span_rows(a, kMain) == 1) return rows_plan(a);
  return {kF32, kF32, 0, slices(main, a.P + std::min<int64_t>(a.C, main_keys(a) + a.Sq), kMaxSlices), 0};
}

// Slices of kTile for `items` blocks of rows over `keys` keys: a block a CU, two of 64
// columns, of up to 128 where each still has 2048 keys (two run side by side, but the
// partial results cost), or where `uneven` rows, those of a prompt from its start, leave
// CUs without work; none under two tiles.  4100 keys of 128 columns, 1 / 2 / 4 / 8 / 16 / 32 slices: 8 blocks of
// 64 rows 95 / 57 / 37 / 24.8 / 21.5 / 21.1 us, 64 blocks - / 56.6 / 39.5 / 41.3, 256 blocks 110.6
// / 113.3; 1100 keys, 256 blocks of 128 rows 36.1 / 46.7; 8700 keys 172 / 148; 8192 keys, 128
// blocks - / 92.9 / 83.7; uneven: 4096 keys, 256 blocks 82 / 67, 2048 keys, 128 blocks - / 37.5 /
// 33.3; 2100 keys of 64 columns, 128 blocks - / 30.1 / 26.2 / 32.5.
int tile_slices(const SpanArgs& a, int64_t items, int64_t keys, int most) {
  const int64_t cus = cu_count_cached();
  const bool uneven = span_rows(a, kMain) > kTileRows && main_keys(a) > a.Sq / 2 && a.P + a.C <= 2 * static_cast<int64_t>(a.Sq);
  const int64_t two = 2 * cus / items;
  const int64_t n = a.D <= 64 || (a.D <= 128 && two > 1 && (uneven || keys / two >= 2048)) ? two : cus / items;
  return static_cast<int>(std::max<int64_t>(1, std::min({static_cast<int64_t>(most), n, ceil_div(keys, 128)})));
}

// Rows of a group up to which kFew takes the prefix, from more on kTile, both in one
// launch with the sequences' own keys: 4 over 32768 with 4 heads (16 rows) 38 / 41 us, 8 over
// 8192 (32 rows) 26.8 / 21.9, 16 over 8192 34.0 / 23.0, 64 over 8192 52.6 / 49.7.
constexpr int64_t kFewFrontRows = 16;
// Prefix keys and values that sequences may read again through the caches before the
// prefix is better attended by itself, and the two results joined.  bf16, 32 / 8 heads of
// 128, one token over a prefix and up to 512 of its own, each sequence over both / apart:
// by kFew 2 over 32768 (134 MB again) 33 / 41 us, 4 over 32768 (403 MB) 54 / 38; by kTile 4 over
// 8192 (101 MB) 21.0 / 21.6, 16 over 1024 (63 MB) 16.6 / 19.2, 16 over 2048 (126 MB) 22.0 /
// 19.8, 64 over 512 (132 MB) 28.8 / 26.3, 8 over 8192 (235 MB) 32.6 / 21.9, 64 over 2048 (528
// MB) 50.8 / 31.5.
int64_t read_again(bool few_front) { return (few_front ? int64_t{140} : int64_t{110}) << 20; }

// The plan for this problem where layouts suit the matrix cores, from sizes alone.
// `joined`: both spans in one pass (without a workspace, they cannot be parted).
Plan make_plan(int dtype, const SpanArgs& a, bool joined = false) {
  if (a.D % (dtype == NTOPS_F32 ? 4 : 8) != 0 || static_cast<int64_t>(a.C) + a.P == 0) return rows_plan(a);
  if (dtype == NTOPS_F32) return f32_plan(a, joined);
  const int64_t heads = static_cast<int64_t>(a.B) * a.Hkv, cus = cu_count_cached();
  const bool few = a.D <= 128 && span_rows(a, kMain) <= kFewRows;
  const double again = static_cast<double>(a.B - a.G) * a.Hkv * a.P * a.D * 4;  // (no size overflows it)
  const int64_t blocks = row_blocks(a, kMain, few ? kFewRows : kTileRows);
  if (!joined && a.P > 0 && a.B > a.G) {
    const int64_t front = row_blocks(a, kFront, kTileRows);
    const bool few_front = few && span_rows(a, kFront) <= kFewFrontRows;
    // many rows: where the rows of a group fill blocks that those of a sequence leave empty
    const auto walked = [](int64_t n, int64_t keys) { return static_cast<double>(n) * static_cast<double>(keys); };
    const bool apart = again > read_again(few_front) &&
                       (few || walked(blocks, static_cast<int64_t>(a.P) + a.C) > 1.75 * (walked(front, a.P) + walked(blocks, a.C)));
    if (apart) {
      // A front block a CU; of kFew on three of four (4 sequences over 32768 with 8 heads, 16 /
      // 24 / 32 slices: 33.7 / 31.1 / 36.4 us, 2 over 100000 80 / 70 / 78; 32 over four of up to 5001
      // with 16 heads, 2 / 3 / 4 slices 28.6 / 27.5 / 28.4); of kTile beside blocks of few rows on
      // half, but of no more than 1024 keys, so that the others find room (64 sequences over
      // 8192 of their group and up to 1024 of their own, 4 / 8 / 12 / 16 slices: 58 / 50 / 55 / 58
      // us; 16 over 32768, 16 / 32: 56 / 46).
      const bool mixed = few && !few_front;
      const int64_t most = ceil_div(a.P, mixed ? 512 : 128);
      const int64_t wide = std::max<int64_t>(1, (mixed ? cus / 2 : few ? cus * 3 / 4 : cus) / front);
      const int64_t cut = std::max<int64_t>(mixed ? ceil_div(a.P, 1024) : 1, std::min(most, wide));
      const int fs = static_cast<int>(std::min<int64_t>(kMaxSlices / 2, cut));
      // own keys: slices no longer than twice the prefix's
      const int64_t ms = std::min({static_cast<int64_t>(kMaxSlices / 2), ceil_div(a.C, 2 * ceil_div(a.P, fs)), 2 * cus / blocks});
      return {few_front ? kFew : kTile, few ? kFew : kTile, fs, static_cast<int>(std::max<int64_t>(1, ms)), 2};
    }
  }
  const int64_t tokens = few ? 0 : std::min<int64_t>(a.Sq, ceil_div(kTileRows, a.Hq / a.Hkv));  // of a block past its first
  const int64_t keys = a.P + std::min<int64_t>(a.C, main_keys(a) + tokens);
  if (few) {
    const int waves = heads < 2 * cus ? 2 : 1;
    // (blocks of one wave are not split)
    return {kFew, kFew, 0, waves == 1 ? 1 : few_slices(heads, keys, waves, a.D > 64 ? 32 : 64), waves};
  }
  return {kTile, kTile, 0, tile_slices(a, blocks, keys, kMaxSlices), 0};
}

int64_t plan_bytes(const SpanArgs& a, const Plan& p) {
  const int n = p.front_slices + p.slices;
  if (n <= 1) return 0;
  return static_cast<int64_t>(a.B) * a.Hq * a.Sq * n * ((a.D + 3) / 4 * 4 + 2) * 4;
}
// The workspace of a call whose layouts are not known yet.
int64_t workspace_bytes(int dtype, const SpanArgs& a) { return std::max(plan_bytes(a, make_plan(dtype, a)), plan_bytes(a, rows_plan(a))); }

// What the matrix cores' kernels read: unit strides along the head dim, rows at
// multiples of 16 bytes that do not overlap, and for 16-bit types every offset within a
// span of a head below 2^31 bytes.
bool matrix_layout(const SpanArgs& a, int dtype) {
  const bool f32 = dtype == NTOPS_F32;
  const int pack = f32 ? 4 : 8;
  const auto rows16 = [&](const int64_t* s) { return s[3] == 1 && s[2] % pack == 0 && s[1] % pack == 0 && s[0] % pack == 0; };
  const auto span = [&](const int64_t* s, int64_t keys) { return f32 || (s[2] >= a.D && (keys + 256) * s[2] * 2 < 0x7fffffffLL); };
  if (!rows16(a.qst) || !aligned16(a.q) || a.ost[3] != 1 || a.ost[2] % 4 != 0 || a.ost[1] % 4 != 0 || a.ost[0] % 4 != 0 ||
      (reinterpret_cast<uintptr_t>(a.o) & (f32 ? 15u : 7u)) != 0)
    return false;
  const int64_t keys = std::min<int64_t>(a.C, static_cast<int64_t>(a.window) + a.Sq);
  if (a.C > 0 && (!rows16(a.kst) || !rows16(a.vst) || !aligned16(a.k) || !aligned16(a.v) || !span(a.kst, keys) || !span(a.vst, keys)))
    return false;
  if (a.C > 0 && a.sinks > 0) {
    const int64_t sinks = std::min<int64_t>(a.C, a.sinks);
    if (!span(a.kst, sinks) || !span(a.vst, sinks)) return false;
  }
  // (the kernel of few rows adds 32-bit offsets to a set's first query)
  const int64_t per = a.pk ? a.B / a.G : 1;
  if (!f32 && (a.qst[0] < 0 || a.qst[1] < 0 || a.qst[2] < 0)) return false;
  if (!f32 && (per - 1) * a.qst[0] + (a.Hq / a.Hkv - 1) * a.qst[1] + (a.Sq - 1) * a.qst[2] + a.D >= 0x3fffffffLL) return false;
  return a.P == 0 || (rows16(a.pkst) && rows16(a.pvst) && aligned16(a.pk) && aligned16(a.pv) && span(a.pkst, a.P) && span(a.pvst, a.P));
}

int run(int dtype, SpanArgs& a, void* ws, int64_t ws_bytes, hipStream_t st) {
  a.group = a.Hq / a.Hkv;
  a.per = a.B / a.G;
  if (ws == nullptr) ws_bytes = 0;
  // Strides that nothing is multiplied with do not decide on the kernel.
  const auto quiet = [](int64_t (&s)[4], int64_t n0, int64_t n1, int64_t n2) {
    if (n0 <= 1) s[0] = 0;
    if (n1 <= 1) s[1] = 0;
    if (n2 <= 1) s[2] = 0;
  };
  quiet(a.qst, a.B, a.Hq, a.Sq);
  quiet(a.ost, a.B, a.Hq, a.Sq);
  const int64_t row = (a.D + 7) / 8 * 8;
  for (auto* s : {&a.kst, &a.vst}) quiet(*s, a.B, a.Hkv, a.C);
  for (auto* s : {&a.pkst, &a.pvst}) quiet(*s, a.G, a.Hkv, a.P);
  if (a.C <= 1) a.kst[2] = a.vst[2] = row;
  if (a.P <= 1) a.pkst[2] = a.pvst[2] = row;
  if (a.C == 0) a.kst[3] = a.vst[3] = 1;
  if (a.P == 0) a.pkst[3] = a.pvst[3] = 1;
  Plan p = make_plan(dtype, a);
  if (plan_bytes(a, p) > ws_bytes) {
    p = make_plan(dtype, a, true);
    if (plan_bytes(a, p) > ws_bytes) p.slices = 1;
  }
  if (p.main != kRows && !matrix_layout(a, dtype)) {
    p = rows_plan(a);
    if (plan_bytes(a, p) > ws_bytes) p.slices = 1;
  }
  const int n = p.front_slices + p.slices;
  SpanPart part{n > 1 ? static_cast<float*>(ws) : nullptr, n, 0, (a.D + 3) / 4 * 4};
  const int mode = p.front_slices > 0 ? kMain : kBoth;
  if (p.front_slices > 0 && p.main != kFew)
    if (int e = p.front == kF32 ? span_f32_run(a, kFront, p.front_slices, part, st) : span_tile_run(dtype, a, kFront, p.front_slices, part, st))
      return e;
  part.first = p.front_slices;
  int e;
  if (p.main == kRows)
    e = span_rows_run(dtype, a, mode, p.slices, part, st);
  else if (p.main == kFew)
    e = (p.front == kFew ? span_few_run : span_mixed_run)(dtype, a, {p.waves, mode, p.front_slices, p.slices}, part, st);
  else if (p.main == kF32)
    e = span_f32_run(a, mode, p.slices, part, st);
  else
    e = span_tile_run(dtype, a, mode, p.slices, part, st);
  if (e) return e;
  return part.p ? merge(dtype, a, part, st) : NTOPS_OK;
}

bool sizes_fit(int64_t B, int64_t Hq, int64_t Sq, int64_t C, int64_t P) {
  return B <= kMaxCount && Hq <= kMaxCount && Sq <= kMaxCount / 2 && C <= kMaxCount / 2 && P <= kMaxCount / 2 && B * Hq <= kMaxCount &&
         B * Hq * Sq <= kMaxCount - 4096 && C + P <= kMaxCount - 4096;
}

}  // namespace

int span_rows_run(int dtype, const SpanArgs& a, int mode, int slices, const SpanPart& part, hipStream_t st) {
  note_kernel("%s rows split%d", a.pk ? "shared_prefix" : "sliding_window", slices);
  return dispatch_float16_32(dtype, "attention", [&](auto tag) {
    using T = decltype(tag);
    if (a.D <= 64) return launch_rows<T, 4>(a, mode, slices, part, st);
    if (a.D <= 128) return launch_rows<T, 8>(a, mode, slices, part, st);
    return launch_rows<T, 16>(a, mode, slices, part, st);
  });
}

}  // namespace ntops

using namespace ntops;

namespace {

// Checks what both operators share, and fills in the arguments.
int span_args(const char* what, SpanArgs& a, int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t C, int64_t D,
              int64_t P, const void* q, const int64_t* q_strides, const void* key, const int64_t* key_strides,
              const void* value, const int64_t* value_strides, const void* lengths, int lengths_dtype, double scale, void* out,
              const int64_t* out_strides, void* workspace, int64_t workspace_bytes) {
  if (dtype != NTOPS_F32 && dtype != NTOPS_F16 && dtype != NTOPS_BF16)
    return set_error(NTOPS_ERR_UNSUPPORTED, "%s: unsupported dtype %d (F32/F16/BF16 only)", what, dtype);
  if (lengths && !index_dtype(lengths_dtype)) return set_error(NTOPS_ERR_INVALID, "%s: lengths are I32 or I64", what);
  if (Hkv <= 0 || Hq % Hkv != 0)
    return set_error(NTOPS_ERR_INVALID, "%s: query heads are not a multiple of key / value heads", what);
  if (!q || !out || !q_strides || !out_strides || (C > 0 && (!key || !value || !key_strides || !value_strides)))
    return set_error(NTOPS_ERR_INVALID, "%s: null pointer", what);
  if (D > kMaxDim) return set_error(NTOPS_ERR_UNSUPPORTED, "%s: head dim over %d", what, kMaxDim);
  if (!sizes_fit(B, Hq, Sq, C, P)) return set_error(NTOPS_ERR_UNSUPPORTED, "%s: problem too large", what);
  if (workspace_bytes < 0 || (workspace != nullptr && !aligned16(workspace)))
    return set_error(NTOPS_ERR_INVALID, "%s: workspace not aligned to 16 bytes", what);
  a.q = q;
  a.o = out;
  a.k = key;
  a.v = value;
  for (int i = 0; i < 4; ++i) {
    a.qst[i] = q_strides[i];
    a.ost[i] = out_strides[i];
    if (C > 0) {
      a.kst[i] = key_strides[i];
      a.vst[i] = value_strides[i];
    }
  }
  a.lengths = lengths;
  a.lengths_dtype = lengths_dtype;
  a.B = static_cast<int>(B);
  a.Hq = static_cast<int>(Hq);
  a.Hkv = static_cast<int>(Hkv);
  a.Sq = static_cast<int>(Sq);
  a.C = static_cast<int>(C);
  a.D = static_cast<int>(D);
  a.G = a.B;
  a.window = static_cast<int>(kMaxCount / 2);
  a.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  return NTOPS_OK;
}

// Sizes alone, for the workspaces; false: nothing to attend, or a call that is refused.
bool span_sizes(SpanArgs& a, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t C, int64_t D, int64_t P) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Sq <= 0 || C < 0 || P < 0 || D <= 0 || D > kMaxDim || Hq % Hkv != 0 || !sizes_fit(B, Hq, Sq, C, P))
    return false;
  a.B = static_cast<int>(B);
  a.Hq = static_cast<int>(Hq);
  a.Hkv = static_cast<int>(Hkv);
  a.Sq = static_cast<int>(Sq);
  a.C = static_cast<int>(C);
  a.D = static_cast<int>(D);
  a.G = a.B;
  a.P = static_cast<int>(P);
  a.window = static_cast<int>(kMaxCount / 2);
  return true;
}

int clamp_count(int64_t n) { return static_cast<int>(std::min<int64_t>(n, kMaxCount / 2)); }

}  // namespace

extern "C" int64_t ntops_sliding_window_attention_workspace(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq,
                                                            int64_t C, int64_t D, int64_t window, int64_t sinks) {
  SpanArgs a{};
  if (!span_sizes(a, B, Hq, Hkv, Sq, C, D, 0) || window < 1 || sinks < 0) return 0;
  a.window = clamp_count(window);
  a.sinks = clamp_count(sinks);
  return workspace_bytes(dtype, a);
}

extern "C" int ntops_sliding_window_attention(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t C, int64_t D,
                                              const void* q, const int64_t* q_strides, const void* key,
                                              const int64_t* key_strides, const void* value, const int64_t* value_strides,
                                              const void* lengths, int lengths_dtype, int64_t window, int64_t sinks,
                                              double scale, void* out, const int64_t* out_strides, void* workspace,
                                              int64_t workspace_bytes, void* stream) {
  constexpr const char* what = "sliding_window_attention";
  if (B < 0 || Hq < 0 || Hkv < 0 || Sq < 0 || C < 0 || D < 0) return set_error(NTOPS_ERR_INVALID, "%s: negative size", what);
  if (window < 1 || sinks < 0) return set_error(NTOPS_ERR_INVALID, "%s: a window of at least 1, sinks of at least 0", what);
  if (B == 0 || Hq == 0 || Sq == 0 || D == 0) return NTOPS_OK;
  SpanArgs a{};
  if (int e = span_args(what, a, dtype, B, Hq, Hkv, Sq, C, D, 0, q, q_strides, key, key_strides, value, value_strides, lengths,
                        lengths_dtype, scale, out, out_strides, workspace, workspace_bytes))
    return e;
  a.window = clamp_count(window);
  a.sinks = clamp_count(sinks);
  return run(dtype, a, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int64_t ntops_shared_prefix_attention_workspace(int dtype, int64_t G, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq,
                                                           int64_t P, int64_t C, int64_t D) {
  SpanArgs a{};
  if (!span_sizes(a, B, Hq, Hkv, Sq, C, D, P) || G <= 0 || B % G != 0) return 0;
  a.G = static_cast<int>(G);
  a.pk = &a;  // (a prefix there is)
  return workspace_bytes(dtype, a);
}

extern "C" int ntops_shared_prefix_attention(int dtype, int64_t G, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t P,
                                             int64_t C, int64_t D, const void* q, const int64_t* q_strides,
                                             const void* prefix_key, const int64_t* prefix_key_strides,
                                             const void* prefix_value, const int64_t* prefix_value_strides,
                                             const void* prefix_lengths, int prefix_lengths_dtype, const void* key,
                                             const int64_t* key_strides, const void* value, const int64_t* value_strides,
                                             const void* lengths, int lengths_dtype, double scale, void* out,
                                             const int64_t* out_strides, void* workspace, int64_t workspace_bytes, void* stream) {
  constexpr const char* what = "shared_prefix_attention";
  if (G < 0 || B < 0 || Hq < 0 || Hkv < 0 || Sq < 0 || P < 0 || C < 0 || D < 0)
    return set_error(NTOPS_ERR_INVALID, "%s: negative size", what);
  if (B == 0 || Hq == 0 || Sq == 0 || D == 0) return NTOPS_OK;
  if (G == 0 || B % G != 0) return set_error(NTOPS_ERR_INVALID, "%s: the batch is not a multiple of the prefixes", what);
  SpanArgs a{};
  if (int e = span_args(what, a, dtype, B, Hq, Hkv, Sq, C, D, P, q, q_strides, key, key_strides, value, value_strides, lengths,
                        lengths_dtype, scale, out, out_strides, workspace, workspace_bytes))
    return e;
  if (P > 0 && (!prefix_key || !prefix_value || !prefix_key_strides || !prefix_value_strides))
    return set_error(NTOPS_ERR_INVALID, "%s: null pointer", what);
  if (prefix_lengths && !index_dtype(prefix_lengths_dtype))
    return set_error(NTOPS_ERR_INVALID, "%s: prefix lengths are I32 or I64", what);
  a.G = static_cast<int>(G);
  a.P = static_cast<int>(P);
  a.pk = P > 0 ? prefix_key : out;  // (no key of it is read)
  a.pv = P > 0 ? prefix_value : out;
  for (int i = 0; i < 4 && P > 0; ++i) {
    a.pkst[i] = prefix_key_strides[i];
    a.pvst[i] = prefix_value_strides[i];
  }
  a.plengths = prefix_lengths;
  a.plengths_dtype = prefix_lengths_dtype;
  return run(dtype, a, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}
