// Shared by the kernels of sliding_window_attention and shared_prefix_attention
// (attn_spans*.hip).
//
// Both operators attend two spans of keys, one behind the other:
//   front   keys that every row of a block sees: the sinks that lie before the
//           window, or a prefix that several sequences share;
//   main    the block's own stretch of a sequence: row t (its token p) sees the
//           keys p - window < j <= p, and of the sinks those that lie in it.
// A block works out its spans from the lengths on the device, so that nothing
// before `first`, the first key that its first row sees, is read or counted.
#pragma once

#include "attention.h"
#include "kv_cache.h"

namespace ntops {

struct SpanArgs {
  const void* q;
  void* o;
  const void* k;  // (B, Hkv, C, D)
  const void* v;
  const void* pk;  // (G, Hkv, P, D), null: no shared prefix
  const void* pv;
  int64_t qst[4], ost[4], kst[4], vst[4], pkst[4], pvst[4];
  const void* lengths;   // tokens of each sequence (null: C)
  const void* plengths;  // tokens of each prefix (null: P)
  int lengths_dtype, plengths_dtype;
  int B, Hq, Hkv, Sq, C, D, G, P;
  int group, per;  // query heads of a cache head; sequences of a prefix
  int window, sinks;  // at least 1; 0 with a shared prefix
  float scale_log2;   // scale * log2(e)
};

// Which spans a launch attends; its rows follow from them:
//  kBoth, kMain  a set of rows is (batch, cache head), row r is token r / group of
//                head r % group (so that a block's rows see nearly the same keys)
//  kFront        a set is (prefix, cache head), and its rows are those of all
//                sequences that share the prefix, one sequence behind the other
enum SpanMode { kBoth = 0, kMain = 1, kFront = 2 };

// Sets of rows and rows of each.
inline int64_t span_sets(const SpanArgs& a, int mode) { return static_cast<int64_t>(mode == kFront ? a.G : a.B) * a.Hkv; }
inline int64_t span_rows(const SpanArgs& a, int mode) {
  const int64_t rows = static_cast<int64_t>(a.Hq / a.Hkv) * a.Sq;
  return mode == kFront ? rows * (a.B / a.G) : rows;
}

// Where a set's rows and keys are.
struct SpanSet {
  int at;  // sequence, or prefix
  int b0;  // first sequence
  int hk;  // cache head
};
// (Every count of blocks and rows is below 2^32: quotients of 64 bits would cost hundreds
// of instructions a wave.)
__device__ __forceinline__ SpanSet span_set(const SpanArgs& a, int mode, uint32_t set) {
  SpanSet s;
  const uint32_t at = set / static_cast<uint32_t>(a.Hkv);
  s.at = static_cast<int>(at);
  s.hk = static_cast<int>(set - at * a.Hkv);
  s.b0 = mode == kFront ? s.at * a.per : s.at;
  return s;
}

// The spans of a block of rows; wave-uniform.
struct Spans : SpanSet {
  const char* k[2];  // front, main: first key
  const char* v[2];
  int n[2];          // keys
  int64_t kld[2], vld[2];  // strides in elements
  int place;         // main key of the first token (t = 0) of a row; -Sq or less: before the main span
  int window, sinks;  // sinks: main keys below it are seen whatever the window
  // main keys [lo, hi) are seen by a row of token t, and those below `sinks`
  __device__ __forceinline__ int hi(int t) const { return max(0, min(n[1], place + t + 1)); }
  __device__ __forceinline__ int lo(int t) const { return max(0, place + t - window + 1); }
};

__device__ __forceinline__ int span_length(const void* p, int dtype, int i, int most) {
  return static_cast<int>(max(int64_t(0), min(static_cast<int64_t>(most), index_at(p, dtype, i, most))));
}

// Spans of the rows of tokens t0 .. t1 of set `set`; ES: bytes of an element.
template <int ES>
__device__ __forceinline__ Spans make_spans(const SpanArgs& a, int mode, uint32_t set, int t0, int t1) {
  Spans s;
  static_cast<SpanSet&>(s) = span_set(a, mode, set);
  const int at = s.at;
  s.n[0] = s.n[1] = 0;
  s.k[0] = s.k[1] = static_cast<const char*>(a.k);
  s.v[0] = s.v[1] = static_cast<const char*>(a.v);
  s.kld[0] = s.kld[1] = a.kst[2];
  s.vld[0] = s.vld[1] = a.vst[2];
  s.place = -a.Sq;
  s.window = a.window;
  s.sinks = 0;
  if (mode != kFront) {
    const int n = span_length(a.lengths, a.lengths_dtype, at, a.C);
    const int p0 = n - a.Sq;
    const int first = max(0, p0 + t0 - a.window + 1);  // (window >= 1: no overflow)
    const int end = max(0, p0 + t1 + 1);               // <= n
    const int64_t kb = at * a.kst[0] + s.hk * a.kst[1], vb = at * a.vst[0] + s.hk * a.vst[1];
    s.n[1] = max(0, end - first);
    s.k[1] += (kb + first * a.kst[2]) * ES;
    s.v[1] += (vb + first * a.vst[2]) * ES;
    s.place = p0 - first;
    s.sinks = a.sinks - first;
    if (a.pk == nullptr) {
      s.n[0] = min(a.sinks, first);
      s.k[0] += kb * ES;
      s.v[0] += vb * ES;
    }
  }
  if (a.pk != nullptr && mode != kMain) {
    const int g = mode == kFront ? at : static_cast<int>(static_cast<uint32_t>(at) / static_cast<uint32_t>(a.per));
    s.n[0] = span_length(a.plengths, a.plengths_dtype, g, a.P);
    s.k[0] = static_cast<const char*>(a.pk) + (g * a.pkst[0] + s.hk * a.pkst[1]) * ES;
    s.v[0] = static_cast<const char*>(a.pv) + (g * a.pvst[0] + s.hk * a.pvst[1]) * ES;
    s.kld[0] = a.pkst[2];
    s.vld[0] = a.pvst[2];
  }
  return s;
}

// Row r of a set: its sequence (from the set's first), token and query head.
struct SpanRow {
  int b, t, h;
};
__device__ __forceinline__ SpanRow span_row(const SpanArgs& a, int mode, const SpanSet& s, int row) {
  const uint32_t group = static_cast<uint32_t>(a.group);
  uint32_t r = static_cast<uint32_t>(row), b = 0;
  if (mode == kFront) {
    const uint32_t ro = group * a.Sq;
    b = r / ro;
    r -= b * ro;
  }
  const uint32_t t = r / group;
  return {s.b0 + static_cast<int>(b), static_cast<int>(t), s.hk * a.group + static_cast<int>(r - t * group)};
}

// Partial results of slices: per query row (batch, head, token) and slice the
// unnormalized O row of `ld` floats, then for each the pair (max in base 2, sum).
struct SpanPart {
  float* p;         // null: one slice, O normalized into the output
  int slices;       // of a row, over all launches
  int first;        // this launch's first slice
  int ld;           // D rounded up to 4
  __device__ __forceinline__ int64_t at(const SpanArgs& a, const SpanRow& x, int slice) const {
    return ((static_cast<int64_t>(x.b) * a.Hq + x.h) * a.Sq + x.t) * slices + first + slice;
  }
  __device__ __forceinline__ float* row(int64_t at) const { return p + at * ld; }
  __device__ __forceinline__ float* ml(const SpanArgs& a, int64_t at) const {
    return p + static_cast<int64_t>(a.B) * a.Hq * a.Sq * slices * ld + 2 * at;
  }
};

// A product rounded by itself, which no fma takes in.  Scores that are compared as rounded
// products have their exponents from the same ones: an fma against a maximum that was rounded is
// off by half a unit of the maximum, which past 2^24 is a factor of two and soon all there is.
__device__ __forceinline__ float product(float a, float b) {
  float p = a * b;
  asm("" : "+v"(p));
  return p;
}
// References (base 2) from which on the 16-bit kernels of the matrix cores take exponents so, by
// two instructions a score; below, one fma, off by a factor under two that all of a row's
// probabilities share.
__device__ __forceinline__ bool span_far(float m) { return fabsf(m) >= 0x1p24f && m != neg_inf(); }

// A mean of values as the type.  It passes none of them, but where probabilities were rounded up
// together it does by up to half a step, and next to f16's largest value that is infinity.
// (bf16 sums of such values pass fp32's range: such rows are computed again, unrounded.)
template <typename T>
__device__ __forceinline__ T mean_as(float x) {
  if constexpr (std::is_same<T, _Float16>::value) x = fabsf(x) < __builtin_huge_valf() ? __builtin_amdgcn_fmed3f(x, -65504.f, 65504.f) : x;
  return static_cast<T>(x);
}

// One query row by one wave, fp32 throughout, any head dim up to 16 EL and any
// strides; reads nothing that the row does not see.  Sixteen lanes share a key
// (lane i the columns i + 16 u), four keys side by side, UNROLL of them in flight
// each; the four streams of keys are joined at the end.  Every lane ends with the
// whole row: o[u] of column (lane & 15) + 16 u.
//
// Front keys [f0, f1) and main keys [m0, m1) of what the row sees.  MEAN: o is divided by
// the sum at every step, so that it never passes the largest value; without, o is the sum
// of values times weights, which may where the result does not.
template <typename T, int EL, int UNROLL, bool MEAN>
__device__ __forceinline__ void span_attend_row(const SpanArgs& a, const Spans& s, const SpanRow x, int f0, int f1, int m0,
                                             int m1, float (&o)[EL], float& m, float& l) {
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  float q[EL];
  const T* Q = static_cast<const T*>(a.q) + x.b * a.qst[0] + x.h * a.qst[1] + x.t * a.qst[2];
#pragma unroll
  for (int u = 0; u < EL; ++u) {
    q[u] = i + 16 * u < a.D ? static_cast<float>(Q[(i + 16 * u) * a.qst[3]]) : 0.f;
    o[u] = 0.f;
  }
  m = neg_inf();
  l = 0.f;
  const int64_t kd[2] = {a.pk ? a.pkst[3] : a.kst[3], a.kst[3]};
  const int64_t vd[2] = {a.pk ? a.pvst[3] : a.vst[3], a.vst[3]};
  const int hi = s.hi(x.t), lo = s.lo(x.t);
  for (int part = 0; part < 3; ++part) {
    // the front; sinks in the main span that the window has left behind; the window
    const int sp = part == 0 ? 0 : 1;
    const int k0 = part == 0 ? f0 : part == 1 ? m0 : max(m0, lo);
    const int k1 = part == 0 ? min(f1, s.n[0]) : part == 1 ? min(m1, min(lo, min(s.sinks, hi))) : min(m1, hi);
    const T* K = reinterpret_cast<const T*>(s.k[sp]);
    const T* V = reinterpret_cast<const T*>(s.v[sp]);
    for (int k = k0 + g; k < k1; k += 4 * UNROLL) {
      float kv[UNROLL][EL], vv[UNROLL][EL];
#pragma unroll
      for (int w = 0; w < UNROLL; ++w) {
        const int64_t key = k + 4 * w;
        const bool in = key < k1;
#pragma unroll
        for (int u = 0; u < EL; ++u) {
          const bool ok = in && i + 16 * u < a.D;
          kv[w][u] = ok ? static_cast<float>(K[key * s.kld[sp] + (i + 16 * u) * kd[sp]]) : 0.f;
          vv[w][u] = ok ? static_cast<float>(V[key * s.vld[sp] + (i + 16 * u) * vd[sp]]) : 0.f;
        }
      }
#pragma unroll
      for (int w = 0; w < UNROLL; ++w) {
        float d = 0.f;
#pragma unroll
        for (int u = 0; u < EL; ++u) d = fmaf(q[u], kv[w][u], d);
        d += dpp_mov<kDppXor1>(d);
        d += dpp_mov<kDppXor2>(d);
        d += dpp_mov<kDppHalfMirror>(d);
        d += dpp_mov<kDppMirror>(d);
        const float sc = k + 4 * w < k1 ? product(d, a.scale_log2) : neg_inf();
        const float m_new = fmaxf(m, sc);
        const float m_use = m_new == neg_inf() ? 0.f : m_new;
        float alpha = fast_exp2(m - m_use), p = fast_exp2(sc - m_use);
        const float l_new = l * alpha + p;
        if (MEAN) {
          const float by = l_new == 0.f ? 0.f : 1.f / l_new;
          alpha *= l * by;
          p *= by;
        }
        l = l_new;
#pragma unroll
        for (int u = 0; u < EL; ++u) o[u] = fmaf(p, vv[w][u], o[u] * alpha);
        m = m_new;
      }
    }
  }
#pragma unroll
  for (int step = 16; step <= 32; step <<= 1) {
    const float m2 = __shfl_xor(m, step, 64);
    const float mm = fmaxf(m, m2), m_use = mm == neg_inf() ? 0.f : mm;
    float f = fast_exp2(m - m_use), f2 = fast_exp2(m2 - m_use);
    const float l2 = __shfl_xor(l, step, 64), l_new = l * f + l2 * f2;
    if (MEAN) {
      const float by = l_new == 0.f ? 0.f : 1.f / l_new;
      f *= l * by;
      f2 *= l2 * by;
    }
    l = l_new;
#pragma unroll
    for (int u = 0; u < EL; ++u) o[u] = o[u] * f + __shfl_xor(o[u], step, 64) * f2;
    m = mm;
  }
}

// Writes such a row: to the output, or as slice `slice` of the partial results -- a mean
// under a sum and a weight of it in (0.5, 1] with a power of two taken into the maximum.
template <typename T, int EL, bool MEAN>
__device__ __forceinline__ void span_write_row(const SpanArgs& a, const SpanPart& part, const SpanRow& x, int slice,
                                               const float (&o)[EL], float m, float l) {
  const int lane = threadIdx.x & 63;
  if (lane >= 16) return;
  if (part.p) {
    const int64_t at = part.at(a, x, slice);
    float f = 1.f;
    if (MEAN && l > 0.f) {
      m += static_cast<float>(__builtin_amdgcn_frexp_expf(l));
      l = f = __builtin_amdgcn_frexp_mantf(l);
    }
    if (lane == 0) {
      float* ml = part.ml(a, at);
      ml[0] = m;
      ml[1] = l;
    }
#pragma unroll
    for (int u = 0; u < EL; ++u)
      if (lane + 16 * u < a.D) part.row(at)[lane + 16 * u] = o[u] * f;
    return;
  }
  const float inv = l == 0.f ? 0.f : MEAN ? 1.f : 1.f / l;  // (a NaN sum, from a NaN score, passes through)
  T* O = static_cast<T*>(a.o) + x.b * a.ost[0] + x.h * a.ost[1] + x.t * a.ost[2];
#pragma unroll
  for (int u = 0; u < EL; ++u)
    if (lane + 16 * u < a.D) O[(lane + 16 * u) * a.ost[3]] = mean_as<T>(o[u] * inv);
}

// What has to be computed again by itself: a sum of a row's columns that is no number, or
// none that fp32 holds, under a sum of weights that is one.
__device__ __forceinline__ bool span_again(float any, float l) { return !(any - any == 0.f) && l == l; }
// The row again, from keys [f0, f1) of the front and [m0, m1) of the main span.  A row that sees
// an infinity or a NaN itself comes here too, for the result that it had: a wave takes such
// rows one after the other, 100 to 200 times as long as the matrix cores.  (1, 32 / 8,
// 4096, window 1024) bf16 of 128 with one infinite value among a head's sinks 15.4 ms (90 us
// without), with one key in flight instead of four 22.7; fp32 6.5 (four keys: 16.8) against 0.61;
// (64, 32 / 8, 1 over 4096) with one in every head 7.4 ms against 0.16.
template <typename T, int EL>
__device__ __forceinline__ void span_row_again(const SpanArgs& a, const Spans& s, const SpanPart& part, const SpanRow& x, int slice, int f0, int f1,
                                               int m0, int m1) {
  float o[EL], m, l;
  span_attend_row<T, EL, (sizeof(T) == 2 && EL == 8 ? 4 : 1), true>(a, s, x, f0, f1, m0, m1, o, m, l);
  span_write_row<T, EL, true>(a, part, x, slice, o, m, l);
}

// ---- paths (host) ------------------------------------------------------------

// Any types, head dims and layouts: a wave per row and slice.
int span_rows_run(int dtype, const SpanArgs& a, int mode, int slices, const SpanPart& part, hipStream_t st);

// 16-bit types, head dims up to 128, at most kFewRows rows of a sequence a cache head.
// front_slices > 0: with the rows of all sequences of a group (span_few_run: at most 16)
// over their prefix, in that many slices that come before the others.
constexpr int kFewRows = 32;
struct FewPlan {
  int waves;  // a block, 1 or 2
  int mode;   // of each sequence's rows
  int front_slices, slices;
};
int span_few_run(int dtype, const SpanArgs& a, const FewPlan& p, const SpanPart& part, hipStream_t st);
int span_mixed_run(int dtype, const SpanArgs& a, const FewPlan& p, const SpanPart& part, hipStream_t st);

// 16-bit types, head dims that are multiples of 8: any number of rows, in blocks of
// kTileRows.
constexpr int kTileRows = 128;
int span_tile_run(int dtype, const SpanArgs& a, int mode, int slices, const SpanPart& part, hipStream_t st);

// fp32, head dims that are multiples of 4, rows at multiples of 16 bytes: any number of
// rows, in blocks of kF32Rows.
constexpr int kF32Rows = 128;
constexpr int kF32FewRows = 16;  // head dims up to 128: a set with no more is one block's
int span_f32_run(const SpanArgs& a, int mode, int slices, const SpanPart& part, hipStream_t st);

}  // namespace ntops
