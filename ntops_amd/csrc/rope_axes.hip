// Rotary positions with several axes on the query and key of a layer, each
// (B, S, H, D):
//   out0 = x0 cos - x1 sin,  out1 = x1 cos + x0 sin
// for the pairs (i, i + D / 2), or (2 i, 2 i + 1) interleaved, with sin and cos of
// pair i from row positions[axis(i)][b][s] of the tables: column i of tables of
// D / 2 columns, the elements' own columns of tables of D.  In fp32, rounded once.
// A pair whose position lies outside of the tables is NaN.
//
// Bound by reading and writing the heads once.  Vector path: a thread owns the pairs of
// a 16-byte pack of each half of a token's head, or of a pack of interleaved pairs,
// gathers their sines and cosines once and rotates several heads with them: the tables'
// bytes, fp32 and from a row of its own for each axis, would otherwise pass the L1 as
// often as the heads' own.  Generic path: a thread per pair, any strides.
#include <algorithm>
#include <cstdlib>

#include "dispatch.h"
#include "kv_cache.h"

namespace ntops {
namespace {

constexpr int kMaxPairs = 256;

struct AxesTensor {
  const void* x;
  void* y;
  int64_t H;
  int64_t xs[4], ys[4];
};

struct AxesArgs {
  int64_t B, S, D;
  AxesTensor t[2];  // query, key; H == 0: none
  const void* sn;
  const void* cs;
  int64_t srs, crs;  // row strides of the tables
  int64_t rows;      // of the tables
  int wide;          // tables of D columns
  int interleaved;
  const void* pos;   // (axes, B, S)
  int64_t ps[3];
  int pos_dtype;
  alignas(8) uint8_t axis[kMaxPairs];
};

template <typename T>
__device__ __forceinline__ void rotate_pair(float x0, float x1, float c0, float s0, float c1, float s1, T& y0, T& y1) {
  float o0 = fmaf(x0, c0, -(x1 * s0)), o1 = fmaf(x1, c1, x0 * s1);
  // One rounding to fp32, then one to the type, wherever a pair comes in the code: else some
  // f16 results are rounded from the exact sum by a mixed-precision fma and others are not,
  // and a head's last bit depends on which thread has it.
  if constexpr (std::is_same<T, _Float16>::value) asm("" : "+v"(o0), "+v"(o1));
  y0 = static_cast<T>(o0);
  y1 = static_cast<T>(o1);
}

// Row of the tables of pair i's axis at token (b, s); -1: outside.
__device__ __forceinline__ int64_t table_row(const AxesArgs& a, int axis, int64_t b, int64_t s) {
  const int64_t p = index_at(a.pos, a.pos_dtype, axis * a.ps[0] + b * a.ps[1] + s * a.ps[2], 0);
  return p >= 0 && p < a.rows ? p : -1;
}

// Sine and cosine of column `col` of row `row`.
template <typename TT>
__device__ __forceinline__ void table_at(const AxesArgs& a, int64_t row, int64_t col, float& sn, float& cs) {
  const float nan = __builtin_nanf("");
  sn = row < 0 ? nan : static_cast<float>(static_cast<const TT*>(a.sn)[row * a.srs + col]);
  cs = row < 0 ? nan : static_cast<float>(static_cast<const TT*>(a.cs)[row * a.crs + col]);
}

// N columns of a table's row, at any element.
template <typename TT, int N>
__device__ __forceinline__ void load_run(const TT* p, float (&v)[N]) {
  if constexpr (std::is_same<TT, float>::value && N % 4 == 0) {
    typedef float Run __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const Run r = reinterpret_cast<const Run*>(p)[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * i + e] = r[e];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = static_cast<float>(p[i]);
  }
}

// T: element type, TT: the tables' type.
template <typename T, typename TT>
__global__ __launch_bounds__(256) void k_rope_axes_generic(AxesArgs a, int64_t pairs0, int64_t pairs) {
  const int64_t half = a.D / 2;
  for (int64_t it = block_id() * 256 + threadIdx.x; it < pairs; it += static_cast<int64_t>(gridDim.x) * gridDim.y * 256) {
    const bool second = it >= pairs0;
    const AxesTensor& d = a.t[second ? 1 : 0];
    const int64_t li = second ? it - pairs0 : it;
    const int64_t i = li % half;
    int64_t r = li / half;
    const int64_t h = r % d.H;
    r /= d.H;
    const int64_t s = r % a.S, b = r / a.S;
    const T* x = static_cast<const T*>(d.x) + b * d.xs[0] + s * d.xs[1] + h * d.xs[2];
    T* y = static_cast<T*>(d.y) + b * d.ys[0] + s * d.ys[1] + h * d.ys[2];
    const int64_t d0 = a.interleaved ? 2 * i : i, d1 = a.interleaved ? 2 * i + 1 : i + half;
    const int64_t row = table_row(a, a.axis[i], b, s);
    float s0, c0, s1, c1;
    table_at<TT>(a, row, a.wide ? d0 : i, s0, c0);
    table_at<TT>(a, row, a.wide ? d1 : i, s1, c1);
    const float x0 = static_cast<float>(x[d0 * d.xs[3]]), x1 = static_cast<float>(x[d1 * d.xs[3]]);
    rotate_pair(x0, x1, c0, s0, c1, s1, y[d0 * d.ys[3]], y[d1 * d.ys[3]]);
  }
}

// Vector path.  A block covers 256 work items: (token, pack j of the head, part of the
// heads); a thread keeps the sines and cosines of its 8 (fp32: 4) pairs -- of an
// interleaved pack of V elements V / 2 pairs -- and takes the heads hp, hp + parts, ...
// of the query and then of the key, kUnroll of them in flight.
template <typename T, typename TT, bool INTER>
__global__ __launch_bounds__(256) void k_rope_axes(AxesArgs a, int parts, uint32_t items) {
  constexpr int V = Pack16<T>::N;
  constexpr int NP = INTER ? V / 2 : V;  // pairs of a thread
  constexpr int kUnroll = 2;
  const uint32_t it = static_cast<uint32_t>(block_id()) * 256 + threadIdx.x;
  if (it >= items) return;
  const uint32_t half = static_cast<uint32_t>(a.D / 2), packs = half / NP;
  const uint32_t j = it % packs;
  uint32_t r = it / packs;
  const uint32_t hp = r % parts;
  r /= parts;
  const uint32_t S = static_cast<uint32_t>(a.S);
  const uint32_t tb = r / S, ts = r - tb * S;
  // heads of both tensors as one list: query heads, then key heads
  const int hq = static_cast<int>(a.t[0].H), heads = hq + static_cast<int>(a.t[1].H);
  const T* x[2];
  T* y[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    x[t] = static_cast<const T*>(a.t[t].x) + tb * a.t[t].xs[0] + ts * a.t[t].xs[1] + (INTER ? j * V : j * NP);
    y[t] = static_cast<T*>(a.t[t].y) + tb * a.t[t].ys[0] + ts * a.t[t].ys[1] + (INTER ? j * V : j * NP);
  }
  Pack16<T> p0[kUnroll], p1[kUnroll];
  const auto load = [&](int h, Pack16<T>& u, Pack16<T>& w) {
    const bool k = h >= hq;
    const T* p = k ? x[1] + (h - hq) * a.t[1].xs[2] : x[0] + h * a.t[0].xs[2];
    u = load16_nt(p);
    if constexpr (!INTER) w = load16_nt(p + half);
  };
#pragma unroll
  for (int u = 0; u < kUnroll; ++u)
    if (static_cast<int>(hp) + u * parts < heads) load(hp + u * parts, p0[u], p1[u]);

  float s0[NP], c0[NP], s1[NP], c1[NP];
  using Axes = std::conditional_t<NP == 8, uint64_t, std::conditional_t<NP == 4, uint32_t, uint16_t>>;
  const Axes axes = reinterpret_cast<const Axes*>(a.axis)[j];  // of the thread's pairs
  const uint32_t pair0 = j * NP;
  if (axes == static_cast<Axes>(static_cast<uint8_t>(axes) * static_cast<Axes>(0x0101010101010101ull)) && !(INTER && a.wide)) {
    // one position, and runs of the tables' columns
    const int64_t row = table_row(a, static_cast<uint8_t>(axes), tb, ts);
    const int64_t so = max(row, int64_t(0)) * a.srs + pair0, co = max(row, int64_t(0)) * a.crs + pair0;
    if (row >= 0) {
      load_run<TT, NP>(static_cast<const TT*>(a.sn) + so, s0);
      load_run<TT, NP>(static_cast<const TT*>(a.cs) + co, c0);
    } else {
#pragma unroll
      for (int i = 0; i < NP; ++i) s0[i] = c0[i] = __builtin_nanf("");
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      s1[i] = s0[i];
      c1[i] = c0[i];
    }
    if (a.wide && row >= 0) {
      load_run<TT, NP>(static_cast<const TT*>(a.sn) + so + half, s1);
      load_run<TT, NP>(static_cast<const TT*>(a.cs) + co + half, c1);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const uint32_t pair = pair0 + i;
      const int64_t row = table_row(a, static_cast<uint8_t>(axes >> (8 * i)), tb, ts);
      const uint32_t d0 = INTER ? 2 * pair : pair, d1 = INTER ? 2 * pair + 1 : pair + half;
      table_at<TT>(a, row, a.wide ? d0 : pair, s0[i], c0[i]);
      s1[i] = s0[i];
      c1[i] = c0[i];
      if (a.wide) table_at<TT>(a, row, d1, s1[i], c1[i]);
    }
  }
  for (int h0 = hp; h0 < heads; h0 += kUnroll * parts) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int h = h0 + u * parts;
      if (h >= heads) break;
      const Pack16<T> v0 = p0[u], v1 = p1[u];
      if (h + kUnroll * parts < heads) load(h + kUnroll * parts, p0[u], p1[u]);
      const bool k = h >= hq;
      T* p = k ? y[1] + (h - hq) * a.t[1].ys[2] : y[0] + h * a.t[0].ys[2];
      Pack16<T> o0, o1;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        if constexpr (INTER)
          rotate_pair(static_cast<float>(v0.v[2 * i]), static_cast<float>(v0.v[2 * i + 1]), c0[i], s0[i], c1[i], s1[i], o0.v[2 * i], o0.v[2 * i + 1]);
        else
          rotate_pair(static_cast<float>(v0.v[i]), static_cast<float>(v1.v[i]), c0[i], s0[i], c1[i], s1[i], o0.v[i], o1.v[i]);
      }
      store16_nt(p, o0);
      if constexpr (!INTER) store16_nt(p + half, o1);
    }
  }
}

template <typename T, typename TT>
int run_axes(const AxesArgs& a, hipStream_t st) {
  constexpr int V = Pack16<T>::N;
  const int64_t tokens = a.B * a.S, heads = a.t[0].H + a.t[1].H;
  // (the vector path's heads are 32-bit: parts <= heads, so h + kUnroll * parts < 3 * 2^29)
  bool vec = (a.D / 2) % (a.interleaved ? V / 2 : V) == 0 && heads <= (int64_t(1) << 29);
  for (const AxesTensor& d : a.t) {
    if (d.H == 0) continue;
    vec = vec && d.xs[3] == 1 && d.ys[3] == 1 && aligned16(d.x) && aligned16(d.y);
    for (int k = 0; k < 3; ++k) vec = vec && d.xs[k] % V == 0 && d.ys[k] % V == 0;
  }
  const int64_t packs = a.D / 2 / (a.interleaved ? V / 2 : V);
  if (vec) {
    // Heads of a thread: as many as leave every CU five blocks, which its registers hold,
    // at most four -- where a thread's pairs belong to several axes, so that it gathers
    // each by itself, eight.  (4, 4096, 32 + 8, 128) bf16, 1 / 2 / 4 / 8 / 20 heads: 75.1 /
    // 63.3 / 60.5 / 62.3 / 71.6 us (344 MB, 5.7 TB/s; a copy of as much takes 64), pairs of
    // axes in turn 175.9 / 110.7 / 85.7 / 76.5 / 78.9; f32 122.5 / 115.3 / 114.3 / 118.8 / 130.5.
    const int np = a.interleaved ? V / 2 : V;
    bool runs = true;
    for (int i = 0; i < a.D / 2; ++i) runs = runs && a.axis[i] == a.axis[i - i % np];
    const int64_t blocks = static_cast<int64_t>(cu_count_cached()) * 5;
    const int64_t per = std::max<int64_t>(1, std::min<int64_t>({heads, tokens * packs * heads / (256 * blocks), runs ? 4 : 8}));
    const int64_t parts = ceil_div(heads, per);
    const int64_t items = tokens * packs * parts;
    if (items < 0xffffff00LL) {
      note_kernel("rope_axes heads%lld", static_cast<long long>(per));
      const dim3 grid = blocks_2d(ceil_div(items, 256));
      if (a.interleaved)
        hipLaunchKernelGGL((k_rope_axes<T, TT, true>), grid, dim3(256), 0, st, a, static_cast<int>(parts), static_cast<uint32_t>(items));
      else
        hipLaunchKernelGGL((k_rope_axes<T, TT, false>), grid, dim3(256), 0, st, a, static_cast<int>(parts), static_cast<uint32_t>(items));
      return check_launch("rope_axes");
    }
  }
  const int64_t pairs0 = tokens * a.t[0].H * (a.D / 2), pairs = tokens * heads * (a.D / 2);
  note_kernel("rope_axes generic");
  hipLaunchKernelGGL((k_rope_axes_generic<T, TT>), blocks_2d(std::min<int64_t>(ceil_div(pairs, 256), 1 << 20)), dim3(256), 0, st, a, pairs0,
                     pairs);
  return check_launch("rope_axes");
}

// ---- what tensors share (host) ------------------------------------------------

using Wide = __int128;  // sums of strides times sizes, whatever the caller gives

// Steps n of 0 .. most of a dim, or of one dim of each of two tensors together.
struct Steps {
  int64_t step, most;
};
struct Layout {
  Steps s[8];
  int n = 0;
  Wide before = 0;  // what steps below zero take from the first element's place
  void add(int64_t step, int64_t most) {
    if (most <= 0 || step == 0) return;
    if (step < 0) {
      before += static_cast<Wide>(step) * most;
      step = -step;
    }
    for (int i = 0; i < n; ++i)
      if (s[i].step == step) {
        s[i].most += most;
        return;
      }
    s[n++] = {step, most};
  }
  Wide reach() const {
    Wide r = 0;
    for (int i = 0; i < n; ++i) r += static_cast<Wide>(s[i].step) * s[i].most;
    return r;
  }
};

// Whether `left` is a sum of step * n over the layout's steps, largest first, which leaves
// few n where strides are those of nested dims; true where `trials` do not tell.
bool reaches(const Layout& a, int i, Wide rest, Wide left, int& trials) {
  if (left == 0) return true;
  if (left < 0 || left > rest) return false;
  const Wide step = a.s[i].step, behind = rest - step * a.s[i].most;
  const Wide last = std::min<Wide>(a.s[i].most, left / step);
  for (Wide n = left > behind ? (left - behind + step - 1) / step : 0; n <= last; ++n) {
    if (--trials < 0 || reaches(a, i + 1, behind, left - n * step, trials)) return true;
  }
  return false;
}
bool reaches(Layout& a, Wide target) {
  std::sort(a.s, a.s + a.n, [](const Steps& x, const Steps& y) { return x.step > y.step; });
  int trials = 10000;
  return reaches(a, 0, a.reach(), target, trials);
}

struct Strided {
  const void* p;
  const int64_t* st;
  int64_t size[4];
};

// Whether two elements of x are the same memory.
bool meets_itself(const Strided& x) {
  // no, where each dim's step passes all that the smaller ones reach
  Steps own[4];
  int n = 0;
  for (int i = 0; i < 4; ++i) {
    if (x.size[i] <= 1) continue;
    if (x.st[i] == 0) return true;
    own[n++] = {std::abs(x.st[i]), x.size[i] - 1};
  }
  std::sort(own, own + n, [](const Steps& x, const Steps& y) { return x.step < y.step; });
  Wide end = 1;
  int nested = 0;
  for (; nested < n && own[nested].step >= end; ++nested) end += static_cast<Wide>(own[nested].step) * own[nested].most;
  if (nested == n) return false;
  for (int i = 0; i < 4; ++i) {
    // index vectors that differ first in dim i, by n + 1, and by -most .. most behind it
    const int64_t most = x.size[i] - 1, step = std::abs(x.st[i]);
    if (most <= 0) continue;
    Layout a;
    a.add(step, most - 1);
    Wide target = -static_cast<Wide>(step);
    for (int j = i + 1; j < 4; ++j) {
      const int64_t s = std::abs(x.st[j]);
      a.add(s, 2 * (x.size[j] - 1));
      target += static_cast<Wide>(s) * (x.size[j] - 1);
    }
    if (reaches(a, target)) return true;
  }
  return false;
}

// Whether an element of x and one of y, of `es` bytes each, are the same memory.
bool meet(const Strided& x, const Strided& y, int es) {
  Layout a, b;
  for (int i = 0; i < 4; ++i) a.add(x.st[i], x.size[i] - 1);
  for (int i = 0; i < 4; ++i) b.add(y.st[i], y.size[i] - 1);
  const Wide apart = static_cast<Wide>(reinterpret_cast<intptr_t>(y.p)) - reinterpret_cast<intptr_t>(x.p);
  // in elements: the places of x are lowest + 0 .. reach, those of y likewise
  const Wide x_low = a.before * es, y_low = apart + b.before * es;
  const Wide x_high = x_low + a.reach() * es, y_high = y_low + b.reach() * es;
  if (y_low >= x_high + es || x_low >= y_high + es) return false;
  if (apart % es != 0) return true;
  // x's steps from its lowest place, and y's down from its highest
  for (int i = 0; i < b.n; ++i) a.add(b.s[i].step, b.s[i].most);
  return reaches(a, (y_high - x_low) / es);
}

}  // namespace
}  // namespace ntops

using namespace ntops;

extern "C" int ntops_rope_axes_qk(int dtype, int64_t B, int64_t S, int64_t Hq, int64_t Hk, int64_t D, const void* q,
                                  const int64_t* q_strides, const void* k, const int64_t* k_strides, int table_dtype,
                                  const void* sin_table, int64_t sin_row_stride, const void* cos_table, int64_t cos_row_stride,
                                  int64_t table_rows, int64_t table_cols, int64_t axes, const void* positions, int positions_dtype,
                                  const int64_t* position_strides, int64_t n_sections, const int64_t* sections, int interleaved,
                                  void* q_out, const int64_t* q_out_strides, void* k_out, const int64_t* k_out_strides,
                                  void* stream) {
  constexpr const char* what = "rope_axes_qk";
  if (B < 0 || S < 0 || Hq < 0 || Hk < 0 || D < 0 || table_rows < 0) return set_error(NTOPS_ERR_INVALID, "%s: negative size", what);
  if (dtype != NTOPS_F32 && dtype != NTOPS_F16 && dtype != NTOPS_BF16)
    return set_error(NTOPS_ERR_UNSUPPORTED, "%s: unsupported dtype %d (F32/F16/BF16 only)", what, dtype);
  if (table_dtype != NTOPS_F32 && table_dtype != dtype)
    return set_error(NTOPS_ERR_INVALID, "%s: tables are F32 or of the tensors' type", what);
  if (D % 2 != 0) return set_error(NTOPS_ERR_INVALID, "%s: the embedding dim must be even", what);
  if (D > 2 * kMaxPairs) return set_error(NTOPS_ERR_UNSUPPORTED, "%s: embedding dim %lld > %d", what, (long long)D, 2 * kMaxPairs);
  if (table_cols != D && table_cols != D / 2) return set_error(NTOPS_ERR_INVALID, "%s: tables must have D or D/2 columns", what);
  if (!index_dtype(positions_dtype)) return set_error(NTOPS_ERR_INVALID, "%s: positions are I32 or I64", what);
  if (axes < 1 || n_sections < 1 || !sections) return set_error(NTOPS_ERR_INVALID, "%s: no axes or sections", what);
  AxesArgs a{};
  int64_t filled = 0;
  for (int64_t s = 0; s < n_sections; ++s) {
    if (sections[s] < 0 || sections[s] > D / 2 - filled)
      return set_error(NTOPS_ERR_INVALID, "%s: the sections must add up to D/2", what);
    if (sections[s] > 0 && s % axes > 255) return set_error(NTOPS_ERR_UNSUPPORTED, "%s: more than 256 axes", what);
    for (int64_t i = 0; i < sections[s]; ++i) a.axis[filled++] = static_cast<uint8_t>(s % axes);
  }
  if (filled != D / 2) return set_error(NTOPS_ERR_INVALID, "%s: the sections must add up to D/2", what);
  if (B == 0 || S == 0 || Hq + Hk == 0 || D == 0) return NTOPS_OK;
  if (!positions || !position_strides || (table_rows > 0 && (!sin_table || !cos_table)) ||
      (Hq > 0 && (!q || !q_out || !q_strides || !q_out_strides)) || (Hk > 0 && (!k || !k_out || !k_strides || !k_out_strides)))
    return set_error(NTOPS_ERR_INVALID, "%s: null pointer", what);
  constexpr int64_t kMost = int64_t(1) << 40;
  if (B > kMost || S > kMost / B || Hq > kMost || Hk > kMost || (Hq + Hk) > kMost / (B * S))
    return set_error(NTOPS_ERR_UNSUPPORTED, "%s: problem too large", what);
  a.B = B;
  a.S = S;
  a.D = D;
  const void* xs[2] = {q, k};
  void* ys[2] = {q_out, k_out};
  const int64_t* xst[2] = {q_strides, k_strides};
  const int64_t* yst[2] = {q_out_strides, k_out_strides};
  const int64_t hs[2] = {Hq, Hk};
  for (int t = 0; t < 2; ++t) {
    a.t[t].H = hs[t];
    if (hs[t] == 0) continue;
    a.t[t].x = xs[t];
    a.t[t].y = ys[t];
    for (int d = 0; d < 4; ++d) {
      a.t[t].xs[d] = xst[t][d];
      a.t[t].ys[d] = yst[t][d];
    }
    if (xs[t] == ys[t])
      for (int d = 0; d < 4; ++d)
        if (xst[t][d] != yst[t][d]) return set_error(NTOPS_ERR_INVALID, "%s: in place needs equal strides", what);
  }
  // What one thread writes, no other may read or write.
  Strided x[2], y[2];
  for (int t = 0; t < 2; ++t) {
    x[t] = {xs[t], xst[t], {B, S, hs[t], D}};
    y[t] = {ys[t], yst[t], {B, S, hs[t], D}};
  }
  const int es = dtype == NTOPS_F32 ? 4 : 2;
  for (int t = 0; t < 2; ++t) {
    if (hs[t] == 0) continue;
    if (meets_itself(y[t])) return set_error(NTOPS_ERR_INVALID, "%s: elements of a result share memory", what);
    if (xs[t] != ys[t] && meet(x[t], y[t], es)) return set_error(NTOPS_ERR_INVALID, "%s: a result and its tensor share elements", what);
  }
  if (Hq > 0 && Hk > 0 && (meet(y[0], y[1], es) || meet(y[0], x[1], es) || meet(x[0], y[1], es)))
    return set_error(NTOPS_ERR_INVALID, "%s: q and k share elements that are written", what);
  a.sn = sin_table;
  a.cs = cos_table;
  a.srs = sin_row_stride;
  a.crs = cos_row_stride;
  a.rows = table_rows;
  a.wide = table_cols == D;
  a.interleaved = interleaved != 0;
  a.pos = positions;
  a.pos_dtype = positions_dtype;
  for (int d = 0; d < 3; ++d) a.ps[d] = position_strides[d];
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return dispatch_float16_32(dtype, what, [&](auto tag) {
    using T = decltype(tag);
    if (table_dtype == NTOPS_F32) return run_axes<T, float>(a, st);
    return run_axes<T, T>(a, st);
  });
}
