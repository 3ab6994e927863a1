// Keys and values into a cache of 8 bits.
//
// A block of tokens of one head has the scale 2^e, e the least integer >= -126
// with max |x| <= 448 2^e over its finite values; the values are x / 2^e
// rounded to e4m3 (NaN for what is not finite).  New tokens that start inside a
// block keep the larger of its scale and theirs; if theirs is larger, the
// block's earlier tokens are rounded again to it -- exactly, but for values that
// fall under e4m3's least exponent, as both scales are powers of two.  Tokens
// behind the new ones are left as they are.
//
// Bound by memory (es read, 1 byte written per value), or for single tokens by
// latency: a wave owns the block of a head -- its new values stay in registers
// between the maximum and the rounding, nothing is shared, no barrier: (32, 8, 1,
// 128) bf16 3.9 us, (4, 8, 2048, 128) 11.4 us and (1, 8, 16384, 128) 23.0 us (4.4
// TB/s) in blocks of 64.  Blocks of more values than a wave's lanes keep are shared
// by eight waves (in blocks of 512 (4, 8, 2048, 128) took one wave 66.4 us, eight
// 12.4; of 4096 tokens 420 and 51.8), and so are those of head dims that are no
// multiple of 8, which go value by value ((4, 8, 2041, 100) 43.6 us and 30.0); past
// what eight waves keep, the values are read twice.
#include <algorithm>

#include "kv_cache.h"

namespace ntops {
namespace {

struct StoreArgs {
  const void* x[2];      // key, value: (B, H, S, D)
  uint8_t* cache[2];     // (B, H, C, D)
  float* scale[2];       // (B, H, blocks)
  int64_t xs[2][3], cs[2][3], ss[2][2];  // strides: batch, head, token; batch, head
  const void* positions;
  const void* lengths;
  int positions_dtype, lengths_dtype;
  int64_t position;      // of every sequence, without positions
  int64_t B, H, S, C;
  int D, shift;          // block = 1 << shift tokens
  int64_t units;         // blocks that a sequence's tokens can lie in: the grid is (units, H, B), a wave for keys and one for values
};

constexpr int kSlots = 16;  // packs of 8 values a lane keeps
constexpr int kWide = 8;    // waves that share a block of more values than a wave's lanes keep

__device__ __forceinline__ float least_scale(uint32_t top) {
  const int e = static_cast<int>(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __builtin_bit_cast(float, static_cast<uint32_t>(max(e, 1)) << 23);
}

// x / s (a power of two: by its exact inverse).
struct Divide {
  float s, inv;
  bool pow2;
  __device__ __forceinline__ explicit Divide(float scale) : s(scale), inv(1.f / scale) {
    const uint32_t b = __builtin_bit_cast(uint32_t, scale);
    pow2 = (b & 0x7fffffu) == 0 && b >= (1u << 23) && b <= (253u << 23);
  }
  __device__ __forceinline__ float operator()(float x) const { return pow2 ? x * inv : x / s; }
};

// What the lanes of W waves do next: slot l, l + 64 W, .. of rows of `per` slots.
template <int W>
struct Walk {
  int row, col, per, drow, dcol;
  __device__ __forceinline__ Walk(int first, int per_row) : per(per_row) {
    row = first / per;
    col = first - row * per;
    drow = 64 * W / per;
    dcol = 64 * W - drow * per;
  }
  __device__ __forceinline__ void next() {
    row += drow;
    col += dcol;
    if (col >= per) {
      col -= per;
      ++row;
    }
  }
};

// Where a block's tokens lie.  W 1: keys in one wave, values in another; else the
// W waves take the values of a block of tokens together.
template <int W>
struct Unit {
  int which, lane;
  int64_t b, h, j;         // sequence, head, block
  int64_t start, p0, p1;   // position of the sequence's first token; positions of the block's new tokens
  int64_t first;           // of the block
  __device__ __forceinline__ bool find(const StoreArgs& a) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    which = W == 1 ? wave : blockIdx.x & 1;
    lane = W == 1 ? threadIdx.x & 63 : threadIdx.x;
    h = blockIdx.y;
    b = blockIdx.z;
    start = max(-a.S, min(a.C, index_at(a.positions, a.positions_dtype, b, a.position)));
    const int64_t count = max(int64_t(0), min(a.S, index_at(a.lengths, a.lengths_dtype, b, a.S)));
    const int64_t lo = max(int64_t(0), start), hi = min(a.C, start + count);
    j = (lo >> a.shift) + (W == 1 ? blockIdx.x : blockIdx.x >> 1);
    first = j << a.shift;
    p0 = max(lo, first);
    p1 = min(hi, first + (int64_t(1) << a.shift));
    return p0 < p1;
  }
};

__device__ __forceinline__ uint32_t wave_max_bits(uint32_t v) {
  // (bits of a non-negative float: the float's order)
  return __builtin_bit_cast(uint32_t, wave_max(__builtin_bit_cast(float, v)));
}

// The largest of all the lanes of a block of tokens (and what each has read of the
// cache before, it has).
template <int W>
__device__ __forceinline__ uint32_t group_max_bits(uint32_t v) {
  v = wave_max_bits(v);
  if constexpr (W > 1) {
    __shared__ uint32_t most[W];
    __syncthreads();  // (an earlier call's reads are over)
    if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = v;
    __syncthreads();
    for (int w = 0; w < W; ++w) v = max(v, most[w]);
  }
  return v;
}

__device__ __forceinline__ void grow(uint32_t& top, float v) {
  const uint32_t m = __builtin_bit_cast(uint32_t, v) & 0x7fffffffu;
  top = max(top, m < 0x7f800000u ? m : 0u);
}

// Largest |x| so far, of 2 16-bit values in a register or of one fp32, as its bits
// (a NaN's above an infinity's above any number's).
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void grow_word(u16x2& top, uint32_t w, _Float16) {
  top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w & 0x7fff7fffu));
}
__device__ __forceinline__ void grow_word(u16x2& top, uint32_t w, __bf16) { grow_word(top, w, _Float16{}); }
__device__ __forceinline__ void grow_word(uint32_t& top, uint32_t w, float) { top = max(top, w & 0x7fffffffu); }
template <typename T>
__device__ __forceinline__ uint32_t top_bits(u16x2 t) {  // as fp32 bits
  const uint16_t m = max(t.x, t.y);
  return __builtin_bit_cast(uint32_t, static_cast<float>(__builtin_bit_cast(T, m)));
}
template <typename T>
__device__ __forceinline__ uint32_t top_bits(uint32_t t) { return t; }

// 8 finite values over a power of two, at most 448 of it, to e4m3.
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
template <typename T>
__device__ __forceinline__ u32x2 scaled_e4m3(const Pack16<T> (&v)[sizeof(T) / 2], float scale) {
  u32x2 c;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    s16x2 w = {0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int e = 4 * i + 2 * h;
      const T x = v[e / Pack16<T>::N].v[e % Pack16<T>::N], y = v[e / Pack16<T>::N].v[e % Pack16<T>::N + 1];
      if constexpr (std::is_same<T, __bf16>::value)
        w = h ? __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, bf16x2{x, y}, scale, true)
              : __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, bf16x2{x, y}, scale, false);
      else if constexpr (std::is_same<T, _Float16>::value)
        w = h ? __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w, f16x2{x, y}, scale, true)
              : __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w, f16x2{x, y}, scale, false);
      else
        w = h ? __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x, y, scale, true)
              : __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x, y, scale, false);
    }
    c[i] = __builtin_bit_cast(uint32_t, w);
  }
  return c;
}

// 8 values at a time: head dim a multiple of 8, aligned rows, a block's rows within
// 31-bit byte offsets.  Buffer loads and stores, which end at the block's last
// value, so that no branch stands between a lane's loads.
template <typename T, int W>
__global__ __launch_bounds__(W == 1 ? 128 : 64 * W) void k_store_kv_cache(StoreArgs a) {
  constexpr int ES = sizeof(T);
  using Walk = Walk<W>;
  Unit<W> u;
  if (!u.find(a)) return;
  const int lane = u.lane;
  const int per = a.D / 8;
  const int rows = static_cast<int>(u.p1 - u.p0), slots = rows * per;
  const T* x = static_cast<const T*>(a.x[u.which]) + u.b * a.xs[u.which][0] + u.h * a.xs[u.which][1] +
               (u.p0 - u.start) * a.xs[u.which][2];
  uint8_t* c = a.cache[u.which] + u.b * a.cs[u.which][0] + u.h * a.cs[u.which][1] + u.p0 * a.cs[u.which][2];
  float* sp = a.scale[u.which] + u.b * a.ss[u.which][0] + u.h * a.ss[u.which][1] + u.j;
  const uint32_t xld = static_cast<uint32_t>(a.xs[u.which][2] * ES), cld = static_cast<uint32_t>(a.cs[u.which][2]);
  const __amdgpu_buffer_rsrc_t rx = buffer_rsrc_uniform(x, (rows - 1) * xld + a.D * ES);
  const __amdgpu_buffer_rsrc_t rc = buffer_rsrc_uniform(c, (rows - 1) * cld + a.D);
  const auto load = [&](const Walk& w, bool in, Pack16<T> (&v)[ES / 2]) {
    const uint32_t at = in ? w.row * xld + w.col * (8 * ES) : kOOB;
#pragma unroll
    for (int k = 0; k < ES / 2; ++k)
      v[k] = __builtin_bit_cast(Pack16<T>, __builtin_amdgcn_raw_buffer_load_b128(rx, at, k * 16, 0));
  };
  const auto value = [](const Pack16<T> (&v)[ES / 2], int e) { return static_cast<float>(v[e / Pack16<T>::N].v[e % Pack16<T>::N]); };
  Pack16<T> v[kSlots][ES / 2];
  const float old = u.p0 > u.first ? *sp : 0.f;
  {
    Walk w(lane, per);
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      load(w, i * (64 * W) + lane < slots, v[i]);
      w.next();
    }
  }
  const auto words = [](const Pack16<T> (&y)[ES / 2], auto& t) {
#pragma unroll
    for (int k = 0; k < ES / 2; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) grow_word(t, __builtin_bit_cast(u32x4, y[k])[e], T{});
  };
  std::conditional_t<ES == 2, u16x2, uint32_t> most{};
#pragma unroll
  for (int i = 0; i < kSlots; ++i) words(v[i], most);  // (slots past the end read as zero)
  for (Walk w(lane + kSlots * 64 * W, per); w.row < rows; w.next()) {
    Pack16<T> y[ES / 2];
    load(w, true, y);
    words(y, most);
  }
  uint32_t top = group_max_bits<W>(top_bits<T>(most));
  const bool finite = top < 0x7f800000u;
  if (!finite) {  // once more, over the finite values
    top = 0;
    for (Walk w(lane, per); w.row < rows; w.next()) {
      Pack16<T> y[ES / 2];
      load(w, true, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) grow(top, value(y, e));
    }
    top = group_max_bits<W>(top);
  }
  const float fits = least_scale(top);
  const bool keeps = old > fits;
  const float scale = keeps ? old : fits;
  const Divide by(scale);
  if (finite && by.pow2) {
    Walk w(lane, per);
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      if (i * (64 * W) < slots)
        __builtin_amdgcn_raw_buffer_store_b64(scaled_e4m3<T>(v[i], scale), rc, i * (64 * W) + lane < slots ? w.row * cld + w.col * 8 : kOOB, 0, 0);
      w.next();
    }
    for (; w.row < rows; w.next()) {
      Pack16<T> y[ES / 2];
      load(w, true, y);
      __builtin_amdgcn_raw_buffer_store_b64(scaled_e4m3<T>(y, scale), rc, w.row * cld + w.col * 8, 0, 0);
    }
  } else {
    for (Walk w(lane, per); w.row < rows; w.next()) {
      Pack16<T> y[ES / 2];
      load(w, true, y);
      float r[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = by(value(y, e));
      __builtin_amdgcn_raw_buffer_store_b64(to_e4m3(r), rc, w.row * cld + w.col * 8, 0, 0);
    }
  }
  if (u.p0 > u.first && !keeps && old != fits) {
    const float ratio = old / fits;
    uint8_t* o = c - (u.p0 - u.first) * a.cs[u.which][2];
    const int before = static_cast<int>(u.p0 - u.first);
    for (Walk r(lane, per); r.row < before; r.next()) {
      u32x2* at = reinterpret_cast<u32x2*>(o + static_cast<int64_t>(r.row) * a.cs[u.which][2] + r.col * 8);
      float y[8];
      from_e4m3(*at, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] *= ratio;
      *at = to_e4m3(y);
    }
  }
  if (lane == 0) *sp = scale;
}

// One value at a time, for any head dim and alignment.
template <typename T, int W>
__global__ __launch_bounds__(W == 1 ? 128 : 64 * W) void k_store_kv_cache_any(StoreArgs a) {
  using Walk = Walk<W>;
  Unit<W> u;
  if (!u.find(a)) return;
  const int lane = u.lane;
  const int rows = static_cast<int>(u.p1 - u.p0);
  const int64_t xld = a.xs[u.which][2], cld = a.cs[u.which][2];
  const T* x = static_cast<const T*>(a.x[u.which]) + u.b * a.xs[u.which][0] + u.h * a.xs[u.which][1] + (u.p0 - u.start) * xld;
  uint8_t* c = a.cache[u.which] + u.b * a.cs[u.which][0] + u.h * a.cs[u.which][1] + u.p0 * cld;
  float* sp = a.scale[u.which] + u.b * a.ss[u.which][0] + u.h * a.ss[u.which][1] + u.j;
  const auto code = [](float v) { return static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(v, 0.f, 0, false)); };
  const float old = u.p0 > u.first ? *sp : 0.f;
  uint32_t top = 0;
  for (Walk w(lane, a.D); w.row < rows; w.next()) grow(top, static_cast<float>(x[w.row * xld + w.col]));
  const float fits = least_scale(group_max_bits<W>(top));
  const bool keeps = old > fits;
  const float scale = keeps ? old : fits;
  const Divide by(scale);
  for (Walk w(lane, a.D); w.row < rows; w.next()) c[w.row * cld + w.col] = code(by(static_cast<float>(x[w.row * xld + w.col])));
  if (u.p0 > u.first && !keeps && old != fits) {
    const float ratio = old / fits;
    uint8_t* o = c - (u.p0 - u.first) * cld;
    const int before = static_cast<int>(u.p0 - u.first);
    for (Walk w(lane, a.D); w.row < before; w.next())
      o[w.row * cld + w.col] = code(__builtin_amdgcn_cvt_f32_fp8(o[w.row * cld + w.col], 0) * ratio);
  }
  if (lane == 0) *sp = scale;
}

}  // namespace
}  // namespace ntops

using namespace ntops;

extern "C" int ntops_store_kv_cache(int dtype, int64_t B, int64_t H, int64_t S, int64_t D, int64_t C, int64_t block,
                                    const void* key, const int64_t* key_strides, const void* value,
                                    const int64_t* value_strides, void* key_cache, const int64_t* key_cache_strides,
                                    void* value_cache, const int64_t* value_cache_strides, float* key_scale,
                                    const int64_t* key_scale_strides, float* value_scale,
                                    const int64_t* value_scale_strides, const void* positions, int positions_dtype,
                                    int64_t position, const void* lengths, int lengths_dtype, void* stream) {
  if (B < 0 || H < 0 || S < 0 || D < 0 || C < 0) return set_error(NTOPS_ERR_INVALID, "store_kv_cache: negative size");
  if (!block_ok(block)) return set_error(NTOPS_ERR_INVALID, "store_kv_cache: a block is a power of two of 16 to 2^24 tokens");
  if ((positions && !index_dtype(positions_dtype)) || (lengths && !index_dtype(lengths_dtype)))
    return set_error(NTOPS_ERR_INVALID, "store_kv_cache: positions and lengths are I32 or I64");
  return dispatch_float16_32(dtype, "store_kv_cache", [&](auto tag) -> int {
    using T = decltype(tag);
    if (B == 0 || H == 0 || S == 0 || D == 0 || C == 0) return NTOPS_OK;
    if (!key || !value || !key_cache || !value_cache || !key_scale || !value_scale || !key_strides || !value_strides ||
        !key_cache_strides || !value_cache_strides || !key_scale_strides || !value_scale_strides)
      return set_error(NTOPS_ERR_INVALID, "store_kv_cache: null pointer");
    if (key_cache == value_cache || key_scale == value_scale)
      return set_error(NTOPS_ERR_INVALID, "store_kv_cache: keys and values share their cache or its scales");
    if (D > 65536 || (D * std::min(block, S) > (int64_t(1) << 30)))
      return set_error(NTOPS_ERR_UNSUPPORTED, "store_kv_cache: blocks too large");
    StoreArgs a{};
    a.x[0] = key;
    a.x[1] = value;
    a.cache[0] = static_cast<uint8_t*>(key_cache);
    a.cache[1] = static_cast<uint8_t*>(value_cache);
    a.scale[0] = key_scale;
    a.scale[1] = value_scale;
    const int64_t* xs[2] = {key_strides, value_strides};
    const int64_t* cs[2] = {key_cache_strides, value_cache_strides};
    const int64_t* ss[2] = {key_scale_strides, value_scale_strides};
    bool vec = D % 8 == 0;
    for (int i = 0; i < 2; ++i) {
      if ((D > 1 && (xs[i][3] != 1 || cs[i][3] != 1)) || (C > block && ss[i][2] != 1))
        return set_error(NTOPS_ERR_INVALID, "store_kv_cache: the last dims need unit strides");
      for (int d = 0; d < 3; ++d) {
        a.xs[i][d] = xs[i][d];
        a.cs[i][d] = cs[i][d];
        vec = vec && xs[i][d] % (16 / static_cast<int>(sizeof(T))) == 0 && cs[i][d] % 8 == 0;
      }
      const int64_t most = std::min(block, S);
      vec = vec && xs[i][2] >= 0 && cs[i][2] >= 0 && most * xs[i][2] * static_cast<int64_t>(sizeof(T)) + D * 4 < 0x7fffffff &&
            most * cs[i][2] + D < 0x7fffffff;
      a.ss[i][0] = ss[i][0];
      a.ss[i][1] = ss[i][1];
      vec = vec && aligned16(a.x[i]) && (reinterpret_cast<uintptr_t>(a.cache[i]) & 7u) == 0;
    }
    a.positions = positions;
    a.positions_dtype = positions_dtype;
    a.position = position;
    a.lengths = lengths;
    a.lengths_dtype = lengths_dtype;
    a.B = B;
    a.H = H;
    a.S = S;
    a.C = C;
    a.D = static_cast<int>(D);
    a.shift = __builtin_ctzll(static_cast<unsigned long long>(block));
    a.units = std::min(ceil_div(S - 1, block) + 1, ceil_div(C, block));
    if (B > 65535 || H > 65535 || a.units > (1 << 24))
      return set_error(NTOPS_ERR_UNSUPPORTED, "store_kv_cache: over 65535 sequences or heads, or too many tokens");
    // a lane's registers hold kSlots packs; of single values a wave takes a few turns;
    // two of eight waves for each block have to be under the 2^32 threads of a grid's x
    // dimension (2^24 of one for keys and one for values are)
    const bool wide = std::min(block, S) * D > (vec ? kSlots * 64 * 8 : 8 * 64) && a.units * (2 * 64 * kWide) < (int64_t(1) << 32);
    const dim3 grid(static_cast<unsigned>(a.units * (wide ? 2 : 1)), static_cast<unsigned>(H), static_cast<unsigned>(B));
    const auto kern = vec ? (wide ? &k_store_kv_cache<T, kWide> : &k_store_kv_cache<T, 1>)
                          : (wide ? &k_store_kv_cache_any<T, kWide> : &k_store_kv_cache_any<T, 1>);
    hipLaunchKernelGGL(kern, grid, dim3(wide ? 64 * kWide : 128), 0, static_cast<hipStream_t>(stream), a);
    return check_launch("store_kv_cache");
  });
}
