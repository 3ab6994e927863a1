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
// between the maximum and the rounding, nothing is shared, no barrier.  Blocks
// of more than kSlots * 64 * 8 values are read twice.
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
  int64_t units;         // blocks that a sequence's tokens can lie in
};

constexpr int kSlots = 16;  // packs of 8 values a lane keeps

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

// VEC: 8 values at a time (head dim a multiple of 8, aligned rows), else one.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void k_store_kv_cache(StoreArgs a) {
  constexpr int N = VEC ? 8 : 1;
  const int lane = threadIdx.x & 63;
  int64_t id = block_id() * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int which = static_cast<int>(id & 1);
  id >>= 1;
  const int64_t unit = id % a.units;
  id /= a.units;
  const int64_t h = id % a.H, b = id / a.H;
  if (b >= a.B) return;
  int64_t start = index_at(a.positions, a.positions_dtype, b, a.position);
  start = max(-a.S, min(a.C, start));
  const int64_t count = max(int64_t(0), min(a.S, index_at(a.lengths, a.lengths_dtype, b, a.S)));
  const int64_t lo = max(int64_t(0), start), hi = min(a.C, start + count);
  const int64_t j = (lo >> a.shift) + unit;
  const int64_t first = j << a.shift;  // of the block
  const int64_t p0 = max(lo, first), p1 = min(hi, first + (int64_t(1) << a.shift));
  if (p0 >= p1) return;

  const T* x = static_cast<const T*>(a.x[which]) + b * a.xs[which][0] + h * a.xs[which][1] + (p0 - start) * a.xs[which][2];
  uint8_t* c = a.cache[which] + b * a.cs[which][0] + h * a.cs[which][1] + p0 * a.cs[which][2];
  float* sp = a.scale[which] + b * a.ss[which][0] + h * a.ss[which][1] + j;
  const int per = a.D / N;  // slots of a token
  const int total = static_cast<int>(p1 - p0) * per;
  const auto load = [&](int s, float (&v)[8]) {
    const int t = s / per, d = (s - t * per) * N;
    const T* at = x + t * a.xs[which][2] + d;
    if constexpr (VEC) {
#pragma unroll
      for (int k = 0; k < static_cast<int>(sizeof(T)) / 2; ++k) {
        const Pack16<T> p = load16(at + k * Pack16<T>::N);
#pragma unroll
        for (int e = 0; e < Pack16<T>::N; ++e) v[k * Pack16<T>::N + e] = static_cast<float>(p.v[e]);
      }
    } else {
      v[0] = static_cast<float>(*at);
    }
  };
  uint32_t top = 0;
  const auto grow = [&](const float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const uint32_t m = __builtin_bit_cast(uint32_t, v[e]) & 0x7fffffffu;
      top = max(top, m < 0x7f800000u ? m : 0u);
    }
  };
  const auto store = [&](int s, const float (&v)[8], const Divide& by) {
    const int t = s / per, d = (s - t * per) * N;
    uint8_t* at = c + t * a.cs[which][2] + d;
    float r[8];
#pragma unroll
    for (int e = 0; e < N; ++e) r[e] = by(v[e]);
    if constexpr (VEC)
      *reinterpret_cast<u32x2*>(at) = to_e4m3(r);
    else
      *at = static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(r[0], 0.f, 0, false));
  };
  constexpr int kKept = VEC ? kSlots : 1;
  float v[kKept][8];
  const float old = p0 > first ? *sp : 0.f;
#pragma unroll
  for (int i = 0; i < kKept; ++i)
    if (i * 64 + lane < total) load(i * 64 + lane, v[i]);
#pragma unroll
  for (int i = 0; i < kKept; ++i)
    if (i * 64 + lane < total) grow(v[i]);
  for (int s = kKept * 64 + lane; s < total; s += 64) {
    float w[8];
    load(s, w);
    grow(w);
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), m, 64)));
  const float fits = least_scale(top);
  const bool keeps = old > fits;
  const float scale = keeps ? old : fits;
  const Divide by(scale);
#pragma unroll
  for (int i = 0; i < kKept; ++i)
    if (i * 64 + lane < total) store(i * 64 + lane, v[i], by);
  for (int s = kKept * 64 + lane; s < total; s += 64) {
    float w[8];
    load(s, w);
    store(s, w, by);
  }
  if (p0 > first && !keeps && old != fits) {
    const float ratio = old / fits;
    uint8_t* o = a.cache[which] + b * a.cs[which][0] + h * a.cs[which][1] + first * a.cs[which][2];
    const int before = static_cast<int>(p0 - first) * per;
    for (int s = lane; s < before; s += 64) {
      const int t = s / per, d = (s - t * per) * N;
      uint8_t* at = o + t * a.cs[which][2] + d;
      float w[8];
      if constexpr (VEC) {
        from_e4m3(*reinterpret_cast<const u32x2*>(at), w);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] *= ratio;
        *reinterpret_cast<u32x2*>(at) = to_e4m3(w);
      } else {
        w[0] = __builtin_amdgcn_cvt_f32_fp8(*at, 0) * ratio;
        *at = static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(w[0], 0.f, 0, false));
      }
    }
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
  if (!block_ok(block)) return set_error(NTOPS_ERR_INVALID, "store_kv_cache: a block is a power of two of at least 16 tokens");
  if ((positions && !index_dtype(positions_dtype)) || (lengths && !index_dtype(lengths_dtype)))
    return set_error(NTOPS_ERR_INVALID, "store_kv_cache: positions and lengths are I32 or I64");
  return dispatch_float16_32(dtype, "store_kv_cache", [&](auto tag) -> int {
    using T = decltype(tag);
    if (B == 0 || H == 0 || S == 0 || D == 0 || C == 0) return NTOPS_OK;
    if (!key || !value || !key_cache || !value_cache || !key_scale || !value_scale || !key_strides || !value_strides ||
        !key_cache_strides || !value_cache_strides || !key_scale_strides || !value_scale_strides)
      return set_error(NTOPS_ERR_INVALID, "store_kv_cache: null pointer");
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
    if (B > (int64_t(1) << 31) || H > (int64_t(1) << 31) || B * H > (int64_t(1) << 33) / a.units)
      return set_error(NTOPS_ERR_UNSUPPORTED, "store_kv_cache: too many blocks");
    const int64_t blocks = ceil_div(2 * B * H * a.units, 4);
    const auto kern = vec ? &k_store_kv_cache<T, true> : &k_store_kv_cache<T, false>;
    hipLaunchKernelGGL(kern, blocks_2d(blocks), dim3(256), 0, static_cast<hipStream_t>(stream), a);
    return check_launch("store_kv_cache");
  });
}
