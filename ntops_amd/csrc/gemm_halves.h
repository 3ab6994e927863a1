// Shared by the persistent 256 x 256 product kernels (gemm_large.hip,
// gemm_mxfp4_large.hip): half tiles of 128 rows x 128 bytes of K in the LDS.
#pragma once

#include "mfma.h"

namespace ntops {

constexpr int kHalf = 128 * 64 * 2;      // bytes of a half tile: 128 rows / columns x 64 k

// The lane id through an empty asm: what is computed from it is computed where
// it is used, not hoisted out of the tile loops to sit in registers.
__device__ __forceinline__ int here(int lane) {
  asm volatile("" : "+v"(lane));
  return lane;
}

// Loads of an operand's half tiles: 2 instructions of 1 KiB per wave.
template <bool KMAJ>
struct HalfLoader {
  uint32_t voff[2];
  uint32_t kbytes;   // byte distance of consecutive k
  uint32_t lds_off;  // of this wave's first instruction

  __device__ __forceinline__ static int lane_k(int wave, int lane, int i) {
    const int q = wave * 2 + i;
    if constexpr (KMAJ) {
      const int row = q * 8 + lane / 8;
      return kslot<64>(row, lane % 8) * 8;
    } else {
      return q * 4 + lane / 16;
    }
  }
  __device__ __forceinline__ void init(int64_t ld, int wave, int lane) {
    lds_off = static_cast<uint32_t>(wave * 2048);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int q = wave * 2 + i;
      if constexpr (KMAJ)
        voff[i] = static_cast<uint32_t>((q * 8 + lane / 8) * ld * 2 + lane_k(wave, lane, i) * 2);
      else
        voff[i] = static_cast<uint32_t>((q * 4 + lane / 16) * ld * 2 + mnslot(q * 4 + lane / 16, lane % 16) * 16);
    }
    kbytes = static_cast<uint32_t>(KMAJ ? 2 : ld * 2);
  }
  // TAIL: the K tile at k0 may reach past K; its chunks there read as zero.
  template <bool TAIL>
  __device__ __forceinline__ void issue(u32x4 rsrc, uint32_t lds, int k0, int K, int wave, int lane) const {
    // (opaque, so that no sum of a fixed tile's is kept in a register)
    uint32_t koff = static_cast<uint32_t>(k0) * kbytes;
    asm volatile("" : "+s"(koff));
    const int l = TAIL ? here(lane) : 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t off = voff[i] + koff;
      if constexpr (TAIL) off = k0 + lane_k(wave, l, i) < K ? off : kOOB;
      dma16(rsrc, lds + lds_off + i * 1024, off);
    }
  }
};

template <int N>
__device__ __forceinline__ void wait_vm() {
  wait_vmcnt<(N < 63 ? N : 63)>();
}

}  // namespace ntops
