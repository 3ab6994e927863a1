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

template <int N>
__device__ __forceinline__ void wait_vm() {
  wait_vmcnt<(N < 63 ? N : 63)>();
}

}  // namespace ntops
