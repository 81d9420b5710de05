// mbarriers with bounded waits and tensor maps, for the kernels that stream
// operands.
#pragma once

#include <cuda.h>

#include "model_ops.h"

namespace ndt {

// A tensor map of bytes with 128-byte swizzle (inner box: 128 bytes); zeros
// outside the tensor.  model_ops.cpp.
CUtensorMap byte_map(const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box);

constexpr long long kWaitLimit = 4000000000ll;  // SM clocks, two seconds or more

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok;
}
// A wait that ends: after some two seconds, or once another wait of this CTA has
// given up, it raises the flags and returns false.
__device__ __forceinline__ bool mbar_wait_slow(uint32_t bar, uint32_t parity, volatile int* gave_up, int* flag,
                                               long long limit = kWaitLimit) {
  const long long t0 = clock64();
  while (true) {
    for (int i = 0; i < 32; i++)
      if (mbar_try(bar, parity)) return true;
    if (*gave_up) return false;
    if (clock64() - t0 > limit) {
      *gave_up = 1;
      atomicExch_system(flag, 1);
      return false;
    }
  }
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* gave_up, int* flag) {
  if (mbar_try(bar, parity)) return true;
  return mbar_wait_slow(bar, parity, gave_up, flag);
}
// After a wait that gave up, by every thread of the CTA before its shared
// memory and TMEM go: a millisecond, in which the copies and matrix instructions
// in flight end (none is issued after a wait that gave up).
__device__ __forceinline__ void settle_in_flight() {
  for (int n = 0; n < 1000; n++) __nanosleep(1000);
}
// For a whole warp: all lanes go on, or none.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* gave_up, int* flag) {
  return __all_sync(~0u, mbar_wait(bar, parity, gave_up, flag));
}

}  // namespace ndt
