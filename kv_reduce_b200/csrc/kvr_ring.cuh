// mbarriers for kernels in which one warp fills a ring of
// shared-memory stages and others work through it (sm_100a).
#pragma once

#include "kvr_common.cuh"

namespace kvr {
namespace ring {

// A wait that runs out (which no input causes) is given up after about a
// second: every later wait of the thread returns at once, the loops end, and
// the caller makes its results NaN.
constexpr long long kWaitClocks = 2000000000ll;

__device__ __forceinline__ void bar_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_arrive_tx(uint32_t bar, int bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, int parity) {
  uint32_t ok;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
static __device__ __noinline__ bool bar_wait_long(uint32_t bar, int parity) {
  const long long begin = clock64();
  while (clock64() - begin < kWaitClocks)
    for (int i = 0; i < 64; ++i)
      if (bar_try(bar, parity)) return true;
  return false;
}
__device__ __forceinline__ void bar_wait(uint32_t bar, int parity, bool& failed) {
  if (bar_try(bar, parity) || failed) return;
  failed = !bar_wait_long(bar, parity);
}

}  // namespace ring
}  // namespace kvr
