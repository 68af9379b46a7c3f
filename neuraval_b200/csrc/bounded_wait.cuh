// Waits on shared-memory barriers that end.
#pragma once

#include <cstdint>

namespace nvs {

__device__ __forceinline__ bool wait_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok;
}
// Tries for `limit_ns` and, if nothing came, once more for as long: the clock also runs
// while another program has the GPU, and what a copy is behind by then is not its fault.
// The clock is read before the try, so each time ends with a try after its limit.
__device__ __noinline__ bool wait_long(uint32_t bar, uint32_t parity, uint32_t limit_ns) {
  for (int again = 0; again < 2; ++again) {
    uint64_t t0, t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
    do {
      asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
      if (wait_try(bar, parity)) return true;
    } while (t - t0 < limit_ns);
  }
  return false;
}
// False: it gave up, after twice `limit_ns`.
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, uint32_t limit_ns) {
  return wait_try(bar, parity) || wait_try(bar, parity) || wait_long(bar, parity, limit_ns);
}

}  // namespace nvs
