// csrc/bounded_wait.cuh: a wait that nothing answers ends after its limit and says so; one
// that is answered, before it or while it waits, does not.
#include <cstdint>
#include <cstdio>

#include <cuda_runtime.h>

#include "bounded_wait.cuh"

struct Seen {
  int alone, late, met, after;
  uint64_t ns;
};

// One warp: lane 0 waits, in the last part while lane 16 arrives.
__global__ void waits(Seen* seen) {
  __shared__ uint64_t bars[2];
  const uint32_t bar = (uint32_t)__cvta_generic_to_shared(bars);
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i)
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar + 8 * i) : "memory");
    uint64_t t0, t1;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
    seen->alone = nvs::wait_for(bar, 0, 1000000u);  // nothing arrives
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t1));
    seen->ns = t1 - t0;
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
    seen->met = nvs::wait_for(bar, 0, 1000000u);
    seen->after = nvs::wait_long(bar, 0, 0u);  // no time at all, but it is there
  }
  __syncwarp();
  if (threadIdx.x == 16) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar + 8) : "memory");
  if (threadIdx.x == 0) seen->late = nvs::wait_for(bar + 8, 0, 1000000u);
}

int main() {
  Seen *d = nullptr, h{};
  if (cudaMalloc(&d, sizeof(Seen)) != cudaSuccess) return 2;
  waits<<<1, 32>>>(d);
  if (cudaMemcpy(&h, d, sizeof(Seen), cudaMemcpyDeviceToHost) != cudaSuccess) return 2;
  cudaFree(d);
  std::printf("alone %d in %llu ns, met %d, after %d, late %d\n", h.alone, (unsigned long long)h.ns, h.met, h.after, h.late);
  // twice the limit; the clock may move in steps of a microsecond, and the GPU may be shared
  return !h.alone && h.ns >= 1990000u && h.ns < 1000000000u && h.met && h.after && h.late ? 0 : 1;
}
