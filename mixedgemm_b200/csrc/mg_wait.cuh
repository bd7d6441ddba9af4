// Bounded waits of the tensor-core kernels.
#pragma once
#include "ptx_sm100.cuh"

namespace mg {

// Bounded mbarrier wait: true once the phase has completed.  When the limit expires the lane
// records `code`, raises the CTA's stop flag and returns false; from then on every wait of the CTA
// that does not find its phase complete at the first probe returns false at once.  A role whose
// wait failed issues no copy and no MMA any more and leaves its loops (an epilogue may walk its remaining
// tiles, storing nothing); the kernel then ends normally.
__device__ __forceinline__ bool wait_parity(uint32_t bar, uint32_t parity, volatile int* stop, int* status,
                                            long long limit, int code) {
  if (ptx::mbar_try_wait(bar, parity)) return true;
  long long t0 = 0;
  for (uint32_t spin = 0;; ++spin) {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    if ((spin & 63u) == 0) {
      if (*stop) return false;
      const long long now = clock64();
      if (spin == 0) t0 = now;
      if (now - t0 > limit) {
        *stop = 1;
        atomicOr(status, code);
        return false;
      }
    }
  }
}

// The same for a barrier whose phase is completed by other CTAs of the cluster.
__device__ __forceinline__ bool wait_parity_cluster(uint32_t bar, uint32_t parity, volatile int* stop, int* status,
                                                    long long limit, int code) {
  if (ptx::mbar_try_wait_cluster(bar, parity)) return true;
  long long t0 = 0;
  for (uint32_t spin = 0;; ++spin) {
    if (ptx::mbar_try_wait_cluster(bar, parity)) return true;
    if ((spin & 63u) == 0) {
      if (*stop) return false;
      const long long now = clock64();
      if (spin == 0) t0 = now;
      if (now - t0 > limit) {
        *stop = 1;
        atomicOr(status, code);
        return false;
      }
    }
  }
}

}  // namespace mg
