// Bounded wait whose only way out, besides the phase's completion, is its time limit: unlike mbar_wait it does not look
// at what other calls have recorded in the status word, so a kernel's waits do not depend on earlier errors.
#pragma once
#include "ptx.cuh"

namespace vxg {

static __device__ __noinline__ bool wait_phase_slow(uint64_t* bar, uint32_t parity, int* status, int code) {
  const uint64_t t0 = globaltimer();
  while (!mbar_try_wait_sleep(bar, parity, 20000u)) {
    if (globaltimer() - t0 > kWaitLimitNs) {
      atomicCAS(status, 0, code);
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, int* status, int code) {
  return mbar_try_wait(bar, parity) || wait_phase_slow(bar, parity, status, code);
}

}  // namespace vxg
