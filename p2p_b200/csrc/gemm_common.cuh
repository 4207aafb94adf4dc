// gemm_common.cuh -- what the tensor-core products share: bounded barrier waits and the host's tensor-map
// encoder.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "kernels.h"
#include "sm100.cuh"

namespace p2p {

constexpr uint64_t kGemmWaitNs = 1000000000ull;

__device__ __forceinline__ bool gemm_wait(volatile int& abort_flag, uint64_t* bar,
                                          uint32_t parity, int32_t* err) {
  if (sm100::mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = sm100::globaltimer_ns();
  while (true) {
    if (sm100::mbar_try_wait(bar, parity)) return true;
    if (abort_flag) return false;
    if (sm100::globaltimer_ns() - t0 > kGemmWaitNs) {
      abort_flag = 1;
      atomicOr(err, kErrTimeout);
      return false;
    }
  }
}

// A wait of a warp: lane 0 polls, the verdict is shared.
__device__ __forceinline__ bool gemm_wait_warp(volatile int& abort_flag, uint64_t* bar,
                                               uint32_t parity, int32_t* err, int lane) {
  bool r = true;
  if (lane == 0) r = gemm_wait(abort_flag, bar, parity, err);
  return __shfl_sync(0xffffffffu, r ? 1 : 0, 0) != 0;
}

// A wait of a whole warp, every lane polling, with one verdict for all of them: the clock and the abort
// flag are looked at once in 64 polls only (a poll of one lane with a reading of the clock each, then a
// shuffle, took 1 us longer over the 16 stages of a small product).
__device__ __forceinline__ bool gemm_wait_all(volatile int& abort_flag, uint64_t* bar,
                                              uint32_t parity, int32_t* err) {
  uint64_t t0 = 0;
  for (uint32_t n = 1; !__all_sync(0xffffffffu, sm100::mbar_try_wait(bar, parity)); ++n) {
    if (n % 64) continue;
    const uint64_t now = sm100::globaltimer_ns();
    if (!t0) t0 = now;
    const bool late = now - t0 > kGemmWaitNs;
    if (__any_sync(0xffffffffu, late)) {
      if (!abort_flag) {
        abort_flag = 1;
        atomicOr(err, kErrTimeout);
      }
      return false;
    }
    if (__any_sync(0xffffffffu, abort_flag != 0)) return false;
  }
  return true;
}

inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

}  // namespace p2p
