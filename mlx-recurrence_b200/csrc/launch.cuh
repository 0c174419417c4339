// Launch preliminaries: dynamic shared memory beyond 48 KB, asked for once per
// kernel and device, and the register count of kernels that redistribute theirs.
#pragma once

#include <atomic>

#include "common.cuh"

namespace mr {

template <auto Kernel> int allow_smem(int bytes, const char* what) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (e == cudaSuccess && (bit == 0 || !(done.load(std::memory_order_relaxed) & bit))) {
    e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(MR_E_LAUNCH, "%s: shared memory: %s", what, cudaGetErrorString(e));
  }
  return MR_OK;
}

// A kernel whose warpgroups pass registers on (setmaxnreg) needs the launch's own
// count to be `regs` a thread: with fewer, the increase would wait for ever.
template <auto Kernel> int expect_regs(int regs, const char* what) {
  static std::atomic<int> seen{0};
  int n = seen.load(std::memory_order_relaxed);
  if (n == 0) {
    cudaFuncAttributes a;
    const cudaError_t e = cudaFuncGetAttributes(&a, Kernel);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return set_error(MR_E_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
    }
    n = a.numRegs;
    seen.store(n, std::memory_order_relaxed);
  }
  if (n != regs) return set_error(MR_E_LAUNCH, "%s: built with %d registers a thread, not %d", what, n, regs);
  return MR_OK;
}

}  // namespace mr
