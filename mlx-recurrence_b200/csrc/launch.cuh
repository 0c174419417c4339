// Dynamic shared memory beyond 48 KB, asked for once per kernel and device.
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

}  // namespace mr
