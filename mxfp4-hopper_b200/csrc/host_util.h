// Launch-side utilities of the persistent tensor-core kernels.
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "common.cuh"

namespace mxb {

// Dynamic shared memory above 48 KB has to be granted per kernel and device.
inline bool grant_smem(const void* kernel, size_t bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (done.load(std::memory_order_acquire) & bit) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) !=
      cudaSuccess)
    return false;
  done.fetch_or(bit, std::memory_order_release);
  return true;
}

inline int sm_count() {
  static std::atomic<int> cached{0};
  int n = cached.load(std::memory_order_relaxed);
  if (n == 0) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)
      return kSMs;
    cached.store(n, std::memory_order_relaxed);
  }
  return n;
}

}  // namespace mxb
