// Launch-side utilities of the persistent tensor-core kernels.
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "capi_util.h"
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

// Launches `clusters` clusters of `size` CTAs.  The kernel may start while the one
// before it in the stream is finishing (it sets up its barriers and tensor memory
// and then waits, see wait_for_previous_kernel()).
template <typename... Args>
mxb_status launch_cluster(const char* what, void (*kernel)(Args...), unsigned clusters, unsigned size,
                          unsigned threads, size_t smem, cudaStream_t s,
                          const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(clusters * size);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    set_error("%s: CUDA launch failed: %s", what, cudaGetErrorString(e));
    return MXB_ERR_CUDA;
  }
  return MXB_OK;
}

}  // namespace mxb
