// Launch helper of the vocabulary-head and embedding kernels.
#pragma once
#include <cuda_runtime.h>

#include <atomic>

namespace dgx {

// Launches `kern` as a programmatic dependent of the kernel before it in the
// stream: its blocks may be placed, and run up to their griddepcontrol.wait,
// while that kernel drains. Every thread of a kernel launched this way executes
// the wait before its first access to global memory, so the stream's order
// holds. cluster > 1: thread-block
// clusters of that many CTAs.
template <typename... P, typename... A>
cudaError_t launch_dependent(void (*kern)(P...), dim3 blocks, int threads, int smem, int cluster, cudaStream_t s,
                             const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = blocks;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// Raises a kernel's dynamic shared-memory limit, once per device (`done` is
// the kernel's own set of devices).
template <typename K>
cudaError_t allow_smem(K kern, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaGetDevice(&dev);
  const unsigned long long bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

}  // namespace dgx
