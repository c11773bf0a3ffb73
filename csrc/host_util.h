// Host-side launch helpers shared by the kernel files.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

namespace omni {

// Raises the dynamic shared-memory limit of `Kernel` to `bytes` once per device.
// The attribute belongs to the device context, so a process that launches on a
// second GPU must set it there too; one bit per device (per kernel: the kernel
// is a template argument, so each kernel has its own mask) records that it was
// done.  Racing threads may both set it, which is harmless (the call is
// idempotent).
template <auto Kernel>
cudaError_t ensure_smem_attr(int bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? (uint64_t{1} << dev) : 0;
  if (bit != 0 && (done.load(std::memory_order_acquire) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && bit != 0) done.fetch_or(bit, std::memory_order_acq_rel);
  return e;
}

// A launch that may start while the one before it on the stream still runs (programmatic dependent
// launch): every thread of its kernel calls grid_dep_wait() before it exits, and before it reads or writes
// memory.  What the kernels before the one before it wrote may be read earlier only if that one calls
// grid_dep_launch() behind its own grid_dep_wait() (kv8_decode_kernel and its join).
template <class... Args>
cudaError_t launch_dependent_cluster(void (*kernel)(Args...), dim3 grid, int block, int smem, int cluster,
                                     cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <class... Args>
cudaError_t launch_dependent(void (*kernel)(Args...), dim3 grid, int block, int smem, cudaStream_t stream,
                             const Args&... args) {
  return launch_dependent_cluster(kernel, grid, block, smem, 1, stream, args...);
}

}  // namespace omni
