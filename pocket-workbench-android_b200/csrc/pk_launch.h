// pk_launch.h -- launches of the drafted-decoding and serving kernels: programmatic (the
// next kernel in the stream may be scheduled before this one ends; every one
// waits for the one before it first, but the second over shared prefixes, see
// pk_cache_attn.cu), optionally in clusters.
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

namespace pk {

// Allows kernel f `smem` bytes of dynamic shared memory on the current device,
// once (the call costs as much as half a launch).
inline cudaError_t allow_smem(const void *f, int smem) {
  if (smem <= 48 * 1024) return cudaSuccess;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  // (kernel, device) pairs already allowed their most; a full table or a lost
  // race only costs the call again
  struct Done {
    std::atomic<const void *> f{nullptr};
    std::atomic<int> dev{-1}, smem{0};
  };
  static Done done[256];
  const size_t at = (reinterpret_cast<uintptr_t>(f) / 16 + (size_t)dev * 37) % 256;
  for (size_t n = 0; n < 8; n++) {
    Done &d = done[(at + n) % 256];
    if (d.f.load(std::memory_order_acquire) == f && d.dev.load(std::memory_order_relaxed) == dev && d.smem.load(std::memory_order_relaxed) >= smem)
      return cudaSuccess;
  }
  e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  for (size_t n = 0; n < 8; n++) {
    Done &d = done[(at + n) % 256];
    int none = -1;
    if (d.dev.compare_exchange_strong(none, dev, std::memory_order_relaxed)) {
      d.smem.store(smem, std::memory_order_relaxed);
      d.f.store(f, std::memory_order_release);
      break;
    }
  }
  return cudaSuccess;
}

// programmatic false: this kernel begins when all work before it in the stream is
// done and its writes are in memory (which those that follow programmatically then
// rely on before they wait, too).
template <class... KArgs, class... Args>
cudaError_t launch_as(bool programmatic, void (*kernel)(KArgs...), int cluster, dim3 grid, dim3 block, int smem, cudaStream_t st, Args... args) {
  const cudaError_t e = allow_smem(reinterpret_cast<const void *>(kernel), smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2] = {};
  cfg.attrs = at;
  if (programmatic) {
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    at[cfg.numAttrs].val.clusterDim.x = (unsigned)cluster;
    at[cfg.numAttrs].val.clusterDim.y = at[cfg.numAttrs].val.clusterDim.z = 1;
    cfg.numAttrs++;
  }
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}
template <class... KArgs, class... Args>
cudaError_t launch_cluster(void (*kernel)(KArgs...), int cluster, dim3 grid, dim3 block, int smem, cudaStream_t st, Args... args) {
  return launch_as(true, kernel, cluster, grid, block, smem, st, args...);
}
template <class... KArgs, class... Args>
cudaError_t launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, int smem, cudaStream_t st, Args... args) {
  return launch_cluster(kernel, 1, grid, block, smem, st, args...);
}

}  // namespace pk
