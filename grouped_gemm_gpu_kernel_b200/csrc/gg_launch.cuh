// gg_launch.cuh -- launches of the mixture-of-experts kernels, which follow one another in a layer: each may be set
// up on the GPU while the kernel before it on the stream still runs (programmatic dependent launch), and
// touches global memory only once that one is done. The wait covers the kernel just before and no other, so the end
// of a kernel has to mean the end of all before it. An ordinary launch starts after them; a programmatic one, as
// these and the second launch of an executor with tile classes, waits before it ends (griddepcontrol.wait).
#pragma once

#include <cuda_runtime.h>

#include <utility>

namespace gg {

// The first statement of a chained kernel that touches global memory: lets the next kernel be set up, and waits
// for the one before.
__device__ __forceinline__ void chained_begin() {
  cudaTriggerProgrammaticLaunchCompletion();
  cudaGridDependencySynchronize();
}

// cudaErrorInvalidDevice where another device is current than the one that a handle's memory is on.
inline cudaError_t expect_device(int device) {
  int now = 0;
  const cudaError_t st = cudaGetDevice(&now);
  return st != cudaSuccess ? st : now == device ? cudaSuccess : cudaErrorInvalidDevice;
}

// cluster > 1: blocks of the grid's clusters.
template <typename... Params, typename... Args>
cudaError_t launch_chained(void (*kernel)(Params...), dim3 grid, unsigned threads, size_t smem, cudaStream_t stream, unsigned cluster,
                           Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attrs[2] = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim = {cluster, 1, 1};
  cfg.attrs = attrs;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

}  // namespace gg
