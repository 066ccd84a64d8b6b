// Launches whose blocks may start while the kernel before them in the stream still runs (programmatic dependent launch): a
// kernel's set-up and the time between two kernels overlap with the end of the one before. What makes it safe: every
// thread calls wait_for_previous() before it reads or writes global memory, which returns once the kernels before have
// ended and their results are there. A kernel calls start_next() once it holds all that it needs of an SM's shared resources
// (its tensor memory above all: a block of the next kernel that took it first would wait for this kernel with it).
// A kernel before that never calls start_next(), any other library's, simply ends first.
#pragma once

#include <cuda_runtime.h>

namespace jla {

__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void start_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// kern<<<grid, block, smem, stream>>>(args...) that way; `cluster` CTAs along x to a cluster where it is not 0.
template <typename... Params, typename... Args>
inline cudaError_t launch_overlapped(void (*kern)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, int cluster,
                                     const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid, cfg.blockDim = block, cfg.dynamicSmemBytes = smem, cfg.stream = stream;
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr, cfg.numAttrs = cluster ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, Params(args)...);
}

}  // namespace jla
