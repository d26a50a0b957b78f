// Launching a kernel so that its start overlaps the end of the one before it
// on the stream (programmatic dependent launch). A kernel launched this way
// calls after_previous() before it touches anything that an earlier kernel
// wrote or reads, and may call let_next_start() from then on; every kernel
// of such a sequence waits, so each has the whole sequence before it behind
// it. The first kernel of a sequence is launched plainly.
#pragma once

#include <cuda_runtime.h>

namespace ngdn2 {

__device__ __forceinline__ void after_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <class... P, class... A>
cudaError_t launch_next(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                        bool overlap, const A&... args) {
  cudaLaunchConfig_t c{};
  c.gridDim = grid;
  c.blockDim = block;
  c.dynamicSmemBytes = smem;
  c.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  c.attrs = at;
  c.numAttrs = overlap ? 1 : 0;
  return cudaLaunchKernelEx(&c, kernel, P(args)...);
}

// A plain launch of clusters of CTAs (1: none).
template <class... P, class... A>
cudaError_t launch_clusters(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                            int cluster, const A&... args) {
  cudaLaunchConfig_t c{};
  c.gridDim = grid;
  c.blockDim = block;
  c.dynamicSmemBytes = smem;
  c.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  c.attrs = at;
  c.numAttrs = cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&c, kernel, P(args)...);
}

}  // namespace ngdn2
