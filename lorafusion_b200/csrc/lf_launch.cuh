// Kernel launches that may start before the kernel ahead of them on the stream has finished
// (programmatic dependent launch), and the two device-side halves of that hand-off.
#pragma once

#include <cuda_runtime.h>

namespace lf {

// The dependent launch on this stream, if it was launched with `pdl`, may start now: its CTAs take
// what resources this grid leaves and run up to their pdl_wait().
__device__ __forceinline__ void pdl_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// Blocks until the kernel ahead on the stream has finished and its writes are visible (returns at
// once in a launch without `pdl`).
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Launch `kernel` on `grid` blocks (clusters of `cluster` consecutive blocks along x when > 1).  With
// `pdl` the kernel may start while its predecessor on the stream still runs and must call
// pdl_wait() before it reads what that one writes.
template <typename... P, typename... A>
inline cudaError_t launch_cluster(void (*kernel)(P...), dim3 grid, unsigned cluster, dim3 block, size_t smem,
                                  cudaStream_t st, bool pdl, A&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}
template <typename... P, typename... A>
inline cudaError_t launch(void (*kernel)(P...), unsigned grid, unsigned block, size_t smem, cudaStream_t st, bool pdl,
                          A&&... args) {
  return launch_cluster(kernel, dim3(grid), 1, dim3(block), smem, st, pdl, args...);
}

}  // namespace lf
