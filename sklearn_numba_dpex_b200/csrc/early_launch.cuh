// Launches that may start before the kernel ahead of them on the stream has ended (programmatic dependent
// launch): set-up and launch latency overlap that kernel's end.  A kernel launched so reads and writes
// nothing in global memory before grid_dependency_wait(), which returns when everything that the kernels
// ahead wrote is there; to the stream the order of the kernels is what it always is.  What the kernels ahead may
// have written is not read-only for such a kernel's whole life, so its inputs are no `const T* __restrict__`,
// which the compiler reads through the non-coherent path.
#pragma once
#include "kmb_common.cuh"

namespace kmb {

// Waits until the grids ahead have ended and their writes can be seen.
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Lets the next grid's CTAs come in once all CTAs of this grid have called this or ended.
__device__ __forceinline__ void next_grid_may_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <typename... Params, typename... Args>
int launch_early(void (*kernel)(Params...), unsigned grid, int threads, size_t smem, int cluster, cudaStream_t s,
                 Args... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  KMB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, Params(args)...));
  return KMB_OK;
}

}  // namespace kmb
