// Launches that overlap the previous kernel's end: a kernel launched here may be
// set up while its predecessor in the stream drains, and waits (prior_done)
// before it touches memory; it lets its successor do the same from its start. A
// layer's short kernels follow one another, so what overlaps is a good part of
// their time.
#pragma once

#include "common.cuh"

namespace scmp {

// All earlier kernels of the stream are complete and their writes visible. Every
// kernel launched with launch_overlapped calls it before its first access to
// global memory.
__device__ __forceinline__ void prior_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <class... P, class... A>
static cudaError_t launch_overlapped(void (*kern)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, int cluster, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  count_launch();
  return e;
}

}  // namespace scmp
