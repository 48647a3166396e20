// Programmatic dependent launches.
#pragma once

#include "common.cuh"

namespace llattn {
namespace {

// Programmatic dependent launch: a kernel may start (set up its barriers, TMEM
// and tensor maps) while the one before it in the stream finishes; pdl_wait
// returns when everything before is complete and visible, so it comes before
// the first access to global memory; pdl_next lets the kernel after start. What a
// kernel before wrote is not read through __restrict__ or __ldg: the read-only path wants it
// unchanged from this kernel's start on, which is before the wait.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Launches a kernel that calls pdl_wait, in clusters of `cluster` CTAs.
template <typename... P, typename... A>
cudaError_t launch_pdl(void (*kernel)(P...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim = {(unsigned)cluster, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

}  // namespace
}  // namespace llattn
