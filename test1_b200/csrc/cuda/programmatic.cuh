// Launches whose prologue may overlap the end of the stream's previous kernel.
#pragma once

#include "common.cuh"

namespace t1 {

// The next kernel of the stream may start its prologue, and this one touches
// nothing of the previous kernel's before it has ended.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// A CTA's shared memory is open to its cluster once the CTA has started: each
// says so at its start, and waits for the others before the first access.
__device__ __forceinline__ void tell_started() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void wait_started() { asm volatile("barrier.cluster.wait;" ::: "memory"); }

// Every kernel launched so waits for the previous one before it touches memory.
template <class... P, class... A>
inline void launch_after(const char* what, void (*kern)(P...), dim3 grid, int threads, size_t smem, const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream();
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...);
  TORCH_CHECK(e == cudaSuccess, what, " launch failed: ", cudaGetErrorString(e));
  count_launch();
}

}  // namespace t1
