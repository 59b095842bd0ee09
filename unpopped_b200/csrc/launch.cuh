// launch.cuh — a launch that may begin while the kernel before it in its stream ends (programmatic dependent launch).
#pragma once

#include <cuda_runtime.h>

namespace up {

// The kernel's CTAs may be placed as soon as every CTA of the kernel before has exited or called let_next_begin, so it calls
// after_previous() in every thread that touches global memory, and before it does. Its lifetime then begins before the kernels ahead have
// written: a CTA can be resident while the one before the one before still reads. So it reads what they may write by ordinary loads only. The
// non-coherent path (ld.global.nc, __ldg, and what the compiler makes of const __restrict__ pointers) is for memory that does not
// change in a kernel's lifetime; its loads may be served from lines that are already in L1 and be moved ahead of the wait.
template <typename... P, typename... A>
cudaError_t launch_early(void (*kernel)(P...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream, A&&... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(grid), config.blockDim = dim3(block), config.dynamicSmemBytes = smem, config.stream = stream;
  config.attrs = &attr, config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, static_cast<P>(args)...);
}

#ifdef __CUDACC__
// Waits until the kernels before in the stream have ended and what they wrote can be seen.
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
#endif

}  // namespace up
