// Launches whose start overlaps the end of the kernel before them in the stream.
#pragma once
#include <cuda_runtime.h>

#include "capi_internal.h"

namespace bfb {

// The serving kernels are short and follow one another, so each may start before the one before it in the stream has ended, does what
// needs none of its results, and then waits for them (wait_for_stream(), in every thread, before the first read or write of global memory).
// let_next_start(): from the moment that all of this kernel's CTAs run, the next kernel's may take what is left of the SMs.
template <typename... P, typename... A>
int launch_early(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream, const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e == cudaSuccess) return BF_OK;
  cudaGetLastError();
  return cuda_fail(e);
}
__device__ __forceinline__ void wait_for_stream() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace bfb
