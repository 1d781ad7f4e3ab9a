// Launches whose start overlaps the end of the kernel before them in the stream.
#pragma once
#include <cuda_runtime.h>

#include "capi_internal.h"

namespace bfb {

// The serving kernels are short and follow one another, so each may start before the one before it in the stream has ended, does what
// needs none of its results, and then waits for them: wait_for_stream(), which returns when the kernel before has ended and all that it wrote is seen.
// let_next_start(): from the moment that all of this kernel's CTAs run, the next kernel's may take what is left of the SMs.
//
// The rule: wait_for_stream() in every thread, before its first read or write of global memory.  Such a kernel may let the next one start at any time.
// What the kernel before may have written is read by plain loads, unless the address itself comes from behind the wait: __ldg says that nobody writes it while this kernel
// runs, which begins before its wait, and leaves the compiler free to take it earlier.
//
// The exception, within one call: a kernel that reads before its wait what is older than the kernel before it.
//   * The kernel before it calls wait_then_let_next_start() in every thread, first of all: then all that is older has ended when the reader starts.  No
//     kernel may come between the two.
//   * What it reads early and any kernel or copy may have written since the last call (ids, lengths, plans, y) it reads past L1, with __ldcg or by a bulk copy, or
//     behind acquire_early() and a barrier.  That memory comes back at the same addresses from call to call, and only the wait promises that L1 holds
//     nothing of before.
//   * Some CTA of it waits, whatever the data, or it could end, and the kernel behind it start, while the one before it still runs.
// The pairs: paged_queries and paged_shared (plan, lengths); adapter_shrink_few and adapter_expand_few (ids, y); adapter_shrink and adapter_expand (what
// adapter_route wrote; y).
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
// For a kernel that reads early through L1, by one thread, a barrier before the others read: the value at p by an acquire at the scope of the GPU, behind which
// L1 holds nothing of before.
__device__ __forceinline__ int acquire_early(const int* p) {
  int x;
  asm volatile("ld.acquire.gpu.global.b32 %0, [%1];" : "=r"(x) : "l"(p) : "memory");
  return x;
}
// for a kernel whose next one reads early
__device__ __forceinline__ void wait_then_let_next_start() {
  wait_for_stream();
  let_next_start();
}

}  // namespace bfb
