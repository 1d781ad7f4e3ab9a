// One layer of an 8-bit page pool as the kernels take it (paged_kv.cu, paged_attn.cu).
#pragma once
#include <stdint.h>

#include <cuda_runtime.h>

#include "../../include/bifrost_b200.h"
#include "capi_internal.h"

namespace bfb {

constexpr int kPG_D = 256;

struct PagePool {
  uint8_t *k, *v;      // [layers left][pages][heads][page][256] codes, from the layer in question
  float *ks, *vs;      // [layers left][pages][heads]
  int32_t* table;      // [slots][width]
  int32_t* lens;       // [slots]
  int layers, pages, heads, page, slots, width;
};

// The cache's kernels are short and follow one another, so each may start before the one before it in the stream has ended, does what
// needs none of its results, and then waits for them (wait_for_stream(), in every thread, before the first read or write of memory).
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

// checks the descriptor and points at `layer`; BF_OK or the status to return
int page_pool(const bf_page_pool* in, int layer, PagePool* out);

}  // namespace bfb
