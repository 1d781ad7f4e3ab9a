// What the attention kernels over 8-bit pages share (paged_attn.cu, paged_shared.cu).
#pragma once
#include <cuda.h>

#include "capi_internal.h"
#include "paged_kv.h"

namespace bfb {

constexpr int kPA_MaxCtas = 160;
constexpr int kPA_MaxGroup = 24;                     // query heads per KV head
constexpr int kPA_Part = kPG_D + 4;                  // floats of a row's partial: accumulator, maximum, sum, two to keep it aligned

// tensor maps of a layer's codes: boxes of one page and 128 dims
int paged_maps(const PagePool& p, CUtensorMap* kmap, CUtensorMap* vmap);

// Partials of the sequences' tails behind their first skip[b] pages: a row's (accumulator, maximum in the log2 domain, sum) in tail[row], or, where
// seg[b][chunk][KV head].x >= 0, cut over the CTAs seg.x .. seg.y: part[2 c + (c == seg.x)][row of the chunk].
struct PagedTail {
  int2* seg;
  float *part, *tail;
  int tc, nqc, rp;      // tokens per chunk, chunks, rows per partial
};
size_t paged_tail_workspace(int B, int t, int H, int G);
int paged_tail(const PagePool& p, const void* q, long long q_sb, long long q_st, long long q_sh, const int32_t* slots, const int32_t* skip, int B,
               int t, int H, int dtype, float scale, void* ws, const DeviceState& st, cudaStream_t stream, PagedTail* out);

}  // namespace bfb
