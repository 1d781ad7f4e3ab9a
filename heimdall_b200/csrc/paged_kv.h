// One layer of an 8-bit page pool as the kernels take it (paged_kv.cu, paged_attn.cu).
#pragma once
#include <stdint.h>

#include "../../include/bifrost_b200.h"

namespace bfb {

constexpr int kPG_D = 256;

struct PagePool {
  uint8_t *k, *v;      // [layers left][pages][heads][page][256] codes, from the layer in question
  float *ks, *vs;      // [layers left][pages][heads]
  int32_t* table;      // [slots][width]
  int32_t* lens;       // [slots]
  int layers, pages, heads, page, slots, width;
};

// A plan of shared pages (bf_page_table_share), int32: kPS_Head words (runs, sequences), then, n entries each, the sequences' slots, their order, their
// places in it, each sequence's last run (-1: none) and the pages that its runs cover, then n runs of kPS_Run words: first place, sequences, first
// page, page behind the last, the run before it on its sequences' way (-1: none), the number of those.
constexpr int kPS_Head = 4, kPS_Run = 6, kPS_Depth = 4;      // a sequence has at most kPS_Depth runs
inline long long plan_words(long long n) { return kPS_Head + 5 * n + kPS_Run * n; }

// checks the descriptor and points at `layer`; BF_OK or the status to return
int page_pool(const bf_page_pool* in, int layer, PagePool* out);

}  // namespace bfb
