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

// checks the descriptor and points at `layer`; BF_OK or the status to return
int page_pool(const bf_page_pool* in, int layer, PagePool* out);

}  // namespace bfb
