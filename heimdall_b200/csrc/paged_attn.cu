// Attention of the last t tokens of each sequence over its 8-bit pages.
//
//   o = sum_j p_j sv_j c^v_j,  p = softmax_j(scale sk_j q . c^k_j)  over the positions j <= the token's own that have a page,
//   with the e4m3 codes c and the scales sk, sv of each (page, KV head).
//
// One warp per (sequence, token, query head): lane l holds dims 8l .. 8l+7.
#include "bifrost_b200.h"
#include "capi_internal.h"
#include "common.cuh"
#include "paged_kv.h"

namespace bfb {

struct PagedAttnArgs {
  PagePool p;
  const void* q;
  long long q_sb, q_st, q_sh;
  const int32_t* slots;
  int B, t, H;
  float c2;
  void* o;
  float* lse;
};

__device__ __forceinline__ void codes8(const uint8_t* at, float (&x)[8]) {
  const uint2 u = *reinterpret_cast<const uint2*>(at);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = i < 2 ? u.x : u.y;
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)(w >> (16 * (i & 1)))));
    const float2 f = __half22float2(*reinterpret_cast<__half2*>(&h));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

template <typename T>
__global__ void __launch_bounds__(128) paged_attn_kernel(PagedAttnArgs a) {
  const int b = blockIdx.x / a.t, i = blockIdx.x % a.t, h = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (h >= a.H) return;
  const int slot = a.slots ? a.slots[b] : b, g = h / (a.H / a.p.heads);
  const int len = slot >= 0 && slot < a.p.slots ? (int)min((long long)a.p.lens[slot], (long long)a.p.width * a.p.page) : 0;
  const int n = len - a.t + 1 + i;
  float q[8], acc[8] = {}, m = -INFINITY, l = 0.f;
  const T* qp = static_cast<const T*>(a.q) + b * a.q_sb + i * a.q_st + h * a.q_sh + 8 * lane;
#pragma unroll
  for (int e = 0; e < 8; ++e) q[e] = (float)qp[e];
  for (int j = 0; j < n; ++j) {
    const int page = a.p.table[(size_t)slot * a.p.width + j / a.p.page];
    if (page < 0 || page >= a.p.pages) continue;
    const size_t pg = (size_t)page * a.p.heads + g, at = (pg * a.p.page + j % a.p.page) * kPG_D + 8 * lane;
    float x[8], s = 0.f;
    codes8(a.p.k + at, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(q[e], x[e], s);
    s = warp_sum(s) * (a.c2 * a.p.ks[pg]);
    const float mn = fmaxf(m, s);
    const float w = exp2f(s - mn), al = m == -INFINITY ? 0.f : exp2f(m - mn), wv = w * a.p.vs[pg];
    codes8(a.p.v + at, x);
    l = l * al + w;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = fmaf(acc[e], al, wv * x[e]);
    m = mn;
  }
  T out[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) out[e] = (T)(l > 0.f || l != l ? acc[e] / l : 0.f);
  *reinterpret_cast<uint4*>(static_cast<T*>(a.o) + (((size_t)b * a.t + i) * a.H + h) * kPG_D + 8 * lane) = *reinterpret_cast<uint4*>(out);
  if (a.lse && lane == 0) a.lse[((size_t)b * a.H + h) * a.t + i] = l > 0.f || l != l ? (m + log2f(l)) * kLn2 : -INFINITY;
}

}  // namespace bfb

using namespace bfb;

extern "C" {

size_t bf_paged_attend_workspace(int B, int t, int H, int G, int D) {
  return B > 0 && t > 0 && H > 0 && G > 0 && D == kPG_D ? 16 : 0;
}

int bf_paged_attend(const bf_page_pool* pool, int layer, const void* q, long long q_sb, long long q_st, long long q_sh,
                    const int32_t* slots, int B, int t, int H, int dtype, float scale, void* o, float* lse, void* ws,
                    size_t ws_bytes, bf_stream_t stream) {
  PagedAttnArgs a{};
  int rc = page_pool(pool, layer, &a.p);
  if (rc) return rc;
  if (B < 0 || t < 0 || H <= 0 || H % a.p.heads || (!slots && B > a.p.slots) || !(scale > 0.f) || scale > 3e38f)
    return BF_ERR_INVALID_ARGUMENT;
  if ((dtype != BF_BF16 && dtype != BF_F16) || H / a.p.heads > 24) return BF_ERR_UNSUPPORTED;
  if (B == 0 || t == 0) return BF_OK;
  if (!q || !o) return BF_ERR_INVALID_ARGUMENT;
  if (!aligned16(q) || !aligned16(o) || ((q_sb | q_st | q_sh) & 7)) return BF_ERR_ALIGNMENT;
  if (ws_bytes < bf_paged_attend_workspace(B, t, H, a.p.heads, kPG_D) || !ws) return BF_ERR_WORKSPACE;
  DeviceState st;
  if ((rc = device_state(&st))) return rc;
  a.q = q;
  a.q_sb = q_sb; a.q_st = q_st; a.q_sh = q_sh;
  a.slots = slots;
  a.B = B; a.t = t; a.H = H;
  a.c2 = scale * kLog2e;
  a.o = o;
  a.lse = lse;
  const dim3 grid(B * t, (H + 3) / 4);
  if (dtype == BF_BF16)
    paged_attn_kernel<__nv_bfloat16><<<grid, 128, 0, stream>>>(a);
  else
    paged_attn_kernel<__half><<<grid, 128, 0, stream>>>(a);
  return launch_status();
}

}  // extern "C"
