// Causal attention of packed prompts (sequences of different lengths in one call) with grouped query heads.
//
//   o_i = sum_j p_ij v_j,  p_i = softmax_j(scale q_i . k_j),  keys j <= i + nk - nq of the query's own sequence.
//
// One warp per (token, query head): lane l holds dims 8l .. 8l+7 of the query and of the output, the keys of the
// sequence pass one by one with the running maximum and sum of the softmax in registers.
#include "bifrost_b200.h"
#include "capi_internal.h"
#include "common.cuh"

namespace bfb {

constexpr int kPA_D = 256;

struct PromptArgs {
  const void *q, *k, *v;
  long long q_st, q_sh, k_st, k_sh, v_st, v_sh;
  const int32_t *cu_q, *cu_k;
  int n_seq, T, Tk, H, G;
  float c2;   // scale * log2(e)
  void* o;
  float* lse;
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
  const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (float)t[e];
}

template <typename T>
__global__ void __launch_bounds__(128) prompt_attn_kernel(PromptArgs a) {
  const int tok = blockIdx.x, h = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (h >= a.H) return;
  // the sequence of this token, the cumulative lengths clamped into [previous, T] and [previous, Tk]
  int q0 = 0, k0 = 0, k1 = 0, q1 = 0, found = 0;
  for (int b = 0; b < a.n_seq && !found; ++b) {
    q0 = b ? q1 : min(max(a.cu_q[0], 0), a.T);
    k0 = b ? k1 : min(max(a.cu_k[0], 0), a.Tk);
    q1 = min(max(a.cu_q[b + 1], q0), a.T);
    k1 = min(max(a.cu_k[b + 1], k0), a.Tk);
    found = tok >= q0 && tok < q1;
  }
  const int nk = found ? min(k1 - k0, tok - q0 + 1 + (k1 - k0) - (q1 - q0)) : 0;
  float q[8], acc[8] = {};
  load8(static_cast<const T*>(a.q) + tok * a.q_st + h * a.q_sh + 8 * lane, q);
  const int g = h / (a.H / a.G);
  const T* k = static_cast<const T*>(a.k) + k0 * a.k_st + g * a.k_sh + 8 * lane;
  const T* v = static_cast<const T*>(a.v) + k0 * a.v_st + g * a.v_sh + 8 * lane;
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j < nk; ++j) {
    float x[8], s = 0.f;
    load8(k + j * a.k_st, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(q[e], x[e], s);
    s = warp_sum(s) * a.c2;
    const float mn = fmaxf(m, s);
    const float w = mn == -INFINITY && s == -INFINITY ? 0.f : exp2f(s - mn), al = m == -INFINITY ? 0.f : exp2f(m - mn);
    load8(v + j * a.v_st, x);
    l = l * al + w;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = fmaf(acc[e], al, w * x[e]);
    m = mn;
  }
  T out[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) out[e] = (T)(l > 0.f || l != l ? acc[e] / l : 0.f);
  *reinterpret_cast<uint4*>(static_cast<T*>(a.o) + ((size_t)tok * a.H + h) * kPA_D + 8 * lane) = *reinterpret_cast<uint4*>(out);
  if (a.lse && lane == 0) a.lse[(size_t)h * a.T + tok] = l > 0.f || l != l ? (m + log2f(l)) * kLn2 : -INFINITY;
}

}  // namespace bfb

using namespace bfb;

extern "C" {

int bf_prompt_attn_fwd(const void* q, long long q_st, long long q_sh, const void* k, long long k_st, long long k_sh,
                       const void* v, long long v_st, long long v_sh, const int32_t* cu_q, const int32_t* cu_k,
                       int n_seq, int T, int Tk, int H, int G, int D, int dtype, float scale, void* o, float* lse,
                       bf_stream_t stream) {
  if (T < 0 || Tk < 0 || n_seq < 0 || H <= 0 || G <= 0 || H % G || !(scale > 0.f) || scale > 3e38f)
    return BF_ERR_INVALID_ARGUMENT;
  if (D != kPA_D || (dtype != BF_BF16 && dtype != BF_F16)) return BF_ERR_UNSUPPORTED;
  if (T == 0) return BF_OK;
  if (!q || !o || (Tk > 0 && (!k || !v)) || (n_seq > 0 && !cu_q)) return BF_ERR_INVALID_ARGUMENT;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || ((q_st | q_sh | k_st | k_sh | v_st | v_sh) & 7))
    return BF_ERR_ALIGNMENT;
  DeviceState st;
  int rc = device_state(&st);
  if (rc) return rc;
  PromptArgs a{q, k, v, q_st, q_sh, k_st, k_sh, v_st, v_sh, cu_q, cu_k ? cu_k : cu_q, n_seq, T, Tk, H, G,
               scale * kLog2e, o, lse};
  const dim3 grid(T, (H + 3) / 4);
  if (dtype == BF_BF16)
    prompt_attn_kernel<__nv_bfloat16><<<grid, 128, 0, stream>>>(a);
  else
    prompt_attn_kernel<__half><<<grid, 128, 0, stream>>>(a);
  return launch_status();
}

}  // extern "C"
