// Head norms and rotary positions of several axes in one pass over the query and key projections.
//
//   y = x rsqrt(mean x^2 + eps) (1 + w),  (y_f, y_{f+F}) turned by the angle p_{a(f)} inv_freq_f for f < F,
//   with a token's positions p_0, p_1, ... (time, height, width of an image's patch; in text all alike) and the axis a(f) of each
//   frequency.  y itself goes out too where the memory path reads it.
//
// What bounds it is HBM: 512 bytes read and 512 or 1024 written per (token, head).  The angles are the same for all heads of a token, so
// a CTA makes the sines and cosines of its tokens once, in shared memory; the product and its reduction by 2 pi are done in 64 bits (in
// fp32 an angle of position 100000 is off by up to 2^-8, as much as the output's rounding).  A warp takes four heads of one token at a
// time (lane l: dims 8 l .. 8 l + 7), so that enough loads are in flight; the rotation's partner dims are F / 8 lanes away.  The rotated
// heads are made from y in fp32, so each output is rounded once.
#include "capi_internal.h"
#include "common.cuh"
#include "launch_early.h"

namespace bfb {

constexpr int kNR_D = 256;
constexpr int kNR_Heads = 4;       // heads per warp at a time
constexpr int kNR_Tokens = 8;      // most tokens per CTA

struct NormRopeArgs {
  const void *qg, *kl;
  long long q_sb, q_st, q_sh, k_sb, k_st, k_sh;   // element strides
  const float *q_w, *k_w, *inv_freq;
  const void* pos;                                // [axes][B][T] int32 or int64
  uint32_t axis[8];                               // two bits per frequency
  int pos64, F, tokens;                           // tokens per CTA
  float eps;
  int T, H, G;
  long long BT;
  void *q, *k, *qr, *kr;
};

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (float)e[j];
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint4 u;
  T* e = reinterpret_cast<T*>(&u);
#pragma unroll
  for (int j = 0; j < 8; ++j) e[j] = (T)f[j];
  return u;
}

template <typename T>
__global__ void __launch_bounds__(256) norm_rope_kernel(NormRopeArgs a) {
  __shared__ float2 s_cs[kNR_Tokens][kNR_D / 2];
  let_next_start();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  wait_for_stream();
  const long long n0 = (long long)blockIdx.x * a.tokens;
  const int tokens = (int)(a.BT - n0 < a.tokens ? a.BT - n0 : a.tokens), F = a.F;
  for (int i = tid; i < tokens * F; i += 256) {
    const int t = i / F, f = i % F, ax = (a.axis[f >> 4] >> (2 * (f & 15))) & 3;
    const long long at = ax * a.BT + n0 + t;
    const double p = a.pos64 ? (double)static_cast<const int64_t*>(a.pos)[at] : (double)static_cast<const int32_t*>(a.pos)[at];
    const double ang = p * (double)a.inv_freq[f], turns = rint(ang * 0.15915494309189535);
    float sn, cs;
    sincosf((float)fma(turns, -6.283185307179586, ang), &sn, &cs);
    s_cs[t][f] = make_float2(cs, sn);
  }
  float wq[8], wk[8];
  {
    const float4* w = reinterpret_cast<const float4*>(a.q_w) + 2 * lane;
    const float4* v = reinterpret_cast<const float4*>(a.k_w) + 2 * lane;
    const float4 w0 = __ldg(w), w1 = __ldg(w + 1), v0 = __ldg(v), v1 = __ldg(v + 1);
    const float x[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w}, y[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      wq[e] = 1.f + x[e];
      wk[e] = 1.f + y[e];
    }
  }
  __syncthreads();
  const int qn = (a.H + kNR_Heads - 1) / kNR_Heads, kn = (a.G + kNR_Heads - 1) / kNR_Heads;
  const int off = F >> 3;                                   // the partner's distance in lanes
  const bool turned = 4 * lane < F, first = lane < off;     // 8 lane < 2 F
  const int partner = turned ? (first ? lane + off : lane - off) : lane;
  for (int it = warp; it < tokens * (qn + kn); it += 8) {
    const int t = it / (qn + kn), j = it % (qn + kn);
    const bool isq = j < qn;
    const int h0 = (isq ? j : j - qn) * kNR_Heads, heads = isq ? a.H : a.G, m = min(kNR_Heads, heads - h0);
    const long long n = n0 + t, b = n / a.T, tt = n % a.T;
    const T* src = static_cast<const T*>(isq ? a.qg : a.kl) + b * (isq ? a.q_sb : a.k_sb) + tt * (isq ? a.q_st : a.k_st) + 8 * lane;
    const long long sh = isq ? a.q_sh : a.k_sh;
    uint4 raw[kNR_Heads];
#pragma unroll
    for (int i = 0; i < kNR_Heads; ++i) raw[i] = i < m ? __ldcs(reinterpret_cast<const uint4*>(src + (h0 + i) * sh)) : make_uint4(0u, 0u, 0u, 0u);
    float2 cs[8];
    if (turned) {
      const float4* c = reinterpret_cast<const float4*>(&s_cs[t][8 * (first ? lane : lane - off)]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float4 x = c[e];
        cs[2 * e] = make_float2(x.x, first ? -x.y : x.y);
        cs[2 * e + 1] = make_float2(x.z, first ? -x.w : x.w);
      }
    }
    float ss[kNR_Heads];
#pragma unroll
    for (int i = 0; i < kNR_Heads; ++i) {
      float x[8];
      unpack8<T>(raw[i], x);
      ss[i] = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss[i] = fmaf(x[e], x[e], ss[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < kNR_Heads; ++i) ss[i] += __shfl_xor_sync(0xffffffffu, ss[i], o);
    T* plain = static_cast<T*>(isq ? a.q : a.k);
    T* rot = static_cast<T*>(isq ? a.qr : a.kr);
#pragma unroll
    for (int i = 0; i < kNR_Heads; ++i) {
      float x[8], o8[8];
      unpack8<T>(raw[i], x);
      const float inv = rsqrtf(ss[i] * (1.f / kNR_D) + a.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * (isq ? wq[e] : wk[e]);
      if (plain && i < m) __stcs(reinterpret_cast<uint4*>(plain + (n * heads + h0 + i) * kNR_D) + lane, pack8<T>(x));
#pragma unroll
      for (int e = 0; e < 8; ++e) o8[e] = __shfl_sync(0xffffffffu, x[e], partner);
      if (turned) {
        // first half: x cos - partner sin, second: x cos + partner sin (the sign is in cs)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = fmaf(o8[e], cs[e].y, x[e] * cs[e].x);
      }
      if (i < m) __stcs(reinterpret_cast<uint4*>(rot + ((b * heads + h0 + i) * a.T + tt) * kNR_D) + lane, pack8<T>(x));
    }
  }
}

}  // namespace bfb

using namespace bfb;

extern "C" int bf_norm_rope(const void* qg, long long q_sb, long long q_st, long long q_sh, const void* kl, long long k_sb, long long k_st,
                            long long k_sh, const float* q_norm_w, const float* k_norm_w, const float* inv_freq, int freqs,
                            const uint8_t* axes, int n_axes, const void* pos, int pos64, float eps, int B, int T, int H, int G, int D,
                            int dtype, void* q, void* k, void* qr, void* kr, bf_stream_t stream) {
  if (B < 0 || T < 0 || H <= 0 || G <= 0 || freqs < 0 || freqs > D / 2 || freqs % 8 || n_axes < 1 || n_axes > 4 || !(eps >= 0.f) ||
      (freqs > 0 && !axes) || !q != !k)
    return BF_ERR_INVALID_ARGUMENT;
  if (D != kNR_D || (dtype != BF_BF16 && dtype != BF_F16)) return BF_ERR_UNSUPPORTED;
  NormRopeArgs a{};
  for (int f = 0; f < freqs; ++f) {
    if (axes[f] >= n_axes) return BF_ERR_INVALID_ARGUMENT;
    a.axis[f >> 4] |= (uint32_t)axes[f] << (2 * (f & 15));
  }
  if (B == 0 || T == 0) return BF_OK;
  if (!qg || !kl || !q_norm_w || !k_norm_w || !qr || !kr || (freqs > 0 && (!inv_freq || !pos))) return BF_ERR_INVALID_ARGUMENT;
  const void* ptrs[] = {qg, kl, q_norm_w, k_norm_w, q, k, qr, kr};
  for (const void* p : ptrs)
    if (!aligned16(p)) return BF_ERR_ALIGNMENT;
  if ((q_sb | q_st | q_sh | k_sb | k_st | k_sh) & 7) return BF_ERR_ALIGNMENT;
  DeviceState st;
  const int rc = device_state(&st);
  if (rc) return rc;
  a.qg = qg; a.kl = kl;
  a.q_sb = q_sb; a.q_st = q_st; a.q_sh = q_sh;
  a.k_sb = k_sb; a.k_st = k_st; a.k_sh = k_sh;
  a.q_w = q_norm_w; a.k_w = k_norm_w; a.inv_freq = inv_freq;
  a.pos = pos; a.pos64 = pos64; a.F = freqs; a.eps = eps;
  a.T = T; a.H = H; a.G = G;
  a.BT = (long long)B * T;
  a.q = q; a.k = k; a.qr = qr; a.kr = kr;
  // tokens per CTA: the sines are made while nothing is loaded, so several CTAs per SM, each with a few tokens
  const long long fill = 8LL * st.sm_count;
  a.tokens = (int)(a.BT / fill < 1 ? 1 : a.BT / fill < kNR_Tokens ? a.BT / fill : kNR_Tokens);
  const long long ctas = (a.BT + a.tokens - 1) / a.tokens;
  if (ctas > 0x7fffffffLL) return BF_ERR_UNSUPPORTED;
  return dtype == BF_BF16 ? launch_early(norm_rope_kernel<__nv_bfloat16>, dim3((unsigned)ctas), 256, 0, stream, a)
                          : launch_early(norm_rope_kernel<__half>, dim3((unsigned)ctas), 256, 0, stream, a);
}
