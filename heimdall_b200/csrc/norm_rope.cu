// Head norms and rotary positions of several axes in one pass over the query and key projections.
//
//   y = x rsqrt(mean x^2 + eps) (1 + w),  (y_f, y_{f+F}) turned by the angle p_{a(f)} inv_freq_f for f < F,
//   with a token's positions p_0, p_1, ... (time, height, width of an image's patch; in text all alike) and the axis a(f) of each
//   frequency.  y itself goes out too where the memory path reads it.
//
// What bounds it is HBM: 512 bytes read and 512 or 1024 written per (token, head).  The angles are the same for all heads of a token, so
// a CTA makes the sines and cosines of its tokens once, in shared memory; the product and its reduction to one turn are done in 64 bits (in
// fp32 an angle of position 100000 is off by up to 2^-8, as much as the output's rounding).  A warp takes four heads of one token at a
// time, with the next four on their way.  Lane l < F / 4 has the dims 4 l .. 4 l + 3 and their partners F further on, the other lanes eight dims that
// are not turned (cos 1, sin 0): no value changes lanes, at the price of 8-byte accesses.  The rotated heads are made from y in fp32, so
// each output is rounded once.
// The instructions of a head come next to HBM as a bound: with the partner's values by shuffles and 64-bit divisions for every four heads it
// took 75 us for 8191 tokens of 24 + 4 heads and 446 for 65536 without q and k, now 65 (5.4 TB/s) and 345 (5.5; sustained, at the board's power cap, 66 and 352 to 364).  Two heads at a time on three or
// four CTAs per SM, which costs spills, 72 to 80 and 394 to 426; 16 tokens per CTA 65 and 350.
#include "capi_internal.h"
#include "common.cuh"
#include "launch_early.h"

namespace bfb {

constexpr int kNR_D = 256;
constexpr int kNR_Heads = 4;       // heads per warp at a time
constexpr int kNR_Tokens = 32;     // most tokens per CTA

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

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
template <typename T>
__device__ __forceinline__ uint64_t widen(uint32_t u) {      // two 16-bit values as fp32
  const T* e = reinterpret_cast<const T*>(&u);
  return pair2((float)e[0], (float)e[1]);
}
template <typename T>
__device__ __forceinline__ uint32_t narrow(uint64_t x);
template <>
__device__ __forceinline__ uint32_t narrow<__nv_bfloat16>(uint64_t x) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo_hi(x, 0), lo_hi(x, 1));
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t narrow<__half>(uint64_t x) {
  return pack_half2(lo_hi(x, 0), lo_hi(x, 1));
}

template <typename T>
__global__ void __launch_bounds__(256, 2) norm_rope_kernel(NormRopeArgs a) {
  __shared__ __align__(16) float s_cos[kNR_Tokens][kNR_D / 2], s_sin[kNR_Tokens][kNR_D / 2];
  __shared__ long long s_at[kNR_Tokens][4];        // elements of q and k behind which a token's heads begin; its rows of q and k turned
  let_next_start();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  wait_for_stream();
  const long long n0 = (long long)blockIdx.x * a.tokens;
  const int tokens = (int)(a.BT - n0 < a.tokens ? a.BT - n0 : a.tokens), F = a.F;
  if (tid < tokens) {
    const long long b = (n0 + tid) / a.T, t = (n0 + tid) - b * a.T;
    s_at[tid][0] = b * a.q_sb + t * a.q_st;
    s_at[tid][1] = b * a.k_sb + t * a.k_st;
    s_at[tid][2] = b * a.H * a.T + t;
    s_at[tid][3] = b * a.G * a.T + t;
  }
  __syncthreads();
  // a warp's items: four heads of a token, j of the token's qn + kn groups of heads
  const int qn = (a.H + kNR_Heads - 1) / kNR_Heads, per = qn + (a.G + kNR_Heads - 1) / kNR_Heads;
  const bool turned = 4 * lane < F;
  const int d0 = turned ? 4 * lane : F + 4 * lane, d1 = turned ? F + 4 * lane : 128 + 4 * lane;      // dims d0 .. d0 + 3 and d1 .. d1 + 3
  uint2 raw[kNR_Heads][2];
  auto load = [&](int t, int j) {
    const bool isq = j < qn;
    const int h0 = (isq ? j : j - qn) * kNR_Heads, m = (isq ? a.H : a.G) - h0;
    const long long sh = isq ? a.q_sh : a.k_sh;
    const T* src = static_cast<const T*>(isq ? a.qg : a.kl) + s_at[t][isq ? 0 : 1] + h0 * sh;
#pragma unroll
    for (int i = 0; i < kNR_Heads; ++i) {
      raw[i][0] = raw[i][1] = make_uint2(0u, 0u);
      if (i < m) {
        raw[i][0] = __ldcs(reinterpret_cast<const uint2*>(src + d0));
        raw[i][1] = __ldcs(reinterpret_cast<const uint2*>(src + d1));
      }
      src += sh;
    }
  };
  int t = 0, j = warp;
  auto settle = [&](int& t, int& j) {
    while (j >= per) {
      j -= per;
      ++t;
    }
  };
  settle(t, j);
  if (t < tokens) load(t, j);
  for (int i = tid; i < tokens * F; i += 256) {
    const int k = i / F, f = i % F, ax = (a.axis[f >> 4] >> (2 * (f & 15))) & 3;
    const long long at = ax * a.BT + n0 + k;
    const double p = a.pos64 ? (double)static_cast<const int64_t*>(a.pos)[at] : (double)static_cast<const int32_t*>(a.pos)[at];
    const double turns = p * (double)a.inv_freq[f] * 0.15915494309189535;
    sincospif((float)(2. * (turns - rint(turns))), &s_sin[k][f], &s_cos[k][f]);
  }
  uint64_t wq[4], wk[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int d = (e < 2 ? d0 : d1) + 2 * (e & 1);
    wq[e] = pair2(1.f + a.q_w[d], 1.f + a.q_w[d + 1]);
    wk[e] = pair2(1.f + a.k_w[d], 1.f + a.k_w[d + 1]);
  }
  __syncthreads();
  float most = 0.f;                // of the warp's square sums
  while (t < tokens) {
    const bool isq = j < qn;
    const int h0 = (isq ? j : j - qn) * kNR_Heads, heads = isq ? a.H : a.G, m = heads - h0, now_t = t;
    uint2 now[kNR_Heads][2];
#pragma unroll
    for (int i = 0; i < kNR_Heads; ++i) {
      now[i][0] = raw[i][0];
      now[i][1] = raw[i][1];
    }
    j += 8;
    settle(t, j);
    if (t < tokens) load(t, j);
    uint64_t c0 = pair2(1.f, 1.f), c1 = c0, s0 = 0, s1 = 0;
    if (turned) {
      const float4 c = *reinterpret_cast<const float4*>(&s_cos[now_t][4 * lane]), s = *reinterpret_cast<const float4*>(&s_sin[now_t][4 * lane]);
      c0 = pair2(c.x, c.y);
      c1 = pair2(c.z, c.w);
      s0 = pair2(s.x, s.y);
      s1 = pair2(s.z, s.w);
    }
    const uint64_t minus = pair2(-1.f, -1.f), n0_ = mul2(s0, minus), n1_ = mul2(s1, minus);
    float ss[kNR_Heads];
#pragma unroll
    for (int i = 0; i < kNR_Heads; ++i) {
      uint64_t x = widen<T>(now[i][0].x), sum = mul2(x, x);
      x = widen<T>(now[i][0].y), sum = fma2(x, x, sum);
      x = widen<T>(now[i][1].x), sum = fma2(x, x, sum);
      x = widen<T>(now[i][1].y), sum = fma2(x, x, sum);
      ss[i] = lo_hi(sum, 0) + lo_hi(sum, 1);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < kNR_Heads; ++i) ss[i] += __shfl_xor_sync(0xffffffffu, ss[i], o);
    most = fmaxf(fmaxf(fmaxf(most, ss[0]), ss[1]), fmaxf(ss[2], ss[3]));
    T* plain = static_cast<T*>(isq ? a.q : a.k);
    if (plain) plain += ((n0 + now_t) * heads + h0) * kNR_D;
    T* rot = static_cast<T*>(isq ? a.qr : a.kr) + (s_at[now_t][isq ? 2 : 3] + (long long)h0 * a.T) * kNR_D;
#pragma unroll
    for (int i = 0; i < kNR_Heads; ++i) {
      const float inv = rsqrtf(ss[i] * (1.f / kNR_D) + a.eps);
      const uint64_t inv2 = pair2(inv, inv);
      uint64_t y[4] = {widen<T>(now[i][0].x), widen<T>(now[i][0].y), widen<T>(now[i][1].x), widen<T>(now[i][1].y)};
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = mul2(mul2(y[e], inv2), isq ? wq[e] : wk[e]);
      if (i < m) {
        if (plain) {
          __stcs(reinterpret_cast<uint2*>(plain + d0), make_uint2(narrow<T>(y[0]), narrow<T>(y[1])));
          __stcs(reinterpret_cast<uint2*>(plain + d1), make_uint2(narrow<T>(y[2]), narrow<T>(y[3])));
        }
        __stcs(reinterpret_cast<uint2*>(rot + d0), make_uint2(narrow<T>(fma2(y[2], n0_, mul2(y[0], c0))), narrow<T>(fma2(y[3], n1_, mul2(y[1], c1)))));
        __stcs(reinterpret_cast<uint2*>(rot + d1), make_uint2(narrow<T>(fma2(y[0], s0, mul2(y[2], c0))), narrow<T>(fma2(y[1], s1, mul2(y[3], c1)))));
      }
      if (plain) plain += kNR_D;
      rot += (long long)a.T * kNR_D;
    }
  }
  // An infinity (and no NaN) in a head makes its own dim NaN and the others 0, and 0 times that NaN has made NaN of dims that are not turned.  Those are y
  // itself: written once more, by the lane that has both.  (Told apart in every head, that takes 370 us for 65536 tokens without q and k, against 361, sustained.)
  if (most < INFINITY) return;
  t = 0;
  j = warp;
#pragma unroll 1
  for (settle(t, j); t < tokens; j += 8, settle(t, j)) {
    const bool isq = j < qn;
    const int h0 = (isq ? j : j - qn) * kNR_Heads, heads = isq ? a.H : a.G;
#pragma unroll 1
    for (int h = h0; h < min(h0 + kNR_Heads, heads); ++h) {
      const T* x = static_cast<const T*>(isq ? a.qg : a.kl) + s_at[t][isq ? 0 : 1] + h * (isq ? a.q_sh : a.k_sh);
      T* rot = static_cast<T*>(isq ? a.qr : a.kr) + (s_at[t][isq ? 2 : 3] + (long long)h * a.T) * kNR_D;
      const float* w = isq ? a.q_w : a.k_w;
      bool nan = false, inf = false;
      for (int e = 0; e < 8; ++e) {
        const float v = fabsf((float)x[(e < 4 ? d0 : d1) + (e & 3)]);
        nan = nan || v != v;
        inf = inf || v == INFINITY;
      }
      if (!__any_sync(0xffffffffu, nan) && inf && !turned)
        for (int e = 0; e < 8; ++e) {
          const int d = (e < 4 ? d0 : d1) + (e & 3);
          rot[d] = (T)((float)x[d] * 0.f * (1.f + w[d]));
        }
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
  const void* ptrs[] = {qg, kl, q, k, qr, kr};
  for (const void* p : ptrs)
    if (!aligned16(p)) return BF_ERR_ALIGNMENT;
  // these are read one at a time
  const auto off = [](const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; };
  if (off(q_norm_w, 4) || off(k_norm_w, 4) || off(inv_freq, 4) || off(pos, pos64 ? 8 : 4)) return BF_ERR_ALIGNMENT;
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
