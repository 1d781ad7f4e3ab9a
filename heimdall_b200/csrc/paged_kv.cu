// A cache of keys and values in 8 bits: writing tokens into pages, and the page bookkeeping.
//
// Codes are e4m3 and a (page, KV head) has one scale, a power of two: with a floating-point code the scale only has to keep
// the block's values inside the code's range, its mantissa would buy nothing, and a power of two makes the division,
// the product and a change of scale exact (a code is rounded a second time only where a grown scale pushes it below
// 2^-6, the code's smallest normal number).
#include "bifrost_b200.h"
#include "capi_internal.h"
#include "common.cuh"
#include "launch_early.h"
#include "paged_kv.h"

#include <cuda_fp8.h>

namespace bfb {

// ------------------------------------------------------------------------------------------------ writing tokens
struct AppendArgs {
  PagePool p;
  const void* x[2];                     // keys, values
  long long sb[2], st[2], sh[2];
  const int32_t *slots, *cu;
  int B, t;
};

// smallest power of two s >= 2^-64 with amax / s <= 448 = 1.75 * 2^8, from amax's exponent and mantissa
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  if (u < 0x00800000u) e = -64;   // zero and subnormal values
  return __uint_as_float((uint32_t)(max(e, -64) + 127) << 23);
}
template <typename T>
__device__ __forceinline__ constexpr uint32_t inf16() { return sizeof(T) == 2 && __is_same(T, __half) ? 0x7c00u : 0x7f80u; }
__device__ __forceinline__ float pow2_inverse(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {   // saturating, NaN stays NaN
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}
__device__ __forceinline__ void from_e4m3x4(uint32_t u, float (&x)[4]) {
  uint32_t h0, h1;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h0) : "h"((uint16_t)u));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h1) : "h"((uint16_t)(u >> 16)));
  const float2 a = __half22float2(*reinterpret_cast<__half2*>(&h0)), b = __half22float2(*reinterpret_cast<__half2*>(&h1));
  x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
}

// One CTA per (sequence, page it writes, NH KV heads), keys and values; thread i takes 16 elements (chunk i % 16) of rows i / 16,
// i / 16 + threads / 16, ...: all of its loads are in flight before the block's maxima are known, so the new tokens are read once.  Bound
// by HBM (2 bytes in and 1 out per element) for prompts, where the way to the first load (cumulative lengths, slot and length, page) is
// what a CTA mostly waits for, so a CTA takes 64 KB where it can: with keys and values in CTAs of their own 32143 tokens of 4 heads took
// 47 us in pages of 64, now 34 (0.9 of HBM; with two CTAs per SM instead of three 46); pages of 16 and 32 with a head per CTA 44 and 43,
// with four and two 38 and 36; pages of 128 with 256 threads, which fill an SM's registers, 44, with 512 42.
// A decode step is bound by latency, 4 to 9 us, and takes a head per CTA (16 tokens: 3.8 us instead of 5.5).
template <int L>
struct AppendCfg {
  static constexpr int Threads = L == 128 ? 512 : 256, Ctas = L == 128 ? 1 : 3;
};
template <typename T, int L, int NH>
__global__ void __launch_bounds__(AppendCfg<L>::Threads, AppendCfg<L>::Ctas) paged_append_kernel(AppendArgs a) {
  constexpr int NT = AppendCfg<L>::Threads, RP = NT / 16, PASS = L / RP;     // rows per pass, heads, passes per head
  __shared__ float s_max[2][NH][NT / 32], s_told[2][NH];
  __shared__ int s_dup;
  let_next_start();
  wait_for_stream();
  const int tid = threadIdx.x, g0 = blockIdx.y * NH;
  int b, ord, tok0 = 0, n = a.t;
  if (a.cu) {
    // sequence b owns the items cu[b] / L + 2 b ...: at least as many as the pages that its tokens can touch.  Every warp cuts
    // the range that b is in into 32 pieces of `step` sequences at a time, which takes cu to ascend: where it does not, items of a
    // sequence go to another, whose tokens are then written more than once or not all, at positions of its own
    b = 0;
    int step = 1;
    while (32 * step < a.B) step *= 32;
#pragma unroll 1
    for (; step > 0; step >>= 5) {
      const int i = b + (tid & 31) * step;
      const unsigned ok = __ballot_sync(0xffffffffu, i < a.B && min(max(a.cu[min(i, a.B)], 0), a.t) / L + 2 * i <= (int)blockIdx.x);
      if (ok) b += (31 - __clz(ok)) * step;
    }
    tok0 = min(max(a.cu[b], 0), a.t);
    n = min(max(a.cu[b + 1], tok0), a.t) - tok0;
    ord = (int)blockIdx.x - (tok0 / L + 2 * b);
  } else {
    const int per = (a.t + L - 2) / L + 1;
    b = blockIdx.x / per;
    ord = blockIdx.x % per;
  }
  const int slot = a.slots ? a.slots[b] : b;
  if (n <= 0 || ord < 0 || slot < 0 || slot >= a.p.slots) return;
  if (a.slots) {   // a slot named twice: the first sequence writes
    if (tid == 0) s_dup = 0;
    __syncthreads();
    for (int i = tid; i < b; i += NT)
      if (a.slots[i] == slot) s_dup = 1;
    __syncthreads();
    if (s_dup) return;
  }
  const int end = a.p.lens[slot], start = max(end - n, 0);
  const int len = (int)min((long long)end, (long long)a.p.width * L);   // what the table has room for
  const int pi = start / L + ord;
  if (len <= 0 || (long long)pi * L >= len) return;
  const int page = a.p.table[(size_t)slot * a.p.width + pi];
  if (page < 0 || page >= a.p.pages) return;
  const int lo = max(start, pi * L), had = lo - pi * L, rows = min(len, (pi + 1) * L) - lo;
  const int skip = n - (end - lo);   // this page's first new token among the sequence's
  if (rows <= 0) return;
  const size_t pg = (size_t)page * a.p.heads + g0;
  const int chunk = (tid & 15) * 16, r0 = tid >> 4, heads = NH == 1 ? 1 : min(NH, a.p.heads - g0);
  // the scales so far, in registers for one head (from shared memory a page of 64 took 40 us instead of 34 of the prompts above)
  float told1[2] = {0.f, 0.f};
  if (NH > 1 && tid < 2 * NH) {
    const int kv = tid / NH, h = tid % NH;
    s_told[kv][h] = had && h < heads ? (kv ? a.p.vs : a.p.ks)[pg + h] : 0.f;
  }
  uint4 w[2][NH][PASS][2];
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const T* src = static_cast<const T*>(a.x[kv]) + g0 * a.sh[kv] + chunk +
                   (a.cu ? (long long)(tok0 + skip) * a.st[kv] : b * a.sb[kv] + (long long)skip * a.st[kv]);
    if (NH == 1) told1[kv] = had ? (kv ? a.p.vs : a.p.ks)[pg] : 0.f;
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int i = 0; i < PASS; ++i) {
        const int r = r0 + RP * i;
        w[kv][h][i][0] = w[kv][h][i][1] = make_uint4(0u, 0u, 0u, 0u);
        if (r < rows && h < heads) {
          const uint4* s = reinterpret_cast<const uint4*>(src + h * a.sh[kv] + r * a.st[kv]);
          w[kv][h][i][0] = __ldg(s);
          w[kv][h][i][1] = __ldg(s + 1);
        }
      }
  }
#pragma unroll
  for (int kv = 0; kv < 2; ++kv)
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      // the largest of the 16-bit patterns without their signs, which are in the order of the values; non-finite ones are left out in
      // a second look
      uint32_t m2 = 0u;
#pragma unroll
      for (int i = 0; i < PASS; ++i) {
        const uint32_t* u = reinterpret_cast<const uint32_t*>(w[kv][h][i]);
#pragma unroll
        for (int c = 0; c < 8; ++c) m2 = __vmaxu2(m2, u[c] & 0x7fff7fffu);
      }
      uint32_t top = max(m2 & 0xffffu, m2 >> 16);
      if (top >= inf16<T>()) {
        top = 0u;
#pragma unroll
        for (int i = 0; i < PASS; ++i) {
          const uint32_t* u = reinterpret_cast<const uint32_t*>(w[kv][h][i]);
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const uint32_t x = u[c] & 0x7fffu, y = (u[c] >> 16) & 0x7fffu;
            top = max(top, max(x < inf16<T>() ? x : 0u, y < inf16<T>() ? y : 0u));
          }
        }
      }
      const uint16_t t16 = (uint16_t)top;
      const float m = warp_max((float)*reinterpret_cast<const T*>(&t16));
      if ((tid & 31) == 0) s_max[kv][h][tid >> 5] = m;
    }
  __syncthreads();
  auto maximum = [&](int kv, int h) {
    float m = s_max[kv][h][0];
#pragma unroll
    for (int i = 1; i < NT / 32; ++i) m = fmaxf(m, s_max[kv][h][i]);
    return m;
  };
  const float amax1[2] = {NH == 1 ? maximum(0, 0) : 0.f, NH == 1 ? maximum(1, 0) : 0.f};
#pragma unroll
  for (int kv = 0; kv < 2; ++kv)
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      if (h >= heads) break;
      const float amax = NH == 1 ? amax1[kv] : maximum(kv, h), told = NH == 1 ? told1[kv] : s_told[kv][h];
      uint8_t* dst = (kv ? a.p.v : a.p.k) + (pg + h) * L * kPG_D + chunk;
      const float s = had ? fmaxf(scale_for(amax), told) : scale_for(amax);
      const float inv = pow2_inverse(s);
#pragma unroll
      for (int i = 0; i < PASS; ++i) {
        const int r = r0 + RP * i;
        if (r < rows) {
          const T* e = reinterpret_cast<const T*>(w[kv][h][i]);
          uint32_t c[4];
#pragma unroll
          for (int q = 0; q < 4; ++q)
            c[q] = e4m3x4((float)e[4 * q] * inv, (float)e[4 * q + 1] * inv, (float)e[4 * q + 2] * inv, (float)e[4 * q + 3] * inv);
          *reinterpret_cast<uint4*>(dst + (size_t)(had + r) * kPG_D) = make_uint4(c[0], c[1], c[2], c[3]);
        }
      }
      if (had && s > told) {   // the page's earlier tokens on the grown scale
        const float ratio = told * inv;
#pragma unroll 1
        for (int r = r0; r < had; r += RP) {
          uint4* at = reinterpret_cast<uint4*>(dst + (size_t)r * kPG_D);
          const uint4 o = *at;
          const uint32_t u[4] = {o.x, o.y, o.z, o.w};
          uint32_t c[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float x[4];
            from_e4m3x4(u[q], x);
            c[q] = e4m3x4(x[0] * ratio, x[1] * ratio, x[2] * ratio, x[3] * ratio);
          }
          *at = make_uint4(c[0], c[1], c[2], c[3]);
        }
      }
      if (tid == 0) (kv ? a.p.vs : a.p.ks)[pg + h] = s;
    }
}

// ------------------------------------------------------------------------------------------------ pages
// The host keeps the page allocator; what changes on the device goes along as kernel arguments (no copy of a list, no
// host memory that has to outlive the call), kPG_List integers a launch.
constexpr int kPG_List = 960;
struct PageList {
  int n;
  int v[kPG_List];
};

// `rows` rows of one head of one page, keys or values: 256 threads, all loads of a thread before its stores
template <int L>
__device__ __forceinline__ void copy_head(const uint8_t* src, uint8_t* dst, int rows) {
  constexpr int PER = L * kPG_D / 16 / 256;
  const int n = rows * (kPG_D / 16);
  uint4 w[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int c = threadIdx.x + 256 * i;
    if (c < n) w[i] = reinterpret_cast<const uint4*>(src)[c];
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int c = threadIdx.x + 256 * i;
    if (c < n) reinterpret_cast<uint4*>(dst)[c] = w[i];
  }
}

// blockIdx = (list entry, layer and head, keys or values)
template <int L>
__device__ __forceinline__ void copy_page(const PagePool& p, int from, int to, int rows) {
  const int layer = blockIdx.y / p.heads, g = blockIdx.y % p.heads;
  const size_t base = (size_t)layer * p.pages;
  const size_t s = (base + from) * p.heads + g, d = (base + to) * p.heads + g;
  uint8_t* x = blockIdx.z ? p.v : p.k;
  copy_head<L>(x + s * L * kPG_D, x + d * L * kPG_D, rows);
  if (threadIdx.x == 0) {
    float* sc = blockIdx.z ? p.vs : p.ks;
    sc[d] = sc[s];
  }
}

__global__ void __launch_bounds__(256) pages_release_kernel(PagePool p, const __grid_constant__ PageList list) {
  let_next_start();
  wait_for_stream();
  const int slot = list.v[blockIdx.x];
  for (int i = threadIdx.x; i < p.width; i += 256) p.table[(size_t)slot * p.width + i] = -1;
  if (threadIdx.x == 0) p.lens[slot] = 0;
}

template <int L>
__global__ void __launch_bounds__(256) pages_fork_kernel(PagePool p, const __grid_constant__ PageList list) {
  let_next_start();
  wait_for_stream();
  const int* f = list.v + 5 * blockIdx.x;
  const int from = f[0], to = f[1], len = f[2];
  if (blockIdx.y == 0 && blockIdx.z == 0) {
    for (int i = threadIdx.x; i < p.width; i += 256)
      p.table[(size_t)to * p.width + i] = f[4] >= 0 && i == len / L ? f[4] : p.table[(size_t)from * p.width + i];
    if (threadIdx.x == 0) p.lens[to] = len;
  }
  if (f[4] >= 0) copy_page<L>(p, f[3], f[4], len % L);
}

template <int L>
__global__ void __launch_bounds__(256) pages_move_kernel(PagePool p, const __grid_constant__ PageList list) {
  let_next_start();
  wait_for_stream();
  copy_page<L>(p, list.v[2 * blockIdx.x], list.v[2 * blockIdx.x + 1], L);
}

// table entries by binary search in the list's ascending sources
__global__ void __launch_bounds__(256) pages_remap_kernel(PagePool p, const __grid_constant__ PageList list) {
  let_next_start();
  wait_for_stream();
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (size_t)p.slots * p.width) return;
  const int page = p.table[i];
  int lo = 0, hi = list.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (list.v[2 * mid] < page) lo = mid + 1; else hi = mid;
  }
  if (list.v[2 * lo] == page) p.table[i] = list.v[2 * lo + 1];
}

__global__ void __launch_bounds__(256) pages_set_kernel(PagePool p, const __grid_constant__ PageList list) {
  let_next_start();
  wait_for_stream();
  for (int i = threadIdx.x; i < list.n; i += 256) {
    const long long at = list.v[2 * i], cells = (long long)p.slots * p.width;
    if (at < cells) p.table[at] = list.v[2 * i + 1]; else p.lens[at - cells] = list.v[2 * i + 1];
  }
}

int page_pool(const bf_page_pool* in, int layer, PagePool* out) {
  if (!in || !in->k_pages || !in->v_pages || !in->k_scale || !in->v_scale || !in->table || !in->lens)
    return BF_ERR_INVALID_ARGUMENT;
  if (in->layers <= 0 || in->pages <= 0 || in->heads <= 0 || in->slots <= 0 || in->width <= 0 || layer < 0 ||
      layer >= in->layers || (long long)in->slots * in->width + in->slots > 0x7fffffffLL)
    return BF_ERR_INVALID_ARGUMENT;
  if (in->dim != kPG_D || (in->page != 16 && in->page != 32 && in->page != 64 && in->page != 128))
    return BF_ERR_UNSUPPORTED;
  // rows of a layer are addressed with 32 bits by the tensor maps of the attention
  if ((long long)in->pages * in->heads * in->page > 0x7fffffffLL || (long long)in->layers * in->heads > 65535)
    return BF_ERR_UNSUPPORTED;
  if (!aligned16(in->k_pages) || !aligned16(in->v_pages)) return BF_ERR_ALIGNMENT;
  const size_t heads = (size_t)layer * in->pages * in->heads;
  out->k = static_cast<uint8_t*>(in->k_pages) + heads * in->page * kPG_D;
  out->v = static_cast<uint8_t*>(in->v_pages) + heads * in->page * kPG_D;
  out->ks = in->k_scale + heads;
  out->vs = in->v_scale + heads;
  out->table = in->table;
  out->lens = in->lens;
  out->layers = in->layers;
  out->pages = in->pages;
  out->heads = in->heads;
  out->page = in->page;
  out->slots = in->slots;
  out->width = in->width;
  return BF_OK;
}

}  // namespace bfb

using namespace bfb;

extern "C" {

int bf_paged_append(const bf_page_pool* pool, int layer, const void* k, long long k_sb, long long k_st, long long k_sh,
                    const void* v, long long v_sb, long long v_st, long long v_sh, const int32_t* slots,
                    const int32_t* cu, int B, int t, int dtype, bf_stream_t stream) {
  AppendArgs a{};
  int rc = page_pool(pool, layer, &a.p);
  if (rc) return rc;
  if (B < 0 || t < 0 || (!slots && B > a.p.slots)) return BF_ERR_INVALID_ARGUMENT;
  if (dtype != BF_BF16 && dtype != BF_F16) return BF_ERR_UNSUPPORTED;
  if (B == 0 || t == 0) return BF_OK;
  if (!k || !v) return BF_ERR_INVALID_ARGUMENT;
  if (!aligned16(k) || !aligned16(v) || ((k_sb | k_st | k_sh | v_sb | v_st | v_sh) & 7)) return BF_ERR_ALIGNMENT;
  const int L = a.p.page;
  const long long items = cu ? (long long)t / L + 2LL * B : (long long)B * ((t + L - 2) / L + 1);
  if (items > 0x7fffffffLL || a.p.heads > 65535) return BF_ERR_UNSUPPORTED;
  DeviceState st;
  if ((rc = device_state(&st))) return rc;
  a.x[0] = k; a.x[1] = v;
  a.sb[0] = k_sb; a.sb[1] = v_sb;
  a.st[0] = k_st; a.st[1] = v_st;
  a.sh[0] = k_sh; a.sh[1] = v_sh;
  a.slots = slots;
  a.cu = cu;
  a.B = B;
  a.t = t;
  const bool many = ((long long)(cu ? t : (long long)B * t) / L + B) * a.p.heads > 3LL * st.sm_count;
  auto go = [&](auto type) {
    using E = decltype(type);
    auto with = [&](auto kernel, int threads, int heads) {
      return launch_early(kernel, dim3((unsigned)items, (a.p.heads + heads - 1) / heads), threads, 0, stream, a);
    };
    if (L == 16 && many) return with(paged_append_kernel<E, 16, 4>, 256, 4);
    if (L == 16) return with(paged_append_kernel<E, 16, 1>, 256, 1);
    if (L == 32 && many) return with(paged_append_kernel<E, 32, 2>, 256, 2);
    if (L == 32) return with(paged_append_kernel<E, 32, 1>, 256, 1);
    if (L == 64) return with(paged_append_kernel<E, 64, 1>, 256, 1);
    return with(paged_append_kernel<E, 128, 1>, AppendCfg<128>::Threads, 1);
  };
  return dtype == BF_BF16 ? go(__nv_bfloat16()) : go(__half());
}

int bf_paged_pages(const bf_page_pool* pool, const int32_t* release, int n_release, const int32_t* fork, int n_fork,
                   const int32_t* move, int n_move, const int32_t* set, int n_set, bf_stream_t stream) {
  PagePool p{};
  int rc = page_pool(pool, 0, &p);
  if (rc) return rc;
  if (n_release < 0 || n_fork < 0 || n_move < 0 || n_set < 0 || (n_release && !release) || (n_fork && !fork) ||
      (n_move && !move) || (n_set && !set))
    return BF_ERR_INVALID_ARGUMENT;
  const long long cells = (long long)p.slots * p.width;
  auto slot_ok = [&](int s) { return s >= 0 && s < p.slots; };
  auto page_ok = [&](int q) { return q >= 0 && q < p.pages; };
  for (int i = 0; i < n_release; ++i)
    if (!slot_ok(release[i])) return BF_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < n_fork; ++i) {
    const int32_t* f = fork + 5 * i;
    if (!slot_ok(f[0]) || !slot_ok(f[1]) || f[2] < 0 || f[2] > (long long)p.width * p.page) return BF_ERR_INVALID_ARGUMENT;
    if (f[4] >= 0 && (!page_ok(f[3]) || !page_ok(f[4]) || f[3] == f[4])) return BF_ERR_INVALID_ARGUMENT;
  }
  for (int i = 0; i < n_move; ++i)
    if (!page_ok(move[2 * i]) || !page_ok(move[2 * i + 1]) || (i && move[2 * i] <= move[2 * i - 2]))
      return BF_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < n_set; ++i)
    if (set[2 * i] < 0 || set[2 * i] >= cells + p.slots) return BF_ERR_INVALID_ARGUMENT;
  DeviceState st;
  if ((rc = device_state(&st))) return rc;
  // every list in pieces of at most kPG_List integers
  auto pieces = [&](const int32_t* from, int n, int ints, auto launch) -> int {
    const int most = kPG_List / ints;
    for (int at = 0; at < n; at += most) {
      PageList l;
      l.n = n - at < most ? n - at : most;
      for (int i = 0; i < l.n * ints; ++i) l.v[i] = from[(size_t)at * ints + i];
      const int e = launch(l);
      if (e) return e;
    }
    return BF_OK;
  };
  const unsigned lh = (unsigned)(p.layers * p.heads);
  rc = pieces(release, n_release, 1, [&](const PageList& l) { return launch_early(pages_release_kernel, dim3(l.n), 256, 0, stream, p, l); });
  if (rc) return rc;
  rc = pieces(fork, n_fork, 5, [&](const PageList& l) {
    return launch_early(p.page == 16 ? pages_fork_kernel<16> : p.page == 32 ? pages_fork_kernel<32> : p.page == 64 ? pages_fork_kernel<64>
                        : pages_fork_kernel<128>, dim3(l.n, lh, 2), 256, 0, stream, p, l);
  });
  if (rc) return rc;
  rc = pieces(move, n_move, 2, [&](const PageList& l) {
    const int e = launch_early(p.page == 16 ? pages_move_kernel<16> : p.page == 32 ? pages_move_kernel<32> : p.page == 64 ? pages_move_kernel<64>
                               : pages_move_kernel<128>, dim3(l.n, lh, 2), 256, 0, stream, p, l);
    return e ? e : launch_early(pages_remap_kernel, dim3((unsigned)((cells + 255) / 256)), 256, 0, stream, p, l);
  });
  if (rc) return rc;
  return pieces(set, n_set, 2, [&](const PageList& l) { return launch_early(pages_set_kernel, dim3(1), 256, 0, stream, p, l); });
}

}  // extern "C"
