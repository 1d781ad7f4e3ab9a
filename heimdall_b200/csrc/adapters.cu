// Low-rank adapters of many requests beside one shared projection.
//
//   out_t = y_t + s_a B_a (A_a x_t)  with token t's adapter a (none: out_t = y_t);  A_a [r_a, d_in], B_a [d_out, r_a], ranks up to 128.
//
// What bounds it is HBM: a decode step reads the adapters in use once (2 r (d_in + d_out) bytes each) and little else; a prompt
// reads x and y once and writes out once, with 4 r (1 / d_out + 1 / d_in)-fold of that in products.  Two kernels, with h = A x between them in
// fp32 (r values per token): the adapters' two halves need a sum over d_in before anything of d_out can begin.
//
// Tokens are taken in groups of one adapter, so that an adapter is read once for many tokens:
//   * few tokens (up to kAD_Few, a decode step): groups of 16; every CTA compares all ids and finds its group.  No pass over the ids before, two launches.
//   * more: adapter_route_kernel sorts the tokens by adapter and lists groups of 128, one M = 128 tile of the tensor core (tcgen05).
// h = A x is split over d_in so that every SM has work; each split's sums are written on their own and added in order.  For many tokens h enters the
// second product as two 16-bit parts of its row's power-of-two scale (hi + lo, 16 bits of bf16, 22 of fp16), so that the only rounding of
// consequence is that of out; of few tokens those that share an adapter are taken so too, one alone keeps fp32.
// (With mma.sync in the place of tcgen05 both kernels of many tokens were bound by its rate, about 32 cycles per m16n8k16 and scheduler:
// 25480 tokens 6144 -> 5120, rank 64: 148 + 324 us.)
#include "capi_internal.h"
#include "common.cuh"
#include "launch_early.h"

namespace bfb {

// Tokens up to which every CTA looks for its group itself (a thread each).  At 256 tokens, 5120 -> 12288, that is the better way for any ids (us, against sorting
// them): one adapter of rank 16 15 (21), of rank 64 22 (25), 32 adapters 16 and 34 (44 and 54), 256 adapters 51 and 153 (222 and 244).
constexpr int kAD_Few = 256;
constexpr int kAD_MaxRank = 128;
constexpr int kAD_MaxAdapters = 4096;
constexpr int kAD_KFew = 1024;     // d_in per CTA for few tokens
constexpr int kAD_Group = 128;     // tokens per group of many: the M of a tcgen05 product

struct AdapterArgs {
  const void *x, *y;
  void* out;
  long long x_st, y_st, o_st;      // row strides, elements
  const int32_t* ids;
  const int32_t* row;              // [n + 1] the adapters' first rows in A, multiples of 16
  const float* scale;              // [n]
  const void *A, *B;               // A [row[n]][d_in]; B: adapter a's [d_out / 8][r_a / 8][8 columns][8 ranks] from element row[a] d_out on
  int n, T, d_in, d_out, rmax, splits, units;
  unsigned int* err;
  float* h;                        // few tokens: [splits][T][rmax]; many: two places per CTA of [kAD_Group][rmax rounded up to 32, 64, 128]
  void* parts;                     // h's two parts: a group's from its first place times 2 rmax on, [2][tokens / 8][r / 8][8 tokens][8 ranks]
  float* back;                     // by place: the scale that undoes theirs, times the adapter's
  int32_t* arrived;                // [groups] parts of h that are done
  int32_t* perm;                   // tokens by adapter, each adapter's from a multiple of 8 places on
  int4* groups;                    // (adapter or n, first of perm, tokens, -)
  int32_t* n_groups;               // all that out needs, and those of adapters
};

template <typename T>
constexpr int kIsBf16 = 0;
template <>
constexpr int kIsBf16<__nv_bfloat16> = 1;

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {      // 16 bytes into shared memory, zeros where there are none
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint4 ldg_stream(const uint4* p) { return __ldcs(p); }      // read once

// an adapter's number, n for none
__device__ __forceinline__ int adapter_of(const AdapterArgs& a, int id) { return id >= 0 && id < a.n ? id : a.n; }

// h as two parts: a power of two takes the row's largest to [2^13, 2^14), so that both keep all of their bits in fp16 too.  (A NaN is no maximum, but its
// row becomes NaN by itself.)
struct RowScale {
  int ex;
  __device__ __forceinline__ explicit RowScale(float big) { ex = big > 0.f && big < INFINITY ? min(max((int)(__float_as_uint(big) >> 23), 14), 253) : 140; }
  template <typename T>
  __device__ __forceinline__ void parts(float h, T& hi, T& lo) const {
    const float x = h * __uint_as_float((uint32_t)(267 - ex) << 23);
    hi = (T)x;
    lo = (T)(x - (float)hi);
  }
  __device__ __forceinline__ float back() const { return __uint_as_float((uint32_t)(ex - 13) << 23); }
};

// Few tokens: group x, the groups being 16 tokens of an adapter in their order, in the order of their first tokens: its tokens in s_tok.  Returns how
// many (0: there are fewer groups), and the adapter.  All 256 threads, thread = token.
struct FewSmem {
  int4 id[kAD_Few / 4];
  unsigned leads[8];
  int first, nth;
};
template <bool Early>        // before the wait: past L1
__device__ __forceinline__ int few_group(const AdapterArgs& a, int x, int* s_tok, FewSmem& s, int& id) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int mine = tid < a.T ? adapter_of(a, Early ? __ldcg(a.ids + tid) : a.ids[tid]) : -1;
  reinterpret_cast<int*>(s.id)[tid] = mine;
  if (tid == 0) s.first = -1;
  __syncthreads();
  int nth = 0;                 // of its adapter's tokens
  if (32 * warp < a.T) {
#pragma unroll 1
    for (int w = 0; w < warp; ++w)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int4 v = s.id[8 * w + i];
        nth += (v.x == mine) + (v.y == mine) + (v.z == mine) + (v.w == mine);
      }
    nth += __popc(__match_any_sync(0xffffffffu, mine) & ((1u << lane) - 1u));
  }
  const bool lead = mine >= 0 && (nth & 15) == 0;
  const unsigned leads = __ballot_sync(0xffffffffu, lead);
  if (lane == 0) s.leads[warp] = leads;
  __syncthreads();
  int before = __popc(leads & ((1u << lane) - 1u));
  for (int w = 0; w < warp; ++w) before += __popc(s.leads[w]);
  if (lead && before == x) {
    s.first = tid;
    s.nth = nth;
  }
  __syncthreads();
  if (s.first < 0) return 0;
  id = reinterpret_cast<const int*>(s.id)[s.first];
  const bool member = mine == id && nth >= s.nth && nth < s.nth + 16;
  if (member) s_tok[nth - s.nth] = tid;
  return __syncthreads_count(member);
}
// no more than so many groups
static int few_groups(int T, int n) { return min(T, T / 16 + min(n + 1, T)); }

// h of a few tokens: CTA = (group, part of d_in, 16 ranks).  A warp takes every eighth 32 values of d_in: lane (g, c) loads the 16 bytes at
// 8 c of x rows g and g + 8 and of ranks g and g + 8, the fragments of two steps (a sum over d_in may take its values in any order as
// long as both operands agree).
template <typename T>
__global__ void __launch_bounds__(256) adapter_shrink_few_kernel(AdapterArgs a) {
  __shared__ int s_tok[16];
  __shared__ FewSmem s_few;
  __shared__ float s_sum[8][16][17];
  wait_then_let_next_start();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  int id;
  const int m = few_group<false>(a, blockIdx.x, s_tok, s_few, id);
  if (m == 0 || id == a.n) return;
  const int r0 = a.row[id], rank = a.row[id + 1] - r0, rc = blockIdx.z * 16;
  if (rc >= rank) return;
  const int k0 = blockIdx.y * kAD_KFew, k1 = min(k0 + kAD_KFew, a.d_in);
  const T* x0 = static_cast<const T*>(a.x) + (long long)s_tok[min(g, m - 1)] * a.x_st + 8 * c;
  const T* x1 = static_cast<const T*>(a.x) + (long long)s_tok[min(g + 8, m - 1)] * a.x_st + 8 * c;
  const T* w0 = static_cast<const T*>(a.A) + (long long)(r0 + rc + g) * a.d_in + 8 * c;
  const T* w1 = w0 + 8ll * a.d_in;
  float acc[2][4] = {};
  const uint4 none = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 4
  for (int k = k0 + 32 * warp; k < k1; k += 256) {
    const bool in = k + 8 * c < k1;      // whole 16 bytes: d_in and the parts are multiples of 8
    const uint4 a0 = in && g < m ? *reinterpret_cast<const uint4*>(x0 + k) : none;
    const uint4 a1 = in && g + 8 < m ? *reinterpret_cast<const uint4*>(x1 + k) : none;
    const uint4 b0 = in ? ldg_stream(reinterpret_cast<const uint4*>(w0 + k)) : none;
    const uint4 b1 = in ? ldg_stream(reinterpret_cast<const uint4*>(w1 + k)) : none;
    mma16816<T>(acc[0], a0.x, a1.x, a0.y, a1.y, b0.x, b0.y);
    mma16816<T>(acc[1], a0.x, a1.x, a0.y, a1.y, b1.x, b1.y);
    mma16816<T>(acc[0], a0.z, a1.z, a0.w, a1.w, b0.z, b0.w);
    mma16816<T>(acc[1], a0.z, a1.z, a0.w, a1.w, b1.z, b1.w);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) s_sum[warp][g + (e >> 1) * 8][8 * j + 2 * c + (e & 1)] = acc[j][e];
  __syncthreads();
  const int row = tid >> 4, col = tid & 15;
  if (row < m) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += s_sum[w][row][col];
    a.h[((size_t)blockIdx.y * a.T + s_tok[row]) * a.rmax + rc + col] = s;
  }
}

// Many tokens: one CTA sorts them by adapter, in their order (a group's place among the others decides where its sums are cut, so a token's group must not
// be left to chance), and lists the groups.  Each of up to 32 warps counts the adapters of a stretch of tokens, 32 at a time, in a row of its own; a running
// sum over the rows then says where each warp's tokens of each adapter begin, and the warps go the same way again.
constexpr int kAD_RouteWords = 55000;           // of shared memory
static int adapter_route_warps(int n) { return min(32, (kAD_RouteWords - 3 * (n + 2)) / (n + 1)); }
__global__ void __launch_bounds__(1024) adapter_route_kernel(AdapterArgs a, int warps) {
  extern __shared__ int s_dyn[];
  int* s_count = s_dyn;               // [n + 2] tokens of each adapter (n: none)
  int* s_at = s_count + a.n + 2;      // first place in perm
  int* s_grp = s_at + a.n + 2;        // first group
  int* s_row = s_grp + a.n + 2;       // [warps][n + 1] a warp's tokens of each adapter, then those of the warps before it
  __shared__ int2 s_warp[32];
  wait_for_stream();
  let_next_start();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, buckets = a.n + 1;
  for (int i = tid; i < warps * buckets; i += 1024) s_row[i] = 0;
  __syncthreads();
  const int per = ((a.T + 31) / 32 + warps - 1) / warps * 32;
  const long long begin = (long long)warp * per;
  const int end = warp < warps ? (int)min(begin + per, (long long)a.T) : 0;
  int* mine = s_row + warp * buckets;
  // what(token, adapter, tokens of it before this one in the warp's stretch), in the order of the tokens
  auto walk = [&](auto what) {
    for (long long t0 = begin; t0 < end; t0 += 256) {
      int id[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) id[k] = t0 + 32 * k + lane < end ? adapter_of(a, a.ids[t0 + 32 * k + lane]) : -1;
      // 256 tokens of one adapter at once
      const int one = __shfl_sync(0xffffffffu, id[0], 0);
      bool alike = one >= 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) alike = alike && id[k] == one;
      if (__all_sync(0xffffffffu, alike)) {
        const int before = mine[one];
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 8; ++k) what((int)t0 + 32 * k + lane, one, before + 32 * k + lane);
        if (lane == 0) mine[one] = before + 256;
        __syncwarp();
        continue;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (t0 + 32 * k >= end) break;
        const unsigned same = __match_any_sync(0xffffffffu, id[k]);
        const int before = id[k] >= 0 ? mine[id[k]] : 0;
        __syncwarp();
        if (id[k] >= 0) {
          what((int)t0 + 32 * k + lane, id[k], before + __popc(same & ((1u << lane) - 1u)));
          if (lane == __ffs(same) - 1) mine[id[k]] = before + __popc(same);
        }
        __syncwarp();
      }
    }
  };
  walk([](int, int, int) {});
  __syncthreads();
  for (int b = warp; b < buckets; b += 32) {
    const int n = lane < warps ? s_row[lane * buckets + b] : 0;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (lane < warps) s_row[lane * buckets + b] = incl - n;
    if (lane == 31) s_count[b] = incl;
  }
  __syncthreads();
  // both running sums over the adapters, thread i holding `each` of them
  const int each = (buckets + 1023) / 1024, lo = min(tid * each, buckets), hi = min(lo + each, buckets);
  int2 sum = make_int2(0, 0);
  for (int b = lo; b < hi; ++b) {
    sum.x += (s_count[b] + 7) & ~7;
    sum.y += (s_count[b] + kAD_Group - 1) / kAD_Group;
  }
  int2 incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, incl.x, o), y = __shfl_up_sync(0xffffffffu, incl.y, o);
    if (lane >= o) {
      incl.x += x;
      incl.y += y;
    }
  }
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  int2 at = make_int2(incl.x - sum.x, incl.y - sum.y);
  for (int w = 0; w < warp; ++w) {
    at.x += s_warp[w].x;
    at.y += s_warp[w].y;
  }
  for (int b = lo; b < hi; ++b) {
    s_at[b] = at.x;
    s_grp[b] = at.y;
    at.x += (s_count[b] + 7) & ~7;
    at.y += (s_count[b] + kAD_Group - 1) / kAD_Group;
  }
  if (lo < hi && hi == buckets) s_grp[buckets] = at.y;
  __syncthreads();
  const int total = s_grp[buckets];
  for (int k = tid; k < total; k += 1024) {
    int b = 0, e = buckets;           // the last bucket that begins at or before k
    while (e - b > 1) {
      const int mid = (b + e) >> 1;
      if (s_grp[mid] <= k) b = mid; else e = mid;
    }
    const int skip = (k - s_grp[b]) * kAD_Group;
    a.groups[k] = make_int4(b, s_at[b] + skip, min(kAD_Group, s_count[b] - skip), 0);
    a.arrived[k] = 0;
  }
  if (tid == 0) {
    a.n_groups[1] = s_grp[a.n];       // tokens without an adapter come last: they have no h, and in place they are done
    a.n_groups[0] = a.out == a.y ? s_grp[a.n] : total;
  }
  walk([&](int t, int id, int nth) { a.perm[s_at[id] + nth] = t; });
}

// h of many tokens: the groups' steps of 128 values of d_in, group by group, an equal run of them to each CTA, one per SM.  x rows (gathered) and A rows come
// through a ring in shared memory (K-major, 128-byte swizzle; eight warps copy); a thread issues the products, D in TMEM (two of them) is the group's h.  A run
// that has part of a group leaves its sums in one of the CTA's two places (its first group, begun by others; its last, ended by others); the CTA that is the
// last to bring a group's part adds them all, in their order, and makes the two parts.  (A grid of groups and parts of d_in, two CTAs per SM: 25480 tokens of
// 6144 took 92 us, 8192 of 5120 37, against 69 and 32; these and the next kernel's times in bursts at 1965 MHz.)
constexpr int kAD_Ctas = 148, kAD_Step = 128, kAD_MinSteps = 8;
template <int RM>
struct ShrinkCfg {
  static constexpr int Stage = (kAD_Group + RM) * 256, Ring = RM <= 32 ? 5 : RM <= 64 ? 4 : 3, Smem = Stage * Ring + 1024;
};

template <typename T, int RM>
__global__ void __launch_bounds__(416, 1) adapter_shrink_kernel(AdapterArgs a) {
  using C = ShrinkCfg<RM>;
  constexpr int ST = C::Ring, kLag = ST - 2;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t ring_at = (smem_u32(smem_raw) + 1023) & ~1023u;
  __shared__ uint64_t x_full[ST], x_free[ST], d_full[2], d_free[2], h_full, h_told;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_last;
  volatile int* abort = &s_abort;
  wait_then_let_next_start();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int spg = (a.d_in + kAD_Step - 1) / kAD_Step;
  const long long total = (long long)a.n_groups[1] * spg, ctas = max(1ll, min((long long)kAD_Ctas, total / kAD_MinSteps));
  if ((int)blockIdx.x >= ctas || total == 0) return;
  const long long first = total * blockIdx.x / ctas;
  const int n = (int)(total * (blockIdx.x + 1) / ctas - first), g0 = (int)(first / spg), k0 = (int)(first - (long long)g0 * spg);
  if (tid == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(x_full + i, 256);
      mbar_init(x_free + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(d_full + i, 1);
      mbar_init(d_free + i, 4);
    }
    mbar_init(&h_full, 4);
    mbar_init(&h_told, 1);
    s_abort = 0;
    fence_barrier_init();
  }
  if (warp == 8) {
    tmem_alloc(&s_tmem, 2 * RM);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  if (warp < 8) {
    // a thread's pieces of 16 bytes: piece tid % 16 of the rows tid / 16 + 16 i, x rows first.  Rows of tokens that are not there repeat the last one
    const int piece = tid & 15, prow = tid >> 4;
    const uint32_t to = ring_at + (piece >> 3) * (kAD_Group * 128) + prow * 128 + (((piece & 7) ^ (prow & 7)) << 4);
    const uint32_t toA = ring_at + kAD_Group * 256 + (piece >> 3) * (RM * 128) + prow * 128 + (((piece & 7) ^ (prow & 7)) << 4);
    const T* src[8] = {};
    const T* srcA = nullptr;
    int rank = 0;
#pragma unroll 1
    for (int j = 0, g = g0, k = k0; j < n + kLag; ++j) {
      if (j < n) {
        if (j == 0 || k == 0) {
          const int4 grp = a.groups[g];
          const int r0 = a.row[grp.x];
          rank = a.row[grp.x + 1] - r0;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            src[i] = static_cast<const T*>(a.x) + (long long)a.perm[grp.y + min(prow + 16 * i, grp.z - 1)] * a.x_st + 8 * piece;
          srcA = static_cast<const T*>(a.A) + (long long)(r0 + prow) * a.d_in + 8 * piece;
        }
        if (!mbar_wait_small(x_free + j % ST, (j / ST & 1) ^ 1, abort, 0x80)) break;
        const bool in = kAD_Step * k + 8 * piece < a.d_in;
        const int at = in ? kAD_Step * k : 0;
        const uint32_t stage = (j % ST) * C::Stage;
#pragma unroll
        for (int i = 0; i < 8; ++i) copy16(to + stage + i * 2048, in ? src[i] + at : static_cast<const T*>(a.x), in);
        const T* w = in ? srcA + at : static_cast<const T*>(a.A);
#pragma unroll
        for (int i = 0; i < RM / 16; ++i, w += in ? 16 * (long long)a.d_in : 0)
          if (16 * i < rank) copy16(toA + stage + i * 2048, w, in);
        if (++k == spg) {
          k = 0;
          ++g;
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      if (j >= kLag) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kLag) : "memory");
        fence_async_smem();
        mbar_arrive(x_full + (j - kLag) % ST);
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  } else if (warp == 8) {
    uint32_t idesc = 0;
    int parts = 0;            // begun
#pragma unroll 1
    for (int j = 0, g = g0, k = k0; j < n; ++j) {
      const bool begins = j == 0 || k == 0, ends = j == n - 1 || k == spg - 1;
      if (begins) {
        const int id = a.groups[g].x;
        idesc = idesc_f16(128, a.row[id + 1] - a.row[id], kIsBf16<T>);
        if (!mbar_wait_warp_small(d_free + (parts & 1), (parts >> 1 & 1) ^ 1, abort, 0x81)) break;
        ++parts;
      }
      if (!mbar_wait_warp_small(x_full + j % ST, j / ST & 1, abort, 0x89)) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t xs = ring_at + (j % ST) * C::Stage, as = xs + kAD_Group * 256, d = tmem + ((parts - 1) & 1) * RM;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
          umma_f16_ss(d, sdesc_sw128(xs + (ks >> 2) * (kAD_Group * 128) + (ks & 3) * 32), sdesc_sw128(as + (ks >> 2) * (RM * 128) + (ks & 3) * 32), idesc,
                      !begins || ks > 0);
        umma_commit(x_free + j % ST);
        if (ends) umma_commit(d_full + ((parts - 1) & 1));
      }
      __syncwarp();
      if (++k == spg) {
        k = 0;
        ++g;
      }
    }
  } else {
    // thread = row of the group; sums of part of d_in lie rank by rank, so that rows are neighbours
    const int row0 = 32 * (warp & 3), r = row0 + lane;
    // the CTA that has step i (no run is empty)
    auto cta_of = [&](long long i) { return (int)(((i + 1) * ctas + total - 1) / total) - 1; };
    uint32_t shared = 0;               // groups that are other CTAs' too
#pragma unroll 1
    for (int p = 0, g = g0, left = n, k = k0; left > 0; ++p, ++g, left -= spg - k, k = 0) {
      const int4 grp = a.groups[g];
      const int m = grp.z, rank = a.row[grp.x + 1] - a.row[grp.x];
      const int b0 = cta_of((long long)g * spg), b1 = cta_of((long long)(g + 1) * spg - 1);
      const float scale = a.scale[grp.x];
      if (!mbar_wait_warp_small(d_full + (p & 1), p >> 1 & 1, abort, 0x8a)) break;
      tc_fence_after();
      float v[RM];
#pragma unroll
      for (int c = 0; c < RM; c += 16)
        if (c < rank) {
          uint32_t x[16];
          tmem_ld16(tmem + (p & 1) * RM + ((uint32_t)row0 << 16) + c, x);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) v[c + i] = __uint_as_float(x[i]);
        }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(d_free + (p & 1));
      if (b0 < b1) {
        auto place = [&](int b) { return a.h + (size_t)(2 * b + (b == b0)) * kAD_Group * RM + r; };
        float* to = place(blockIdx.x);
#pragma unroll
        for (int c = 0; c < RM; ++c)
          if (c < rank) __stcg(to + c * kAD_Group, v[c]);
        __threadfence();
        __syncwarp();
        if (lane == 0) mbar_arrive(&h_full);
        const uint32_t phase = shared++ & 1;
        if (warp == 9) {
          if (!mbar_wait_warp_small(&h_full, phase, abort, 0x8b)) break;
          if (lane == 0) {
            s_last = atomicAdd(a.arrived + g, 1) == b1 - b0;
            mbar_arrive(&h_told);
          }
          __syncwarp();
        }
        if (!mbar_wait_warp_small(&h_told, phase, abort, 0x8c)) break;
        if (!s_last) continue;         // (s_last is written again when all four warps are behind the next part's stores)
        __threadfence();
        // 32 loads at a time, those of ranks that are not there too
#pragma unroll
        for (int c = 0; c < RM; c += 32)
          if (c < rank) {
#pragma unroll 1
            for (int b = b0; b <= b1; ++b) {
              const float* from = place(b) + c * kAD_Group;
              float x[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) x[i] = __ldcg(from + i * kAD_Group);
#pragma unroll
              for (int i = 0; i < 32; ++i) v[c + i] = b == b0 ? x[i] : v[c + i] + x[i];
            }
          }
      }
      float big = 0.f;
#pragma unroll
      for (int c = 0; c < RM; ++c)
        if (c < rank) big = fmaxf(big, fabsf(v[c]));
      const RowScale rs(big);
      if (r < m) {
        T* to = static_cast<T*>(a.parts) + (size_t)grp.y * 2 * a.rmax + (r >> 3) * 8 * rank + (r & 7) * 8;
        const int other = ((m + 7) & ~7) * rank;
#pragma unroll
        for (int c = 0; c < RM; c += 8)
          if (c < rank) {
            uint4 h, l;
            T *hi = reinterpret_cast<T*>(&h), *lo = reinterpret_cast<T*>(&l);
#pragma unroll
            for (int i = 0; i < 8; ++i) rs.parts(v[c + i], hi[i], lo[i]);
            *reinterpret_cast<uint4*>(to + 8 * c) = h;
            *reinterpret_cast<uint4*>(to + other + 8 * c) = l;
          }
        a.back[grp.y + r] = scale * rs.back();
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0) report_abort(abort, a.err);
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * RM);
  }
}

// out of a few tokens: CTA = (group, `units` times 512 columns), a warp 64 of them.  One token: a lane has columns l and l + 32, whose ranks it loads 16 bytes at a
// time, the next 16 ranks ahead, and h in fp32: most of a tensor-core tile would be empty.
template <typename T, typename F>
__device__ __forceinline__ void expand_one(const AdapterArgs& a, const T* w, int rank, int tok, const float* s_h, float scale, int col0, int units, F h_there) {
  const int lane = threadIdx.x & 31;
  const T* y0 = static_cast<const T*>(a.y) + (long long)tok * a.y_st;
  T* out0 = static_cast<T*>(a.out) + (long long)tok * a.o_st;
  T y[2], y_next[2];
  uint4 b[4];
  const uint4 *p, *q;
  // unit u's y and first 16 ranks
  auto begin = [&](int u) {
    const int col = col0 + 512 * u + lane;
    if (u >= units || col >= a.d_out) return;
    const bool two = col + 32 < a.d_out;
    y_next[0] = y0[col];
    if (two) y_next[1] = y0[col + 32];
    p = reinterpret_cast<const uint4*>(w + (long long)(col >> 3) * 8 * rank + (col & 7) * 8);
    q = two ? p + 4 * rank : p;
    b[0] = __ldg(p), b[1] = __ldg(p + 8), b[2] = __ldg(q), b[3] = __ldg(q + 8);
  };
  begin(0);
  h_there();
#pragma unroll 1
  for (int u = 0; u < units; ++u) {
    const int col = col0 + 512 * u + lane;
    if (col >= a.d_out) return;
    uint64_t acc[2] = {0, 0};
    y[0] = y_next[0], y[1] = y_next[1];
#pragma unroll 1
    for (int r = 0; r < rank; r += 16) {
      uint4 now[4] = {b[0], b[1], b[2], b[3]};
      if (r + 16 < rank) {
        p += 16;
        q += 16;
        b[0] = __ldg(p), b[1] = __ldg(p + 8), b[2] = __ldg(q), b[3] = __ldg(q + 8);
      } else {
        begin(u + 1);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const ulonglong2* h = reinterpret_cast<const ulonglong2*>(s_h + r + 8 * i);
        const ulonglong2 h0 = h[0], h1 = h[1];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const T* e = reinterpret_cast<const T*>(&now[2 * k + i]);
          uint64_t wf[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) wf[x] = pair2((float)e[2 * x], (float)e[2 * x + 1]);
          acc[k] = fma2(wf[3], h1.y, fma2(wf[2], h1.x, fma2(wf[1], h0.y, fma2(wf[0], h0.x, acc[k]))));
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (k == 0 || col + 32 < a.d_out) out0[col + 32 * k] = (T)fmaf(lo_hi(acc[k], 0) + lo_hi(acc[k], 1), scale, (float)y[k]);
  }
}

// 2 to 16 tokens: mma.sync with h's two parts (as for many tokens), 32 columns at a time.  Column 8 (n / 2) + 2 j + n % 2 of them is column n of product j, so
// that a lane ends with 8 consecutive columns of two tokens.
constexpr int kAD_FewPitch = kAD_MaxRank + 8;       // from row to row of h's parts in shared memory
template <typename T, typename F>
__device__ __forceinline__ void expand_several(const AdapterArgs& a, const T* w, int rank, int m, const int* s_tok, const T* s_parts, const float* s_back, int col0,
                                               int units, F h_there) {
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  auto col_of = [&](int u) { return col0 + 512 * (u >> 1) + 32 * (u & 1); };
  uint32_t b[8];                   // product j's two values of k 0 .. 7 and 8 .. 15
  auto load = [&](int u, int r) {
    const int col = col_of(u) + 8 * (g >> 1);
    const T* from = w + (long long)(col >> 3) * 8 * rank + 8 * r + 8 * (g & 1) + 2 * c;
    const bool in = u < 2 * units && col < a.d_out;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      b[2 * j] = in ? __ldg(reinterpret_cast<const uint32_t*>(from + 16 * j)) : 0u;
      b[2 * j + 1] = in ? __ldg(reinterpret_cast<const uint32_t*>(from + 16 * j + 64)) : 0u;
    }
  };
  load(0, 0);
  h_there();
#pragma unroll 1
  for (int u = 0; u < 2 * units; ++u) {
    if (col_of(u) >= a.d_out) return;
    const int col = col_of(u) + 8 * c;
    uint4 y[2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (g + 8 * e < m && col < a.d_out)
        y[e] = ldg_stream(reinterpret_cast<const uint4*>(static_cast<const T*>(a.y) + (long long)s_tok[g + 8 * e] * a.y_st + col));
    float acc[4][4] = {};
#pragma unroll 1
    for (int r = 0; r < rank; r += 16) {
      uint32_t now[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) now[j] = b[j];
      if (r + 16 < rank) load(u, r + 16); else load(u + 1, 0);
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        const T* h = s_parts + (part * 16 + g) * kAD_FewPitch + r + 2 * c;
        const uint32_t a0 = *reinterpret_cast<const uint32_t*>(h), a1 = *reinterpret_cast<const uint32_t*>(h + 8 * kAD_FewPitch),
                       a2 = *reinterpret_cast<const uint32_t*>(h + 8), a3 = *reinterpret_cast<const uint32_t*>(h + 8 * kAD_FewPitch + 8);
#pragma unroll
        for (int j = 0; j < 4; ++j) mma16816<T>(acc[j], a0, a1, a2, a3, now[2 * j], now[2 * j + 1]);
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (g + 8 * e < m && col < a.d_out) {
        const float back = s_back[g + 8 * e];
        T* x = reinterpret_cast<T*>(&y[e]);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (T)fmaf(acc[i >> 1][2 * e + (i & 1)], back, (float)x[i]);
        *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (long long)s_tok[g + 8 * e] * a.o_st + col) = y[e];
      }
  }
}

template <typename T>
__global__ void __launch_bounds__(256, 3) adapter_expand_few_kernel(AdapterArgs a) {
  __shared__ __align__(16) float s_h[kAD_MaxRank];
  __shared__ __align__(16) T s_parts[2 * 16 * kAD_FewPitch];
  __shared__ float s_back[16];
  __shared__ int s_tok[16];
  __shared__ FewSmem s_few;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  let_next_start();
  int id;
  // ids and y are older than the kernel before this one (launch_early.h; y past L1 takes 0.2 us more of 64 tokens' 20)
  if (tid == 255) acquire_early(a.ids);
  const int m = few_group<true>(a, blockIdx.x, s_tok, s_few, id);
  if (m == 0 || (id == a.n && a.out == a.y)) {
    if (blockIdx.x == 0) wait_for_stream();
    return;
  }
  const int col0 = blockIdx.y * a.units * 512 + warp * 64;
  if (id == a.n) {
    wait_for_stream();
    for (int u = 0; u < a.units; ++u) {
      const int col = col0 + 512 * u + 2 * lane;
      if (col >= a.d_out) break;
      for (int t = 0; t < m; ++t)
        *reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + (long long)s_tok[t] * a.o_st + col) =
            *reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.y) + (long long)s_tok[t] * a.y_st + col);
    }
    return;
  }
  const int r0 = a.row[id], rank = a.row[id + 1] - r0;
  const float scale = a.scale[id];
  const T* w = static_cast<const T*>(a.B) + (long long)r0 * a.d_out;
  // B, and y, which is older than the kernel before this one (launch_early.h), are on their way before h is there
  auto h_there = [&]() {
    wait_for_stream();
    // a warp a token at a time, lane l the ranks l, l + 32, ...
    for (int t = warp; t < m; t += 8) {
      float v[kAD_MaxRank / 32], big = 0.f;
      bool finite = true;
#pragma unroll
      for (int k = 0; k < kAD_MaxRank / 32; ++k) {
        v[k] = 0.f;
        const float* p = a.h + (size_t)s_tok[t] * a.rmax + 32 * k + lane;
        if (32 * k + lane < rank) {
#pragma unroll 8
          for (int i = 0; i < a.splits; ++i) v[k] += p[(size_t)i * a.T * a.rmax];
        }
        big = fmaxf(big, fabsf(v[k]));
        finite = finite && fabsf(v[k]) < INFINITY;
      }
      if (m == 1) {
        // NaN for all ranks where one is not finite, as the parts of several tokens give it
        finite = __all_sync(0xffffffffu, finite);
#pragma unroll
        for (int k = 0; k < kAD_MaxRank / 32; ++k)
          if (32 * k + lane < rank) s_h[32 * k + lane] = finite ? v[k] : NAN;
      } else {
        const RowScale rs(warp_max(big));
#pragma unroll
        for (int k = 0; k < kAD_MaxRank / 32; ++k)
          if (32 * k + lane < rank) {
            T* to = s_parts + t * kAD_FewPitch + 32 * k + lane;
            rs.parts(v[k], to[0], to[16 * kAD_FewPitch]);
          }
        if (lane == 0) s_back[t] = scale * rs.back();
      }
    }
    __syncthreads();               // (of h's parts, rows of tokens that are not there are left as they were: nobody reads their sums)
  };
  if (m == 1) expand_one<T>(a, w, rank, s_tok[0], s_h, scale, col0, a.units, h_there);
  else expand_several<T>(a, w, rank, m, s_tok, s_parts, s_back, col0, a.units, h_there);
}

// out of many tokens: tiles of a group (128 tokens) and 128 columns, group by group, an equal run of them to each SM's one CTA.  Four warps bring y's rows into
// a ring of shared memory (256 bytes a copy), one
// thread B's columns (N operand) and, when the group changes, h's two parts (M operand), both of which lie in memory as the products read them; a thread issues
// the products, and eight warps add D (TMEM, two of them) to y where it lies and send the rows out; a thread has half a row.
// HBM under reads and writes at once wants about 130 KB of reads in flight per SM, whatever the products do (a bare copy of 8192 x 12288 by
// such tiles: 72 us with four tiles of y on their way, 106 to 112 with two or three).  So y goes through shared memory: 68 us for those sizes and ranks up to 64,
// against 106 with y in registers, two or three CTAs to an SM, and 85 with B and h gathered and swizzled by threads (cp.async) in the place of one copy a tile.  A warp issues a copy of its own bytes about every 70 cycles: one warp for all rows
// of y took 198 us.
constexpr int kAD_Tile = 128, kAD_Pitch = 272;      // bytes from row to row of y in shared memory: no two of eight neighbouring rows in the same banks
// an operand [rows / 8][steps][2][8 rows][8 values]: blocks of 8 rows of 16 bytes, 128 bytes from block to block along K, 256 steps bytes along the rows
__device__ __forceinline__ uint64_t sdesc_core(uint32_t addr, int steps) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)(128 >> 4) << 16 | (uint64_t)(16 * steps) << 32 | 1ull << 46;
}
template <typename T, int RM>
struct ExpandCfg {
  static constexpr int Atoms = RM <= 64 ? 1 : 2, Ring = RM <= 64 ? 4 : 2;       // of 64 ranks; tiles of y
  static constexpr int HBytes = 2 * Atoms * kAD_Group * 128, BBytes = Atoms * kAD_Tile * 128, YBytes = kAD_Group * kAD_Pitch;
  static constexpr int Smem = HBytes + 2 * BBytes + Ring * YBytes + 1024;
};

template <typename T, int RM>
__global__ void __launch_bounds__(448, 1) adapter_expand_kernel(AdapterArgs a) {
  using C = ExpandCfg<T, RM>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* s_h = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_y = s_h + C::HBytes + 2 * C::BBytes;
  const uint32_t hs = smem_u32(s_h), bs = hs + C::HBytes;
  // full: bytes of y; bytes of B (and h); the products.  free: eight warps' stores; the products; eight warps' reads of D
  __shared__ uint64_t y_full[C::Ring], y_free[C::Ring], b_full[2], b_free[2], d_full[2], d_free[2];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  volatile int* abort = &s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  let_next_start();
  if (tid == 0) {
    for (int i = 0; i < C::Ring; ++i) {
      mbar_init(y_full + i, 4);
      mbar_init(y_free + i, 8);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(b_full + i, 1);
      mbar_init(b_free + i, 1);
      mbar_init(d_full + i, 1);
      mbar_init(d_free + i, 8);
    }
    s_abort = 0;
    fence_barrier_init();
  }
  __syncthreads();
  // y and the groups are older than the kernel before this one: warps 0 to 3 read them before the others' wait is over (launch_early.h)
  const int tpg = (a.d_out + kAD_Tile - 1) / kAD_Tile;
  const long long total = (long long)__ldcg(a.n_groups) * tpg;
  const long long first = total * blockIdx.x / gridDim.x;
  const int n = (int)(total * (blockIdx.x + 1) / gridDim.x - first), g0 = (int)(first / tpg), c0 = (int)(first - (long long)g0 * tpg);
  bool ok = true;
  if (warp < 4) {
    const int r = tid;
    const T* src = nullptr;
    int m = 0;
#pragma unroll 1
    for (int j = 0, g = g0, c = c0; j < n; ++j) {
      if (j == 0 || c == 0) {
        const int4 grp = __ldcg(a.groups + g);
        m = grp.z;
        if (r < m) src = static_cast<const T*>(a.y) + (long long)__ldcg(a.perm + grp.y + r) * a.y_st;
      }
      const int s = j % C::Ring, bytes = 2 * min(kAD_Tile, a.d_out - c * kAD_Tile);
      if (!mbar_wait_warp_small(y_free + s, (j / C::Ring & 1) ^ 1, abort, 0x82)) break;
      if (lane == 0) mbar_expect_tx(y_full + s, min(max(m - r, 0), 32) * bytes);
      __syncwarp();
      if (r < m) bulk_load_1d(s_y + s * C::YBytes + r * kAD_Pitch, src + c * kAD_Tile, bytes, y_full + s);
      if (++c == tpg) {
        c = 0;
        ++g;
      }
    }
  } else if (warp == 4) {
    wait_for_stream();
    const T* w = nullptr;
    int rank = 0;
#pragma unroll 1
    for (int j = 0, g = g0, c = c0; j < n; ++j) {
      int rows = 0;                  // of h
      const T* h = nullptr;
      if (j == 0 || c == 0) {
        const int4 grp = a.groups[g];
        const int r0 = grp.x < a.n ? a.row[grp.x] : 0;
        rank = grp.x < a.n ? a.row[grp.x + 1] - r0 : 0;
        w = static_cast<const T*>(a.B) + (long long)r0 * a.d_out;
        h = static_cast<const T*>(a.parts) + (size_t)grp.y * 2 * a.rmax;
        rows = (grp.z + 7) & ~7;     // (rows that are not there are left as they were: nobody reads their sums)
        // h is in use until the products of tile j - 1 are done
        if (j > 0 && !mbar_wait_warp_small(b_free + ((j - 1) & 1), (j - 1) >> 1 & 1, abort, 0x83)) break;
      }
      if (!mbar_wait_warp_small(b_free + (j & 1), (j >> 1 & 1) ^ 1, abort, 0x84)) break;
      if (lane == 0) {
        const uint32_t bytes = 2 * rank * min(kAD_Tile, a.d_out - c * kAD_Tile), part = 2 * rank * rows;
        mbar_expect_tx(b_full + (j & 1), bytes + 2 * part);
        if (bytes) bulk_load_1d(s_h + C::HBytes + (j & 1) * C::BBytes, w + (long long)c * kAD_Tile * rank, bytes, b_full + (j & 1));
        if (part) {
          bulk_load_1d(s_h, h, part, b_full + (j & 1));
          bulk_load_1d(s_h + C::HBytes / 2, h + rows * rank, part, b_full + (j & 1));
        }
      }
      __syncwarp();
      if (++c == tpg) {
        c = 0;
        ++g;
      }
    }
  } else {
    wait_for_stream();
    if (warp == 5) {
      tmem_alloc(&s_tmem, 2 * kAD_Tile);
      tmem_relinquish();
    }
    tc_fence_before();
    asm volatile("bar.sync 1, 288;" ::: "memory");       // warps 5 to 13
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    if (warp == 5) {
      const uint32_t idesc = idesc_f16(128, kAD_Tile, kIsBf16<T>);
      int steps = 0;
#pragma unroll 1
      for (int j = 0, g = g0, c = c0; j < n; ++j) {
        if (j == 0 || c == 0) {
          const int id = a.groups[g].x;
          steps = id < a.n ? (a.row[id + 1] - a.row[id]) / 16 : 0;
        }
        if (!mbar_wait_warp_small(d_free + (j & 1), (j >> 1 & 1) ^ 1, abort, 0x85)) break;
        if (!mbar_wait_warp_small(b_full + (j & 1), j >> 1 & 1, abort, 0x86)) break;
        tc_fence_after();
        if (lane == 0) {
          const uint32_t b = bs + (j & 1) * C::BBytes, d = tmem + (j & 1) * kAD_Tile;
#pragma unroll 1
          for (int part = 0; part < 2; ++part)
#pragma unroll 1
            for (int ks = 0; ks < steps; ++ks) {
              umma_f16_ss(d, sdesc_core(hs + part * (C::HBytes / 2) + 256 * ks, steps), sdesc_core(b + 256 * ks, steps), idesc, part > 0 || ks > 0);
            }
          umma_commit(b_free + (j & 1));
          umma_commit(d_full + (j & 1));
        }
        __syncwarp();
        if (++c == tpg) {
          c = 0;
          ++g;
        }
      }
    } else {
      const int row0 = 32 * (warp & 3), r = row0 + lane, at = 64 * ((warp - 6) >> 2);
      const uint8_t* from = s_y + (row0 + (lane >> 3)) * kAD_Pitch + 2 * at + 16 * (lane & 7);      // eight lanes write a row
      T* out = nullptr;
      float scale = 0.f;
      int m = 0;
      bool adapted = false;
#pragma unroll 1
      for (int j = 0, g = g0, c = c0; j < n; ++j) {
        if (j == 0 || c == 0) {
          const int4 grp = a.groups[g];
          m = grp.z;
          adapted = grp.x < a.n;
          if (r < m) {
            out = static_cast<T*>(a.out) + (long long)a.perm[grp.y + r] * a.o_st + at;
            if (adapted) scale = a.back[grp.y + r];
          }
        }
        const int s = j % C::Ring, cols = min(64, a.d_out - c * kAD_Tile - at);
        if (!mbar_wait_warp_small(d_full + (j & 1), j >> 1 & 1, abort, 0x87)) break;
        if (!mbar_wait_warp_small(y_full + s, j / C::Ring & 1, abort, 0x88)) break;
        tc_fence_after();
        uint8_t* y = s_y + s * C::YBytes + r * kAD_Pitch + 2 * at;
        if (adapted && row0 < m) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (16 * k >= cols) break;
            uint32_t d[16];
            tmem_ld16(tmem + (j & 1) * kAD_Tile + at + 16 * k + ((uint32_t)row0 << 16), d);
            tmem_wait_ld();
            if (r < m) {
              // (behind d_out the second eight are no values: they go nowhere)
              uint4 v[2] = {*reinterpret_cast<const uint4*>(y + 32 * k), *reinterpret_cast<const uint4*>(y + 32 * k + 16)};
              T* x = reinterpret_cast<T*>(v);
#pragma unroll
              for (int i = 0; i < 16; ++i) x[i] = (T)fmaf(__uint_as_float(d[i]), scale, (float)x[i]);
              *reinterpret_cast<uint4*>(y + 32 * k) = v[0];
              *reinterpret_cast<uint4*>(y + 32 * k + 16) = v[1];
            }
          }
        }
        tc_fence_before();
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(d_free + (j & 1));
        uint4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const uint4*>(from + s * C::YBytes + 4 * i * kAD_Pitch);
        __syncwarp();
        if (lane == 0) mbar_arrive(y_free + s);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          T* to = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(out), 4 * i + (lane >> 3)));
          if (row0 + 4 * i + (lane >> 3) < m && 8 * (lane & 7) < cols) *reinterpret_cast<uint4*>(to + c * kAD_Tile + 8 * (lane & 7)) = v[i];
        }
        if (++c == tpg) {
          c = 0;
          ++g;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0) report_abort(abort, a.err);
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(s_tmem, 2 * kAD_Tile);
  }
}

static long long adapter_groups(int T, int n) { return T / kAD_Group + (n + 1 < T ? n + 1 : T); }

// the workspace: its bytes, and the arrays in it
static size_t adapter_layout(AdapterArgs& a, uint8_t* ws) {
  size_t at = 0;
  auto take = [&](size_t bytes) {
    uint8_t* p = ws ? ws + at : nullptr;
    at += (bytes + 15) / 16 * 16;
    return p;
  };
  if (a.T > kAD_Few) {
    const size_t groups = (size_t)adapter_groups(a.T, a.n);
    a.n_groups = reinterpret_cast<int32_t*>(take(8));
    a.groups = reinterpret_cast<int4*>(take(groups * sizeof(int4)));
    a.arrived = reinterpret_cast<int32_t*>(take(groups * 4));
    const size_t places = (size_t)a.T + 7 * (size_t)(a.n + 1 < a.T ? a.n + 1 : a.T) + 8;
    a.perm = reinterpret_cast<int32_t*>(take(places * 4));
    a.back = reinterpret_cast<float*>(take(places * 4));
    a.parts = take(places * 2 * a.rmax * 2);
    a.h = reinterpret_cast<float*>(take((size_t)2 * kAD_Ctas * kAD_Group * (a.rmax <= 32 ? 32 : a.rmax <= 64 ? 64 : 128) * 4));
  } else {
    a.h = reinterpret_cast<float*>(take((size_t)a.splits * a.T * a.rmax * 4));
  }
  return at;
}

template <typename T, int RM>
static int launch_shrink(const AdapterArgs& a, cudaStream_t stream) {
  const int rc = ensure_smem_attr((const void*)adapter_shrink_kernel<T, RM>, ShrinkCfg<RM>::Smem);
  return rc ? rc : launch_early(adapter_shrink_kernel<T, RM>, dim3(kAD_Ctas), 416, ShrinkCfg<RM>::Smem, stream, a);
}

template <typename T, int RM>
static int launch_expand(const AdapterArgs& a, int sms, cudaStream_t stream) {
  using C = ExpandCfg<T, RM>;
  const int rc = ensure_smem_attr((const void*)adapter_expand_kernel<T, RM>, C::Smem);
  return rc ? rc : launch_early(adapter_expand_kernel<T, RM>, dim3(sms), 448, C::Smem, stream, a);
}

template <typename T>
static int launch_adapters(AdapterArgs a, int sms, cudaStream_t stream) {
  int rc;
  if (a.T <= kAD_Few) {
    const int groups = few_groups(a.T, a.n);
    rc = launch_early(adapter_shrink_few_kernel<T>, dim3(groups, a.splits, a.rmax / 16), 256, 0, stream, a);
    if (rc) return rc;
    // about four CTAs per SM if there are as many groups as there can be
    const int blocks = (a.d_out + 511) / 512, cut = (4 * sms + groups - 1) / groups;
    a.units = (blocks + cut - 1) / cut;
    return launch_early(adapter_expand_few_kernel<T>, dim3(groups, (blocks + a.units - 1) / a.units), 256, 0, stream, a);
  }
  const int warps = adapter_route_warps(a.n);
  if ((rc = ensure_smem_attr((const void*)adapter_route_kernel, kAD_RouteWords * 4))) return rc;
  if ((rc = launch_early(adapter_route_kernel, dim3(1), 1024, (size_t)(3 * (a.n + 2) + warps * (a.n + 1)) * 4, stream, a, warps))) return rc;
  rc = a.rmax <= 32 ? launch_shrink<T, 32>(a, stream) : a.rmax <= 64 ? launch_shrink<T, 64>(a, stream) : launch_shrink<T, 128>(a, stream);
  if (rc) return rc;
  return a.rmax <= 64 ? launch_expand<T, 64>(a, sms, stream) : launch_expand<T, 128>(a, sms, stream);
}

}  // namespace bfb

using namespace bfb;

extern "C" {

size_t bf_adapter_workspace(int T, int n, int d_in, int rmax) {
  if (T <= 0 || n <= 0 || n > kAD_MaxAdapters || d_in <= 0 || rmax <= 0 || rmax > kAD_MaxRank) return 0;
  AdapterArgs a{};
  a.T = T; a.n = n; a.rmax = rmax; a.splits = (d_in + kAD_KFew - 1) / kAD_KFew;
  return adapter_layout(a, nullptr);
}

int bf_adapter_add(const void* x, long long x_st, const int32_t* ids, int T, int d_in, int d_out, const void* A, const void* B,
                   const int32_t* row, const float* scale, int n, int rmax, const void* y, long long y_st, void* out, long long o_st,
                   int dtype, void* ws, size_t ws_bytes, bf_stream_t stream) {
  if (T < 0 || d_in <= 0 || d_out <= 0 || n <= 0 || rmax <= 0) return BF_ERR_INVALID_ARGUMENT;
  if ((dtype != BF_BF16 && dtype != BF_F16) || d_in % 8 || d_out % 8 || rmax % 16 || rmax > kAD_MaxRank || n > kAD_MaxAdapters ||
      T > 1 << 28)
    return BF_ERR_UNSUPPORTED;
  if (T == 0) return BF_OK;
  if (!x || !ids || !A || !B || !row || !scale || !y || !out) return BF_ERR_INVALID_ARGUMENT;
  if (!aligned16(x) || !aligned16(A) || !aligned16(B) || !aligned16(y) || !aligned16(out) || ((x_st | y_st | o_st) & 7)) return BF_ERR_ALIGNMENT;
  if (!ws || ws_bytes < bf_adapter_workspace(T, n, d_in, rmax)) return BF_ERR_WORKSPACE;
  if (!aligned16(ws)) return BF_ERR_ALIGNMENT;
  DeviceState st;
  const int rc = device_state(&st);
  if (rc) return rc;
  AdapterArgs a{};
  a.x = x; a.y = y; a.out = out;
  a.x_st = x_st; a.y_st = y_st; a.o_st = o_st;
  a.ids = ids; a.row = row; a.scale = scale;
  a.A = A; a.B = B;
  a.err = st.err;
  a.n = n; a.T = T; a.d_in = d_in; a.d_out = d_out; a.rmax = rmax;
  a.splits = (d_in + kAD_KFew - 1) / kAD_KFew;
  adapter_layout(a, static_cast<uint8_t*>(ws));
  return dtype == BF_BF16 ? launch_adapters<__nv_bfloat16>(a, st.sm_count, stream) : launch_adapters<__half>(a, st.sm_count, stream);
}

}  // extern "C"
