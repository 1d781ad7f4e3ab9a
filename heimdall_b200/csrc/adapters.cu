// Low-rank adapters of many requests beside one shared projection.
//
//   out_t = y_t + s_a B_a (A_a x_t)  with token t's adapter a (none: out_t = y_t);  A_a [r_a, d_in], B_a [d_out, r_a], ranks up to 128.
//
// What bounds it is HBM: a decode step reads the adapters in use once (2 r (d_in + d_out) bytes each) and little else; a prompt
// reads x and y once and writes out once, with 4 r (1 / d_out + 1 / d_in)-fold of that in products.  Two kernels, with h = A x between them in
// fp32 (r values per token): the adapters' two halves need a sum over d_in before anything of d_out can begin.
//
// Tokens are taken in groups of one adapter, so that an adapter is read once for many tokens:
//   * few tokens (up to kAD_Few, a decode step): every token stands for a possible group of 16; a CTA compares all ids with its token's
//     and goes on if its token is the first of a group.  No pass over the ids before, two launches.
//   * more: adapter_route_kernel sorts the tokens by adapter and lists groups of 64.
// h = A x is split over d_in so that every SM has work; each split's sums are written on their own and added in order.  h enters the second
// product as two 16-bit parts of its row's power-of-two scale (hi + lo, 16 bits of bf16, 22 of fp16), so that the only rounding of consequence
// is that of out.  The order of a group's tokens, which the sort leaves to chance, has no part in their values.
// The products run on mma.sync: the first has 8 r FLOPs for the 2 bytes of an x value, the second 16 r for the 4 bytes of a y and an out, which
// its rate covers up to r = 64, and its fragments come from registers (weights) or shared memory without a layout change.
#include "capi_internal.h"
#include "common.cuh"
#include "launch_early.h"

namespace bfb {

constexpr int kAD_Few = 256;       // tokens up to which every CTA looks for its group itself (one thread each)
constexpr int kAD_MaxRank = 128;
constexpr int kAD_MaxAdapters = 4096;
constexpr int kAD_KFew = 1024;     // d_in per CTA for few tokens
constexpr int kAD_Group = 64;      // tokens per group of many

struct AdapterArgs {
  const void *x, *y;
  void* out;
  long long x_st, y_st, o_st;      // row strides, elements
  const int32_t* ids;
  const int32_t* row;              // [n + 1] the adapters' first rows in A, multiples of 16
  const float* scale;              // [n]
  const void *A, *B;               // A [row[n]][d_in]; B: adapter a's [d_out][r_a] from element row[a] d_out on
  int n, T, d_in, d_out, rmax, splits, kper, units;
  float* h;                        // [splits][T][rmax]
  int32_t* perm;                   // [T] tokens by adapter
  int4* groups;                    // (adapter or n, first of perm, tokens, -)
  int32_t* n_groups;
};

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
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {      // 16 bytes into shared memory, zeros where there are none
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint4 ldg_stream(const uint4* p) { return __ldcs(p); }

// an adapter's number, n for none
__device__ __forceinline__ int adapter_of(const AdapterArgs& a, int id) { return id >= 0 && id < a.n ? id : a.n; }

// Few tokens: the group that token `lead` begins, if it begins one: the 16 tokens of its adapter from it on, in s_tok.  Returns how many
// (0: another CTA's), and the adapter.  All 256 threads.
__device__ __forceinline__ int few_group(const AdapterArgs& a, int lead, int* s_tok, unsigned* s_mask, int& id) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  id = adapter_of(a, a.ids[lead]);
  const bool mine = tid < a.T && adapter_of(a, a.ids[tid]) == id;
  const unsigned m = __ballot_sync(0xffffffffu, mine);
  if (lane == 0) s_mask[warp] = m;
  __syncthreads();
  int before_lead = 0, before_me = 0, total = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const unsigned x = s_mask[w];
    total += __popc(x);
    before_lead += w < (lead >> 5) ? __popc(x) : w == (lead >> 5) ? __popc(x & ((1u << (lead & 31)) - 1u)) : 0;
    before_me += w < warp ? __popc(x) : w == warp ? __popc(x & ((1u << lane) - 1u)) : 0;
  }
  if (before_lead & 15) return 0;
  if (mine && before_me >= before_lead && before_me < before_lead + 16) s_tok[before_me - before_lead] = tid;
  __syncthreads();
  return min(16, total - before_lead);
}

// h of a few tokens: CTA = (group, part of d_in, 16 ranks).  A warp takes every eighth 32 values of d_in: lane (g, c) loads the 16 bytes at
// 8 c of x rows g and g + 8 and of ranks g and g + 8, the fragments of two steps (a sum over d_in may take its values in any order as
// long as both operands agree).
template <typename T>
__global__ void __launch_bounds__(256) adapter_shrink_few_kernel(AdapterArgs a) {
  __shared__ int s_tok[16];
  __shared__ unsigned s_mask[8];
  __shared__ float s_sum[8][16][17];
  wait_for_stream();
  let_next_start();        // only now: what the next kernel reads before its own wait is older than this one
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  int id;
  const int m = few_group(a, blockIdx.x, s_tok, s_mask, id);
  if (m == 0 || id == a.n) return;
  const int r0 = a.row[id], rank = a.row[id + 1] - r0, rc = blockIdx.z * 16;
  if (rc >= rank) return;
  const int k0 = blockIdx.y * a.kper, k1 = min(k0 + a.kper, a.d_in);
  const T* x0 = static_cast<const T*>(a.x) + (long long)s_tok[min(g, m - 1)] * a.x_st + 8 * c;
  const T* x1 = static_cast<const T*>(a.x) + (long long)s_tok[min(g + 8, m - 1)] * a.x_st + 8 * c;
  const T* w0 = static_cast<const T*>(a.A) + (long long)(r0 + rc + g) * a.d_in + 8 * c;
  const T* w1 = w0 + 8ll * a.d_in;
  float acc[2][4] = {};
  const uint4 none = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 4
  for (int k = k0 + 32 * warp; k < k1; k += 256) {
    const bool in = k + 8 * c < k1;      // whole 16 bytes: d_in and the parts are multiples of 8
    const uint4 a0 = in && g < m ? __ldg(reinterpret_cast<const uint4*>(x0 + k)) : none;
    const uint4 a1 = in && g + 8 < m ? __ldg(reinterpret_cast<const uint4*>(x1 + k)) : none;
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

// The sorted list of many tokens and their groups, by one CTA.  A thread takes consecutive tokens, whose adapters come in runs, and
// counts whole runs.
__global__ void __launch_bounds__(1024) adapter_route_kernel(AdapterArgs a) {
  extern __shared__ int s_dyn[];
  int* s_at = s_dyn;                  // [n + 2] count, then first place in perm of each adapter (n: none)
  int* s_grp = s_dyn + a.n + 2;       // [n + 2] first group
  __shared__ int2 s_warp[32];
  wait_for_stream();
  let_next_start();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, buckets = a.n + 1;
  for (int i = tid; i < buckets + 1; i += 1024) s_at[i] = 0;
  __syncthreads();
  const int per = min((a.T + 1023) / 1024, 32);
  auto runs = [&](auto&& done) {
    for (int t0 = 0; t0 < a.T; t0 += 1024 * per) {
      const int first = t0 + tid * per, n = min(per, a.T - first);
      int v[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = i < n ? adapter_of(a, __ldg(a.ids + first + i)) : -1;
      int begin = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        if (i < n && (i + 1 == n || v[i + 1 < 32 ? i + 1 : 31] != v[i])) {
          done(v[i], first + begin, i + 1 - begin);
          begin = i + 1;
        }
      }
    }
  };
  runs([&](int b, int, int n) { atomicAdd(&s_at[b], n); });
  __syncthreads();
  // both running sums over the adapters, thread i holding `each` of them
  const int each = (buckets + 1023) / 1024, lo = min(tid * each, buckets), hi = min(lo + each, buckets);
  int2 mine = make_int2(0, 0);
  for (int b = lo; b < hi; ++b) {
    mine.x += s_at[b];
    mine.y += (s_at[b] + kAD_Group - 1) / kAD_Group;
  }
  int2 incl = mine;
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
  int2 at = make_int2(incl.x - mine.x, incl.y - mine.y);
  for (int w = 0; w < warp; ++w) {
    at.x += s_warp[w].x;
    at.y += s_warp[w].y;
  }
  for (int b = lo; b < hi; ++b) {
    const int n = s_at[b];
    s_at[b] = at.x;
    s_grp[b] = at.y;
    at.x += n;
    at.y += (n + kAD_Group - 1) / kAD_Group;
  }
  if (lo < hi && hi == buckets) {
    s_at[buckets] = at.x;
    s_grp[buckets] = at.y;
  }
  __syncthreads();
  const int total = s_grp[buckets];
  for (int k = tid; k < total; k += 1024) {
    int b = 0, e = buckets;           // the last bucket that begins at or before k
    while (e - b > 1) {
      const int mid = (b + e) >> 1;
      if (s_grp[mid] <= k) b = mid; else e = mid;
    }
    const int first = s_at[b] + (k - s_grp[b]) * kAD_Group;
    a.groups[k] = make_int4(b, first, min(kAD_Group, s_at[b + 1] - first), 0);
  }
  if (tid == 0) *a.n_groups = total;
  __syncthreads();
  runs([&](int b, int first, int n) {
    const int to = atomicAdd(&s_at[b], n);
    for (int i = 0; i < n; ++i) a.perm[to + i] = first + i;
  });
}

// h of a group of 64 tokens: CTA = (group, part of d_in); x rows and A rows come 64 values at a time through a ring in shared memory
// (rows of 128 bytes, 16-byte pieces at (piece ^ row)); warps 0 - 3 take 16 tokens and the first half of the 64 values, warps 4 - 7
// the second, added at the end.
template <typename T, int RM, int ST>
__global__ void __launch_bounds__(256) adapter_shrink_kernel(AdapterArgs a) {
  constexpr int kStage = (kAD_Group + RM) * 128;
  extern __shared__ __align__(128) uint8_t s_ring[];
  __shared__ int s_tok[kAD_Group];
  wait_for_stream();
  let_next_start();
  if ((int)blockIdx.x >= *a.n_groups) return;
  const int4 grp = a.groups[blockIdx.x];
  if (grp.x == a.n) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3, m = grp.z;
  const int r0 = a.row[grp.x], rank = a.row[grp.x + 1] - r0;
  if (tid < kAD_Group) s_tok[tid] = a.perm[grp.y + min(tid, m - 1)];
  __syncthreads();
  const int k0 = blockIdx.y * a.kper, k1 = min(k0 + a.kper, a.d_in), steps = (k1 - k0 + 63) / 64;
  const uint32_t ring = smem_u32(s_ring);
  // a thread's pieces: piece tid & 7 of rows tid / 8 + 32 i, x rows first
  const int piece = tid & 7, prow = tid >> 3;
  const T* src[2 + RM / 32];
#pragma unroll
  for (int i = 0; i < 2 + RM / 32; ++i) {
    const int r = prow + 32 * i;
    src[i] = (i < 2 ? static_cast<const T*>(a.x) + (long long)s_tok[r] * a.x_st
                    : static_cast<const T*>(a.A) + (long long)(r0 + min(r - kAD_Group, rank - 1)) * a.d_in) + 8 * piece;
  }
  auto fetch = [&](int s) {
    if (s < steps) {
      const int k = k0 + 64 * s;
      const bool in = k + 8 * piece < k1;
      const uint32_t dst = ring + (s % ST) * kStage;
#pragma unroll
      for (int i = 0; i < 2 + RM / 32; ++i) {
        const int r = prow + 32 * i;
        if (i < 2 ? r < m : r - kAD_Group < rank) copy16(dst + r * 128 + ((piece ^ (r & 7)) << 4), in ? src[i] + k : src[i], in);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // rows of tokens that are not there: zeros, once (their products are not written, but may not be read uninitialised)
  for (int i = tid; i < (kAD_Group - m) * 8 * ST; i += 256) {
    const int s = i / ((kAD_Group - m) * 8), j = i % ((kAD_Group - m) * 8);
    *reinterpret_cast<uint4*>(s_ring + s * kStage + m * 128 + j * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int s = 0; s < ST - 1; ++s) fetch(s);
  float acc[RM / 8][4] = {};
  const int wr = (warp & 3) * 16, half = warp >> 2;
  for (int s = 0; s < steps; ++s) {
    asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
    __syncthreads();
    fetch(s + ST - 1);
    const uint32_t xs = ring + (s % ST) * kStage, ws = xs + kAD_Group * 128;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int p = half * 4 + ks * 2;           // the 16-byte piece at which these 16 values begin
      uint32_t x[4];
      const int xr = wr + (lane & 15);
      ldsm4(x, xs + xr * 128 + (((p + (lane >> 4)) ^ (xr & 7)) << 4));
#pragma unroll
      for (int j = 0; j < RM / 16; ++j) {
        if (16 * j < rank) {
          uint32_t w[4];
          const int r = 16 * j + (lane & 7) + ((lane >> 4) << 3);
          ldsm4(w, ws + r * 128 + (((p + ((lane >> 3) & 1)) ^ (r & 7)) << 4));
          mma16816<T>(acc[2 * j], x[0], x[1], x[2], x[3], w[0], w[1]);
          mma16816<T>(acc[2 * j + 1], x[0], x[1], x[2], x[3], w[2], w[3]);
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float* s_half = reinterpret_cast<float*>(s_ring);      // [64][RM + 2]
  if (half) {
#pragma unroll
    for (int j = 0; j < RM / 8; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *reinterpret_cast<float2*>(s_half + (wr + g + 8 * e) * (RM + 2) + 8 * j + 2 * c) = make_float2(acc[j][2 * e], acc[j][2 * e + 1]);
  }
  __syncthreads();
  if (!half) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = wr + g + 8 * e;
      if (r >= m) continue;
      float* to = a.h + ((size_t)blockIdx.y * a.T + s_tok[r]) * a.rmax;
#pragma unroll
      for (int j = 0; j < RM / 8; ++j) {
        if (8 * j >= rank) break;
        const float2 o = *reinterpret_cast<const float2*>(s_half + r * (RM + 2) + 8 * j + 2 * c);
        *reinterpret_cast<float2*>(to + 8 * j + 2 * c) = make_float2(acc[j][2 * e] + o.x, acc[j][2 * e + 1] + o.y);
      }
    }
  }
}

// out of a group: CTA = (group, `units` times 256 columns), a warp 32 columns at a time.  B's fragments come straight from memory: in step
// ks lane (g, c) loads the 8 bytes of ranks 16 ks + 4 c .. + 3 of the columns that it stands for, and reads the same ranks of h's rows g and
// g + 8.  Column n of product j is column 8 (n / 2) + 2 j + n % 2 of the 32, so that a lane ends with 8 consecutive columns of two
// rows: 16-byte accesses to y and out.
template <typename T, int GT>      // GT: 16 (few tokens) or 64 tokens per group
__global__ void __launch_bounds__(256) adapter_expand_kernel(AdapterArgs a) {
  constexpr int KS = 4;            // steps of 16 ranks whose weights stay in registers
  constexpr int kRow = kAD_MaxRank * 4 + 32;       // bytes: hi and lo parts of a row of h; 32 more spread the rows over the banks
  extern __shared__ __align__(16) uint8_t s_h[];
  __shared__ int s_tok[GT];
  __shared__ float s_scale[GT];
  __shared__ unsigned s_mask[8];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  let_next_start();
  int m, id;
  // the ids and groups are older than the kernel before this one, which began by waiting for what was before it
  if constexpr (GT == 16) {
    m = few_group(a, blockIdx.x, s_tok, s_mask, id);
    if (m == 0) return;
  } else {
    if ((int)blockIdx.x >= *a.n_groups) return;
    const int4 grp = a.groups[blockIdx.x];
    id = grp.x;
    m = grp.z;
    if (tid < m) s_tok[tid] = a.perm[grp.y + tid];
  }
  if (id == a.n && a.out == a.y) return;
  const int r0 = id < a.n ? a.row[id] : 0, rank = id < a.n ? a.row[id + 1] - r0 : 0;
  const T* w = static_cast<const T*>(a.B) + (long long)r0 * a.d_out;
  const int col0 = blockIdx.y * a.units * 256 + warp * 32, steps = rank / 16;
  uint2 b[KS][4];
  auto weights = [&](int cu, int k0) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int col = cu + 8 * (g >> 1) + 2 * j + (g & 1);
        b[ks][j] = k0 + ks < steps && col < a.d_out ? __ldg(reinterpret_cast<const uint2*>(w + (long long)col * rank + 16 * (k0 + ks) + 4 * c))
                                                    : make_uint2(0u, 0u);
      }
  };
  weights(col0, 0);
  wait_for_stream();
  __syncthreads();
  if (rank) {
    for (int r = warp; r < GT; r += 8) {
      float v[kAD_MaxRank / 32];
      float big = 0.f;
#pragma unroll
      for (int i = 0; i < kAD_MaxRank / 32; ++i) {
        v[i] = 0.f;
        if (r < m && 32 * i + lane < rank)
          for (int s = 0; s < a.splits; ++s) v[i] += a.h[((size_t)s * a.T + s_tok[r]) * a.rmax + 32 * i + lane];
        big = fmaxf(big, fabsf(v[i]));
      }
      big = warp_max(big);
      // a power of two that takes the row's largest to [2^13, 2^14): both parts then keep all of their bits in fp16 too
      const int ex = big > 0.f && big < INFINITY ? min(max((int)(__float_as_uint(big) >> 23), 14), 253) : 140;
      const float up = __uint_as_float((uint32_t)(267 - ex) << 23);
      T* hi = reinterpret_cast<T*>(s_h + r * kRow);
#pragma unroll
      for (int i = 0; i < kAD_MaxRank / 32; ++i) {
        if (32 * i + lane < rank) {
          const float z = v[i] * up;
          const T p = (T)z;
          hi[32 * i + lane] = p;
          hi[rank + 32 * i + lane] = (T)(z - (float)p);
        }
      }
      if (lane == 0) s_scale[r] = id < a.n ? a.scale[id] * __uint_as_float((uint32_t)(ex - 13) << 23) : 0.f;
    }
  }
  __syncthreads();
  for (int u = 0; u < a.units; ++u) {
    const int cu = col0 + u * 256;
    if (cu >= a.d_out) break;
    if (u && steps <= KS) weights(cu, 0);
    const bool in = cu + 8 * c < a.d_out;
#pragma unroll 1
    for (int rt = 0; rt < GT && rt < m; rt += 16) {
      uint4 yv[2];
      long long at[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = rt + g + 8 * e;
        if (r < m && in) {
          yv[e] = ldg_stream(reinterpret_cast<const uint4*>(static_cast<const T*>(a.y) + (long long)s_tok[r] * a.y_st + cu + 8 * c));
          at[e] = (long long)s_tok[r] * a.o_st + cu + 8 * c;
        }
      }
      float acc[4][4] = {};
      for (int k0 = 0; k0 < steps; k0 += KS) {
        if (steps > KS) weights(cu, k0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          if (k0 + ks < steps) {
            const uint8_t* p0 = s_h + (rt + g) * kRow + (16 * (k0 + ks) + 4 * c) * 2;
            const uint2 h0 = *reinterpret_cast<const uint2*>(p0), h1 = *reinterpret_cast<const uint2*>(p0 + 8 * kRow);
            const uint2 l0 = *reinterpret_cast<const uint2*>(p0 + 2 * rank), l1 = *reinterpret_cast<const uint2*>(p0 + 8 * kRow + 2 * rank);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              mma16816<T>(acc[j], h0.x, h1.x, h0.y, h1.y, b[ks][j].x, b[ks][j].y);
              mma16816<T>(acc[j], l0.x, l1.x, l0.y, l1.y, b[ks][j].x, b[ks][j].y);
            }
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = rt + g + 8 * e;
        if (r < m && in) {
          const float sc = rank ? s_scale[r] : 0.f;
          T* v = reinterpret_cast<T*>(&yv[e]);
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int q = 0; q < 2; ++q)
              if (rank) v[2 * j + q] = (T)fmaf(acc[j][2 * e + q], sc, (float)v[2 * j + q]);
          *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + at[e]) = yv[e];
        }
      }
    }
  }
}

// how d_in is split: few tokens in parts of kAD_KFew; many so that there are about six CTAs for every SM
static void adapter_split(int T, int d_in, int sms, int* splits, int* kper) {
  if (T <= kAD_Few) {
    *kper = kAD_KFew;
  } else {
    const int groups = (T + kAD_Group - 1) / kAD_Group, most = (d_in + 511) / 512;
    int s = (6 * sms + groups - 1) / groups;
    s = s < 1 ? 1 : s > most ? most : s;
    *kper = ((d_in + s - 1) / s + 63) / 64 * 64;
  }
  *splits = (d_in + *kper - 1) / *kper;
}

static long long adapter_groups(int T, int n) { return T / kAD_Group + (n + 1 < T ? n + 1 : T); }

template <typename T, int RM, int ST>
static int launch_shrink(const AdapterArgs& a, unsigned groups, cudaStream_t stream) {
  constexpr int smem = (kAD_Group + RM) * 128 * ST;
  const int rc = ensure_smem_attr((const void*)adapter_shrink_kernel<T, RM, ST>, smem);
  return rc ? rc : launch_early(adapter_shrink_kernel<T, RM, ST>, dim3(groups, a.splits), 256, smem, stream, a);
}

template <typename T>
static int launch_adapters(AdapterArgs a, int sms, cudaStream_t stream) {
  constexpr int kRow = kAD_MaxRank * 4 + 32;
  int rc;
  if (a.T <= kAD_Few) {
    rc = launch_early(adapter_shrink_few_kernel<T>, dim3(a.T, a.splits, a.rmax / 16), 256, 0, stream, a);
    if (rc) return rc;
    a.units = 2;
    return launch_early(adapter_expand_kernel<T, 16>, dim3(a.T, (a.d_out + 256 * a.units - 1) / (256 * a.units)), 256, 16 * kRow, stream, a);
  }
  const unsigned groups = (unsigned)adapter_groups(a.T, a.n);
  if ((rc = launch_early(adapter_route_kernel, dim3(1), 1024, (size_t)(2 * (a.n + 2)) * 4, stream, a))) return rc;
  rc = a.rmax <= 32 ? launch_shrink<T, 32, 6>(a, groups, stream)
       : a.rmax <= 64 ? launch_shrink<T, 64, 6>(a, groups, stream) : launch_shrink<T, 128, 4>(a, groups, stream);
  if (rc) return rc;
  // columns per CTA: h's parts are made once for all of them, but there have to be enough CTAs
  const long long real = (a.T + kAD_Group - 1) / kAD_Group;
  a.units = 4;
  while (a.units > 1 && real * ((a.d_out + 256 * a.units - 1) / (256 * a.units)) < 4LL * sms) a.units >>= 1;
  return launch_early(adapter_expand_kernel<T, 64>, dim3(groups, (a.d_out + 256 * a.units - 1) / (256 * a.units)), 256, 64 * kRow, stream, a);
}

}  // namespace bfb

using namespace bfb;

extern "C" {

size_t bf_adapter_workspace(int T, int n, int d_in, int rmax) {
  if (T <= 0 || n <= 0 || n > kAD_MaxAdapters || d_in <= 0 || rmax <= 0 || rmax > kAD_MaxRank) return 0;
  int splits, kper;
  adapter_split(T, d_in, 148, &splits, &kper);
  return 16 + (size_t)adapter_groups(T, n) * sizeof(int4) + ((size_t)T * 4 + 15) / 16 * 16 + (size_t)splits * T * rmax * 4;
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
  a.n = n; a.T = T; a.d_in = d_in; a.d_out = d_out; a.rmax = rmax;
  adapter_split(T, d_in, 148, &a.splits, &a.kper);
  uint8_t* p = static_cast<uint8_t*>(ws);
  a.n_groups = reinterpret_cast<int32_t*>(p);
  a.groups = reinterpret_cast<int4*>(p + 16);
  p += 16 + (size_t)adapter_groups(T, n) * sizeof(int4);
  a.perm = reinterpret_cast<int32_t*>(p);
  a.h = reinterpret_cast<float*>(p + ((size_t)T * 4 + 15) / 16 * 16);
  return dtype == BF_BF16 ? launch_adapters<__nv_bfloat16>(a, st.sm_count, stream) : launch_adapters<__half>(a, st.sm_count, stream);
}

}  // extern "C"
