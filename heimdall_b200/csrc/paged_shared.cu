// Attention of sequences that have pages in common, each shared page read once for all of them.
//
//   o_b = softmax over [the runs of shared pages on b's way, b's own tail]; every part gives (m, l, acc) for each row, joined as
//   o = sum 2^(m_i - M) acc_i / sum 2^(m_i - M) l_i.
//
// A run of pages that `count` sequences share is met by count * t * R rows of queries per KV head at once, 128 of them to a tile of the
// tensor core; a tail is a run of one sequence.  A tile of 128 tokens is 64 KB from HBM per KV head, 2900 cycles of an SM's share, and with 128
// rows 2048 cycles of 8-bit products, however many of the rows are there: bound by HBM while a row block is alone with its pages, by the
// tensor core when several share them through L2.
// The e4m3 codes go untouched from TMA to the products (kind::f8f6f4); the other operands are split into e4m3 parts that add up, x = x0 + x1 (+ x2
// in fp16), so that a product's parts accumulate in one place:
//   S[row, token] = sum_p Q_p K^T     M = 128 rows, N = 128 tokens, K = 256 dims x parts
//   O[row, dim]   = sum_p P_p V       M = 128 rows, N = 2 x 128 dims, K = 128 tokens x parts      (P in TMEM over S; V as it lies: N-major)
// Two parts hold 9 bits, three 13.  A query's row is scaled to [128, 256), a weight to its row's largest in the tile = 256: the parts end at 2^-9
// of that scale, so a component is off by at most 2^-17 of its row's largest, a weight by 2^-18 of the tile's largest (weights beside a
// heavy token of another tile keep their bits: every tile's O is scaled for itself and added up in registers, in fp32).
// V's power-of-two scales join the exponents: w = 2^(s + log2 sv - m) with m their largest, and the sum of weights takes 1 / sv back.
//
// Kernels: paged_queries_kernel makes the query parts, paged_shared_kernel the partials, paged_merge_kernel the output, in a fixed order.
// Work of the second: the tiles of all (run or tail, KV head, row block) in one line, cut into equal pieces, one CTA per SM; an item's start counts as
// kSH_Start tiles.
// Warps: 0 the walk along the line, TMA of the queries and of K; 1 the products S; 2 TMA of V; 3 the products O; two warpgroups of softmax (thread = row
// and half of the tokens: what a tile waits for is one thread's way through its scores, 4600 cycles for all 128); two of accumulators (thread = row and half of the dims).  What the others have to know of a tile (pages, scales, where
// an item begins and ends) comes from warp 0 through a ring of four entries.
#include "bifrost_b200.h"
#include "capi_internal.h"
#include "common.cuh"
#include "launch_early.h"
#include "paged_kv.h"
#include "tmap.h"

namespace bfb {

constexpr int kSH_MaxCtas = 160;
constexpr int kSH_MaxGroup = 24;                     // query heads per KV head, as attend
constexpr int kSH_M = 128, kSH_N = 128;              // rows, tokens of a tile
constexpr int kSH_Unit = 128 * 128;                  // bytes of half a K or V tile: 128 tokens, 128 dims
constexpr int kSH_Threads = 640;
constexpr int kSH_Start = 1;
constexpr int kSH_Ways = kPS_Depth + 1;              // pieces of the line that a sequence can have
// register split (setmaxnreg) of the 96 per thread at launch
constexpr uint32_t kSH_RegsCtl = 48, kSH_RegsSoftmax = 64, kSH_RegsAcc = 152;
static_assert(kSH_RegsCtl + 2 * kSH_RegsSoftmax + 2 * kSH_RegsAcc <= 5 * 96, "register split");

template <typename T>
struct SharedCfg {
  static constexpr int Parts = 3, NK = 4, NV = 3;    // half tiles of K and V that fit beside the queries
};
template <>
struct SharedCfg<__nv_bfloat16> {
  static constexpr int Parts = 2, NK = 4, NV = 4;
};

// what a tile's roles have to know of it
struct SharedTile {
  float ks[8], e[8], inv[8];      // its pages' K scales, V scales' exponents and inverses
  int prow[8];                    // rows of its pages in the codes' tensor map
  unsigned have;                  // which pages are there
  int valid;                      // tokens that the sequences have
  long long pos0;                 // position of its first token
  int first, last, item;          // first and last of its item in this CTA, the item's number
  int rows, base;                 // of the item: rows, rows of the pieces before it
  int row0, from;                 // its first row among its run's, its first row among the KV head's
  int stop, pad[2];               // no more tiles
};
template <typename T>
struct SharedSmem {
  using C = SharedCfg<T>;
  static constexpr int Q = C::Parts * 2 * kSH_Unit;
  static constexpr int Tiles = (C::NK + C::NV) * kSH_Unit + Q;
  static constexpr int Bytes = Tiles + 512 + 4 * (int)sizeof(SharedTile) + 8 * kSH_M * 8 + 1024;
};
static_assert(SharedSmem<__half>::Bytes <= 232448 && SharedSmem<__nv_bfloat16>::Bytes <= 232448, "shared memory");

// where a run, or a tail, lies in the line, for the sequence at a place that has it
struct SharedWay {
  int unit, before;     // its first unit, the rows before it
  int rows, tiles;      // its rows per KV head, its tiles (0: no pieces)
  int first, pad[3];    // its first place
};
struct SharedArgs {
  PagePool p;
  const void* q;
  long long q_sb, q_st, q_sh;
  const int32_t* plan;
  int n, t, H, R;
  int page_log, cap;    // cap: tokens that the table has room for
  float c2;             // scale * log2(e)
  uint8_t* qp;          // [KV heads][n t R rows, in the plan's order][parts][256]
  float* qs;            // [KV heads][n t R] the rows' scales
  int4* head;           // units per CTA, CTAs with one more, -, -
  SharedWay* ways;      // [n places][kSH_Ways]: the tail, then the runs
  float* part;          // [CTAs * 128 + rows][256], a piece as [64][rows][4 dims]
  float2* ml;           // [CTAs * 128 + rows] maximum, sum
  void* o;
  float* lse;
  unsigned int* err;
};

// the plan's arrays
struct Plan {
  const int32_t *slots, *order, *last, *skip, *runs;
  int n_runs;
  __device__ __forceinline__ Plan(const int32_t* p, int n, int runs_said)
      : slots(p + kPS_Head), order(slots + n), last(order + 2 * (size_t)n), skip(last + n), runs(skip + n), n_runs(min(max(runs_said, 0), n)) {}
};

// a piece of the line: run e, or, behind the runs, the tail of the sequence at place e - n_runs
struct Stretch {
  int first, rows, page0, tokens, lead;      // first place; lead: the slot whose table names its pages
  Stretch() = default;
  __device__ __forceinline__ Stretch(const SharedArgs& a, const Plan& pl, int e) {
    if (e < pl.n_runs) {
      const int32_t* r = pl.runs + (size_t)e * kPS_Run;
      first = r[0];
      rows = r[1] * a.t * a.R;
      page0 = r[2];
      tokens = (r[3] - r[2]) << a.page_log;
      lead = pl.slots[pl.order[first]];
    } else {
      first = e - pl.n_runs;
      const int b = pl.order[first], slot = pl.slots[b];
      rows = a.t * a.R;
      page0 = pl.skip[b];
      lead = slot;
      tokens = slot >= 0 && slot < a.p.slots ? max(0, min(a.p.lens[slot], a.cap) - (page0 << a.page_log)) : 0;
    }
  }
  __device__ __forceinline__ int tiles() const { return (tokens + kSH_N - 1) / kSH_N; }
  __device__ __forceinline__ int blocks() const { return (rows + kSH_M - 1) / kSH_M; }
  __device__ __forceinline__ int units(int heads) const { return tokens > 0 ? heads * blocks() * (tiles() + kSH_Start) : 0; }
};

__device__ __forceinline__ uint16_t to_e4m3(__half2 x) {      // two values
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(*reinterpret_cast<uint32_t*>(&x)));
  return r;
}
__device__ __forceinline__ __half2 from_e4m3(uint16_t x) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(x));
  return *reinterpret_cast<__half2*>(&r);
}

// The query parts: a warp a row, in the order of the plan's places, lane l dims 8 l .. 8 l + 7.
template <typename T>
__global__ void __launch_bounds__(256) paged_queries_kernel(SharedArgs a) {
  constexpr int Parts = SharedCfg<T>::Parts;
  wait_then_let_next_start();
  const int lane = threadIdx.x & 31, g = blockIdx.y, per_seq = a.t * a.R;
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), rows = (long long)a.n * per_seq;
  if (row >= rows) return;
  const Plan pl(a.plan, a.n, a.plan[0]);
  const int place = (int)(row / per_seq), rem = (int)(row - (long long)place * per_seq), i = rem / a.R, h = g * a.R + rem - i * a.R;
  const uint4 raw = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + pl.order[place] * a.q_sb + i * a.q_st + h * a.q_sh + 8 * lane);
  const uint32_t v[4] = {raw.x, raw.y, raw.z, raw.w};
  // the largest value of the row, as 16-bit patterns without their sign
  const uint32_t m2 = __vmaxu2(__vmaxu2(v[0] & 0x7fff7fffu, v[1] & 0x7fff7fffu), __vmaxu2(v[2] & 0x7fff7fffu, v[3] & 0x7fff7fffu));
  const uint32_t m = __reduce_max_sync(0xffffffffu, max(m2 & 0xffffu, m2 >> 16));
  const uint16_t m16 = (uint16_t)m;
  const float mf = (float)*reinterpret_cast<const T*>(&m16);
  const bool fin = mf < INFINITY;          // false for NaN too
  const int ex = mf > 0.f ? max((int)(__float_as_uint(mf) >> 23), 16) : 127;
  const float up = fin ? __uint_as_float((uint32_t)(254 + 7 - ex) << 23) : 0.f;      // to [128, 256)
  uint16_t c[4][Parts];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const T* e = reinterpret_cast<const T*>(&v[k]);
    // parts that add up; each remainder is exact in fp16
    __half2 x = __floats2half2_rn(fin ? (float)e[0] * up : 0.f, fin ? (float)e[1] * up : 0.f);
#pragma unroll
    for (int p = 0; p < Parts; ++p) {
      c[k][p] = to_e4m3(x);
      x = __hsub2(x, from_e4m3(c[k][p]));
    }
  }
  const size_t at = (size_t)g * rows + row;
#pragma unroll
  for (int p = 0; p < Parts; ++p)
    reinterpret_cast<uint2*>(a.qp + (at * Parts + p) * kPG_D)[lane] = make_uint2(c[0][p] | ((uint32_t)c[1][p] << 16), c[2][p] | ((uint32_t)c[3][p] << 16));
  // a row with a value that is not finite has no finite scores
  if (lane == 0) a.qs[at] = fin ? __uint_as_float((uint32_t)(ex - 7) << 23) * a.c2 : NAN;
}

// Barriers and the abort word by their addresses in shared memory: through pointers every one of the many uses makes its address anew.
struct Bar {
  uint32_t at;
  __device__ __forceinline__ Bar operator+(int i) const { return Bar{at + 8u * i}; }
  __device__ __forceinline__ void init(uint32_t count) const { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(at), "r"(count) : "memory"); }
  __device__ __forceinline__ void arrive() const { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(at) : "memory"); }
  __device__ __forceinline__ void expect(uint32_t bytes) const {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(at), "r"(bytes) : "memory");
  }
  __device__ __forceinline__ void commit() const {      // arrive once this thread's products so far are done
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(at) : "memory");
  }
};
struct Waits {
  uint32_t abort;          // the address of the CTA's abort word
  __device__ __forceinline__ int aborted() const {
    int x;
    asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(x) : "r"(abort) : "memory");
    return x;
  }
  // as mbar_wait_warp_small
  __device__ __forceinline__ bool operator()(Bar bar, uint32_t parity, int site) const {
    bool ok = mbar_try_wait(bar.at, parity);
    if (!ok) {
      const long long t0 = clock64();
#pragma unroll 1
      while (!(ok = mbar_try_wait(bar.at, parity)) && !aborted()) {
        if (clock64() - t0 > kWaitCycles) asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(abort), "r"(site) : "memory");
      }
    }
    return __all_sync(0xffffffffu, ok) != 0;
  }
};
__device__ __forceinline__ void load_2d(uint32_t dst, const void* tmap, Bar bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar.at), "r"(c0), "r"(c1) : "memory");
}

// D[tmem] (+)= A[tmem] * B[smem desc], 8-bit operands: row m of A in lane m, four values to a 32-bit column, 8 columns to a step of K = 32
__device__ __forceinline__ void umma_f8_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
__device__ __forceinline__ uint64_t scale2(uint64_t a, float f) { return pair2(lo_hi(a, 0) * f, lo_hi(a, 1) * f); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

template <typename T>
__global__ void __launch_bounds__(kSH_Threads, 1)
    paged_shared_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ CUtensorMap qmap,
                        SharedArgs a) {
  using C = SharedCfg<T>;
  constexpr int Parts = C::Parts, NK = C::NK, NV = C::NV;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));   // K's half tiles, then V's
  uint8_t* sQ = ring + (NK + NV) * kSH_Unit;           // [parts][2 atoms][128 rows][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sQ + SharedSmem<T>::Q);
  const Bar k_full{smem_u32(bars)}, k_empty = k_full + 4, v_full = k_full + 8, v_empty = k_full + 12, s_full = k_full + 16, p_full = k_full + 18,
            p_free = k_full + 20, o_free = k_full + 22, o_full = k_full + 24, q_full = k_full + 25, q_free = k_full + 26, t_full = k_full + 28,
            t_free = k_full + 32, met = k_full + 60;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 36);
  volatile int* abort = reinterpret_cast<volatile int*>(bars + 37);
  const Waits wait{smem_u32(bars + 37)};
  const uint32_t ring_at = smem_u32(ring), q_at = smem_u32(sQ);
  int* s_sum = reinterpret_cast<int*>(bars + 38);      // [16][2] totals of the warps that scan
  Stretch* s_first = reinterpret_cast<Stretch*>(bars + 54);       // the stretch that this CTA begins in
  int* s_start = reinterpret_cast<int*>(bars + 58);    // stretch, unit in it, rows before it; the plan's runs
  SharedTile* s_tile = reinterpret_cast<SharedTile*>(bars + 64);  // [4]
  float2* s_ml = reinterpret_cast<float2*>(s_tile + 4);           // [4][2][128] a tile's maxima and sums, of both halves of its tokens
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < 4; ++i) {
      (k_full + i).init(1);
      (k_empty + i).init(1);
      (v_full + i).init(1);
      (v_empty + i).init(1);
      (t_full + i).init(1);
      (t_free + i).init(19);       // V, S, O, eight of softmax, eight accumulators
    }
    for (int i = 0; i < 2; ++i) {
      (s_full + i).init(1);
      (p_full + i).init(8);
      (p_free + i).init(1);
      (o_free + i).init(8);
    }
    o_full.init(1);
    q_full.init(1);
    q_free.init(1);
    for (int i = 0; i < 4; ++i) (met + i).init(2);       // the two warps of softmax that have the same rows
    *abort = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch(&kmap);
    tma_prefetch(&qmap);
  }
  if (warp == 2 && lane == 0) tma_prefetch(&vmap);
  let_next_start();
  if (tid == 96) s_start[3] = acquire_early(a.plan);
  __syncthreads();
  // this CTA's part of the line: the stretches' units summed over the warps of softmax and accumulators, thread i holding `per` consecutive ones.  (The plan and
  // the lengths are older than the kernel before this one: launch_early.h.)
  constexpr int kScan = kSH_Threads - 128;
  const Plan pl(a.plan, a.n, s_start[3]);
  const int stretches = pl.n_runs + a.n, per = (stretches + kScan - 1) / kScan, e0 = (tid - 128) * per;
  Stretch mine0;                       // thread's first
  int2 mine = make_int2(0, 0);
  if (warp >= 4) {
    for (int i = 0; i < per && e0 + i < stretches; ++i) {
      const Stretch x(a, pl, e0 + i);
      if (i == 0) mine0 = x;
      mine.x += x.units(a.p.heads);
      mine.y += x.rows * a.p.heads;
    }
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
  if (warp >= 4 && lane == 31) {
    s_sum[2 * (warp - 4)] = incl.x;
    s_sum[2 * (warp - 4) + 1] = incl.y;
  }
  __syncthreads();
  int total = lane < kScan / 32 ? s_sum[2 * lane] : 0;
  const int rows_w = lane < kScan / 32 ? s_sum[2 * lane + 1] : 0;
  int2 before = make_int2(lane < warp - 4 ? total : 0, lane < warp - 4 ? rows_w : 0);
  total = (int)__reduce_add_sync(0xffffffffu, (unsigned)total);
  before.x = (int)__reduce_add_sync(0xffffffffu, (unsigned)before.x) + incl.x - mine.x;
  before.y = (int)__reduce_add_sync(0xffffffffu, (unsigned)before.y) + incl.y - mine.y;
  const int ctas = max(1, min(total, (int)gridDim.x)), each = total / ctas, more = total - each * ctas;
  const int u0 = min((int)blockIdx.x, ctas) * each + min((int)blockIdx.x, more);
  const int u1 = u0 + ((int)blockIdx.x < ctas ? each + ((int)blockIdx.x < more ? 1 : 0) : 0);
  if (warp >= 4 && u0 < u1 && before.x <= u0 && u0 < before.x + mine.x) {
    int2 at = before;
    for (int i = 0; i < per && e0 + i < stretches; ++i) {
      const Stretch x = i == 0 ? mine0 : Stretch(a, pl, e0 + i);
      const int units = x.units(a.p.heads);
      if (at.x <= u0 && u0 < at.x + units) {
        s_start[0] = e0 + i;
        s_start[1] = u0 - at.x;
        s_start[2] = at.y;
        *s_first = x;
      }
      at.x += units;
      at.y += x.rows * a.p.heads;
    }
  }
  wait_for_stream();
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  if (warp >= 4) {
    // for paged_merge_kernel: every CTA writes some stretches' part
    int2 at = before;
    for (int i = 0; i < per; ++i) {
      const int e = e0 + i;
      if (e >= stretches) break;
      const bool here = e % (int)gridDim.x == (int)blockIdx.x;
      if (!here && per == 1) break;
      const Stretch x = i == 0 ? mine0 : Stretch(a, pl, e);
      if (here) {
        const bool run = e < pl.n_runs;
        const int32_t* r = pl.runs + (size_t)e * kPS_Run;
        const int k = run ? 1 + r[5] : 0, many = run ? r[1] : 1, tiles = x.tiles();
        for (int i = 0; i < many; ++i) {
          int4* to = reinterpret_cast<int4*>(a.ways + (size_t)(x.first + i) * kSH_Ways + k);
          to[0] = make_int4(at.x, at.y, x.rows, tiles);
          to[1] = make_int4(x.first, 0, 0, 0);
        }
        if (!run) {                                     // and that there are no more than its sequence's runs
          const int last = pl.last[pl.order[x.first]];
          for (int i = last >= 0 ? 2 + pl.runs[(size_t)last * kPS_Run + 5] : 1; i < kSH_Ways; ++i) a.ways[(size_t)x.first * kSH_Ways + i].tiles = 0;
        }
      }
      at.x += x.units(a.p.heads);
      at.y += x.rows * a.p.heads;
    }
    if (blockIdx.x == 0 && tid == 128) *a.head = make_int4(each, more, 0, 0);
    __syncwarp();
  }
  const int L = a.p.page, ppt = kSH_N >> a.page_log, per_seq = a.t * a.R;
  bool ok = true;
  // every role: wait for tile j's entry (false: no more tiles, or a wait gave up)
  auto tile = [&](int j) {
    ok = wait(t_full + (j & 3), (j >> 2) & 1, 0x90);
    return ok && !s_tile[j & 3].stop;
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kSH_RegsCtl));
    if (warp == 0) {
      // ---------------------------------------------------------------- the walk, the queries, K
      int j = 0, u = 0, uphase = 1, used = 0, items = 0, unit = u0;
      if (u0 < u1) {
        int e = s_start[0], base = s_start[2], in = s_start[1];
#pragma unroll 1
        for (; e < stretches && unit < u1 && ok; ++e) {
          const Stretch x = e == s_start[0] ? *s_first : Stretch(a, pl, e);
          const int ntiles = x.tiles(), len = ntiles + kSH_Start, blocks = x.blocks(), n_items = x.tokens > 0 ? a.p.heads * blocks : 0;
          const int pages = (x.tokens + L - 1) >> a.page_log;
          const int32_t* table = a.p.table + (size_t)max(x.lead, 0) * a.p.width + x.page0;
          int item = in / len;
          in -= item * len;
#pragma unroll 1
          for (; item < n_items && unit < u1 && ok; ++item) {
            const int g = item / blocks, rb = item - g * blocks;
            int k = max(in - kSH_Start, 0);
            unit += max(kSH_Start - in, 0);                    // the units before its first tile
            in = 0;
            const int k1 = min(ntiles, k + u1 - unit);
            if (k >= k1) continue;
            unit += k1 - k;
            if (items && !(ok = wait(q_free, (items - 1) & 1, 0x91))) break;
            ++items;
            const int from = g * a.n * per_seq + x.first * per_seq + rb * kSH_M;
            if (lane == 0) q_full.expect(Parts * 2 * kSH_Unit);
            __syncwarp();
            if (elect_one()) {
#pragma unroll
              for (int p = 0; p < 2 * Parts; ++p) load_2d(q_at + p * kSH_Unit, &qmap, q_full, p * 128, from);
            }
            __syncwarp();
            // lane i: page i of the tile, loaded a tile ahead
            auto page_of = [&](int k) {
              const int i = k * ppt + lane;
              if (lane >= ppt || k >= k1 || i >= pages || x.page0 + i >= a.p.width) return -1;
              const int page = table[i];
              return page >= 0 && page < a.p.pages ? page : -1;
            };
            int page = page_of(k);
#pragma unroll 1
            for (int f = k; k < k1; ++k, ++j) {
              const int next = page_of(k + 1);
              const bool there = page >= 0;
              const unsigned have = __ballot_sync(0xffffffffu, there);
              const int row = there ? (page * a.p.heads + g) * L : 0;
              float ks = 1.f;
              int ex = 0;
              if (there) {
                ks = a.p.ks[(size_t)page * a.p.heads + g];
                // scales are powers of two, 2^-64 at least; 0 where nothing was written, whose codes are 0 too: any scale does, but its inverse times 2^8,
                // summed over the tokens, has to stay in fp32
                const int e8 = (int)(__float_as_uint(a.p.vs[(size_t)page * a.p.heads + g]) >> 23);
                ex = e8 ? max(e8 - 127, -110) : -64;
              }
              if (j >= 4 && !(ok = wait(t_free + (j & 3), ((j >> 2) - 1) & 1, 0x92))) break;
              SharedTile* d = s_tile + (j & 3);
              if (lane < 8) {
                d->ks[lane] = ks;
                d->e[lane] = (float)ex;
                d->inv[lane] = __uint_as_float((uint32_t)(127 - ex) << 23);
                d->prow[lane] = row;
              }
              if (lane == 0) {
                d->have = have;
                d->valid = min(x.tokens - k * kSH_N, kSH_N);
                d->pos0 = ((long long)x.page0 << a.page_log) + (long long)k * kSH_N;
                d->first = k == f;
                d->last = k + 1 == k1;
                d->item = items;
                d->rows = min(kSH_M, x.rows - rb * kSH_M);
                d->base = base + g * x.rows + rb * kSH_M;
                d->row0 = x.first * per_seq + rb * kSH_M;
                d->from = from;
                d->stop = 0;
              }
              __syncwarp();
              if (lane == 0) (t_full + (j & 3)).arrive();
#pragma unroll 1
              for (int half = 0; half < 2; ++half) {
                if (used >= NK && !(ok = wait(k_empty + u, uphase, 0x93))) break;
                if (lane == 0) {
                  if (have) (k_full + u).expect((uint32_t)__popc(have) * L * 128); else (k_full + u).arrive();
                }
                __syncwarp();
#pragma unroll 1
                for (int i = 0; i < ppt; ++i) {
                  const int r = __shfl_sync(0xffffffffu, row, i);
                  if (((have >> i) & 1u) && elect_one()) load_2d(ring_at + u * kSH_Unit + i * L * 128, &kmap, k_full + u, 128 * half, r);
                  __syncwarp();
                }
                ++used;
                if (++u == NK) {
                  u = 0;
                  uphase ^= 1;
                }
              }
              if (!ok) break;
              page = next;
            }
          }
          base += x.rows * a.p.heads;
          in = 0;
        }
      }
      // the end of the line
      if (ok && (j < 4 || (ok = wait(t_free + (j & 3), ((j >> 2) - 1) & 1, 0x92)))) {
        if (lane == 0) {
          s_tile[j & 3].stop = 1;
          (t_full + (j & 3)).arrive();
        }
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- S = sum_p Q_p K^T
      constexpr uint32_t id = idesc_e4m3(kSH_M, kSH_N);
      const uint64_t dk0 = sdesc_sw128(ring_at), dq0 = sdesc_sw128(q_at);
      int u = 0, uphase = 0, items = 0;
#pragma unroll 1
      for (int j = 0; tile(j); ++j) {
        const int s = j & 1;
        const bool first = s_tile[j & 3].first, last = s_tile[j & 3].last;
        __syncwarp();
        if (lane == 0) (t_free + (j & 3)).arrive();
        if (first && !(ok = wait(q_full, items & 1, 0x94))) break;
        items += first;
        // tile j - 2's weights, which lie over S, have been read
        if (j >= 2 && !(ok = wait(p_free + s, ((j >> 1) - 1) & 1, 0x95))) break;
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          if (!(ok = wait(k_full + u, uphase, 0x97))) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t dk = dk0 + (uint32_t)(u * (kSH_Unit >> 4));
#pragma unroll
            for (int p = 0; p < Parts; ++p)
#pragma unroll
              for (int ks = 0; ks < 4; ++ks)
                umma_f8_ss(tmem + s * kSH_N, dq0 + (uint32_t)((p * 2 + half) * (kSH_Unit >> 4) + ks * 2), dk + ks * 2, id, half > 0 || p > 0 || ks > 0);
            (k_empty + u).commit();
            if (half) {
              (s_full + s).commit();
              if (last) q_free.commit();
            }
          }
          __syncwarp();
          if (++u == NK) {
            u = 0;
            uphase ^= 1;
          }
        }
        if (!ok) break;
      }
    } else if (warp == 2) {
      // ---------------------------------------------------------------- V
      int u = 0, uphase = 1, used = 0;
#pragma unroll 1
      for (int j = 0; tile(j); ++j) {
        const unsigned have = s_tile[j & 3].have;
        const int row = s_tile[j & 3].prow[lane & 7];
        __syncwarp();
        if (lane == 0) (t_free + (j & 3)).arrive();
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          if (used >= NV && !(ok = wait(v_empty + u, uphase, 0x98))) break;
          if (lane == 0) {
            if (have) (v_full + u).expect((uint32_t)__popc(have) * L * 128); else (v_full + u).arrive();
          }
          __syncwarp();
#pragma unroll 1
          for (int i = 0; i < ppt; ++i) {
            const int r = __shfl_sync(0xffffffffu, row, i);
            if (((have >> i) & 1u) && elect_one()) load_2d(ring_at + (NK + u) * kSH_Unit + i * L * 128, &vmap, v_full + u, 128 * half, r);
            __syncwarp();
          }
          ++used;
          if (++u == NV) {
            u = 0;
            uphase ^= 1;
          }
        }
        if (!ok) break;
      }
    } else {
      // ---------------------------------------------------------------- O = sum_p P_p V
      constexpr uint32_t id = idesc_e4m3(kSH_M, 128) | kIdescBMn;
      const uint64_t dv0 = sdesc_sw128_mn(ring_at + NK * kSH_Unit, 16384);
      int u = 0, uphase = 0;
#pragma unroll 1
      for (int j = 0; tile(j); ++j) {
        const int s = j & 1;
        __syncwarp();
        if (lane == 0) (t_free + (j & 3)).arrive();
        if (!(ok = wait(p_full + s, (j >> 1) & 1, 0x99))) break;
        if (j >= 1 && !(ok = wait(o_free + (s ^ 1), ((j - 1) >> 1) & 1, 0x9a))) break;
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          if (!(ok = wait(v_full + u, uphase, 0x9b))) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t dv = dv0 + (uint32_t)(u * (kSH_Unit >> 4));
#pragma unroll
            for (int p = 0; p < Parts; ++p)
#pragma unroll
              for (int ks = 0; ks < 4; ++ks)
                umma_f8_ts(tmem + 256 + half * 128, tmem + s * kSH_N + 32 * ks + 8 * p, dv + ks * (4096 >> 4), id, p > 0 || ks > 0);
            (v_empty + u).commit();
            if (half) {
              (p_free + s).commit();
              o_full.commit();
            }
          }
          __syncwarp();
          if (++u == NV) {
            u = 0;
            uphase ^= 1;
          }
        }
        if (!ok) break;
      }
    }
  } else {
    const int wq = warp & 3, r = wq * 32 + lane;      // this thread's row
    if (warp < 12) {
      // ---------------------------------------------------------------- softmax: thread = row and half of the tokens
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kSH_RegsSoftmax));
      const int hh = (warp - 4) >> 2, c0 = 64 * hh;
      float qs = 0.f;
      int limit = -1, rows = 0, item = 0;            // the last position that the row sees
      uint32_t meetings = 0;
#pragma unroll 1
      for (int j = 0; tile(j); ++j) {
        const int s = j & 1;
        const uint32_t trow = tmem + ((uint32_t)(wq * 32) << 16) + s * kSH_N;
        const SharedTile& d = s_tile[j & 3];
        if (d.item != item) {
          item = d.item;
          rows = d.rows;
          limit = -1;
          if (r < rows) {
            const int idx = d.row0 + r, place = idx / per_seq;
            const int slot = pl.slots[pl.order[place]];
            if (slot >= 0 && slot < a.p.slots) limit = a.p.lens[slot] - a.t + (idx - place * per_seq) / a.R;
            qs = a.qs[d.from + r];
          }
        }
        const unsigned have = d.have;
        const int valid = d.valid;
        // the row sees the tile's first `vis` tokens, of pages that are there
        const int vis = (int)max(min((long long)limit - d.pos0 + 1, (long long)valid), 0ll);
        const bool whole = valid == kSH_N && have == (1u << ppt) - 1u, busy = wq * 32 < rows;
        const bool all = whole && __all_sync(0xffffffffu, vis == kSH_N || r >= rows);
        if (!whole) {
          // the values of tokens that are not there may be anything (a weight of 0 times NaN would be NaN): zeros
          const int n = 2 * j + hh, u = n % NV;
          // half n - NV was in this place before, of tile j - 2 (four places) or j - 1 (three): while it is on its way, a wait for half n would take n - 2 NV
          // for it.  (The products of tile j - 3 are done: the scores of tile j - 1 were there.)
          constexpr int kBefore = NV < 4 ? 1 : 2;
          if (j >= kBefore && !(ok = wait(p_free + ((j - kBefore) & 1), ((j - kBefore) >> 1) & 1, 0xa4))) break;
          if (!(ok = wait(v_full + u, (n / NV) & 1, 0x9c))) break;
          if (r >= valid || !((have >> (r >> a.page_log)) & 1u)) {
            uint4* row = reinterpret_cast<uint4*>(ring + (NK + u) * kSH_Unit + r * 128);
#pragma unroll
            for (int i = 0; i < 8; ++i) row[(i + r) & 7] = make_uint4(0u, 0u, 0u, 0u);     // rows are as long as all banks
          }
          fence_async_smem();
        }
        if (!(ok = wait(s_full + s, (j >> 1) & 1, 0x9d))) break;
        tc_fence_after();
        if (busy) {
          if (!all) {
            // scores of what the row does not see: -infinity, in a way of its own (in the loops below it would cost every tile)
#pragma unroll 1
            for (int c = c0; c < c0 + 64; c += 16) {
              uint32_t x[16];
              tmem_ld16(trow + c, x);
              tmem_wait_ld();
              const int seen = (have >> (c >> a.page_log)) & 1u ? vis - c : 0;
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (i >= seen) x[i] = 0xff800000u;
              tmem_st16(trow + c, x);
            }
            tmem_wait_st();
          }
          // two ways through the row's scores (they do not fit the registers): its largest, then the weights
          float mt = -INFINITY, lt = 0.f;
#pragma unroll 1
          for (int c = c0; c < c0 + 64; c += 32) {
            uint32_t x[32];
            tmem_ld32(trow + c, x);
            tmem_wait_ld();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              float m0 = __uint_as_float(x[16 * q]), m1 = __uint_as_float(x[16 * q + 1]);
#pragma unroll
              for (int i = 2; i < 16; i += 4) {
                m0 = fmaxf(fmaxf(m0, __uint_as_float(x[16 * q + i])), __uint_as_float(x[16 * q + i + 1]));
                if (i + 2 < 16) m1 = fmaxf(fmaxf(m1, __uint_as_float(x[16 * q + i + 2])), __uint_as_float(x[16 * q + i + 3]));
              }
              const int pi = (c + 16 * q) >> a.page_log;
              mt = fmaxf(mt, fmaf(fmaxf(m0, m1), d.ks[pi] * qs, d.e[pi]));
            }
          }
          // the row's maximum of both halves (the two warps of these rows meet)
          float2* ml = s_ml + (j & 3) * 2 * kSH_M + r;
          ml[hh * kSH_M].x = mt;
          __syncwarp();
          if (lane == 0) (met + wq).arrive();
          if (!(ok = wait(met + wq, meetings++ & 1, 0xa3))) break;
          mt = fmaxf(mt, ml[(hh ^ 1) * kSH_M].x);
          const float ref = 8.f - (mt == -INFINITY ? 0.f : mt);       // the largest weight becomes 2^8
          // 16 tokens at a time, the next 16 scores on their way; every step for all of them before the next one, a value's own way through the
          // steps takes 60 cycles
          uint32_t x[16];
          tmem_ld16(trow + c0, x);
          tmem_wait_ld();
#pragma unroll 1
          for (int c = c0; c < c0 + 64; c += 16) {
            const int pi = c >> a.page_log;
            // (never 0, which would make NaN of the -infinity of what the row does not see; 2^25 times 1e-38 is nothing to a score)
            const float f = fmaf(d.ks[pi], qs, 1e-38f), off = d.e[pi] + ref;
            const uint64_t f2 = pair2(f, f), off2 = pair2(off, off);
            float w[16];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint64_t y = fma2(pair2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), f2, off2);
              w[2 * i] = lo_hi(y, 0);
              w[2 * i + 1] = lo_hi(y, 1);
            }
            if (c + 16 < c0 + 64) tmem_ld16(trow + c + 16, x);
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = ex2_approx(w[i]);
            uint64_t sum = 0;
            __half2 h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              sum = add2(sum, pair2(w[2 * i], w[2 * i + 1]));
              h[i] = __floats2half2_rn(w[2 * i], w[2 * i + 1]);
            }
            lt = fmaf(lo_hi(sum, 0) + lo_hi(sum, 1), d.inv[pi], lt);
            uint32_t out[Parts][4];
#pragma unroll
            for (int p = 0; p < Parts; ++p) {
              uint16_t e[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) e[i] = to_e4m3(h[i]);
#pragma unroll
              for (int i = 0; i < 4; ++i) out[p][i] = e[2 * i] | ((uint32_t)e[2 * i + 1] << 16);
              if (p + 1 < Parts) {
#pragma unroll
                for (int i = 0; i < 8; ++i) h[i] = __hsub2(h[i], from_e4m3(e[i]));
              }
            }
            // the tokens' parts take the place of scores that have been read: of 32 tokens in the columns of those
            tmem_wait_ld();
#pragma unroll
            for (int p = 0; p < Parts; ++p) tmem_st4(trow + (c & ~31) + 8 * p + ((c >> 2) & 4), out[p]);
          }
          tmem_wait_st();
          ml[hh * kSH_M].y = lt;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          (t_free + (j & 3)).arrive();
          (p_full + s).arrive();
        }
      }
    } else {
      // ---------------------------------------------------------------- accumulators: thread = row, half of the dims
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSH_RegsAcc));
      const int half = (warp - 12) >> 2;
      const uint32_t trow = tmem + 256 + half * 128 + ((uint32_t)(wq * 32) << 16);
      uint64_t acc[64];
      float m_ref = -INFINITY, l = 0.f;
#pragma unroll
      for (int i = 0; i < 64; ++i) acc[i] = 0;
#pragma unroll 1
      for (int j = 0; tile(j); ++j) {
        const int rows = s_tile[j & 3].rows, base = s_tile[j & 3].base;
        const bool end = s_tile[j & 3].last, busy = wq * 32 < rows;
        if (s_tile[j & 3].first) {       // (zeroed at the end of an item instead, the compiler keeps the accumulators twice)
          m_ref = -INFINITY;
          l = 0.f;
#pragma unroll
          for (int i = 0; i < 64; ++i) acc[i] = 0;
        }
        if (!(ok = wait(p_full + (j & 1), (j >> 1) & 1, 0x9e))) break;      // the tile's maxima
        float2 t = make_float2(-INFINITY, 0.f);
        if (busy) {
          const float2 *ml = s_ml + (j & 3) * 2 * kSH_M + r, t0 = ml[0], t1 = ml[kSH_M];
          t = make_float2(fmaxf(t0.x, t1.x), t0.y + t1.y);
        }
        __syncwarp();
        if (lane == 0) (t_free + (j & 3)).arrive();      // the entry and the maxima may be written over
        // the accumulators are relative to the first tile's maximum, until one is 2^40 times it: then to that
        if (t.x > m_ref + 40.f) {
          const float al = m_ref == -INFINITY ? 0.f : ex2_approx(m_ref - t.x);
          l *= al;
#pragma unroll
          for (int i = 0; i < 64; ++i) acc[i] = scale2(acc[i], al);
          m_ref = t.x;
        }
        // (a tile without a maximum holds zeros, or NaN to be passed on)
        const float ff = t.x == -INFINITY ? 1.f / 256.f : ex2_approx(t.x - m_ref) * (1.f / 256.f);
        l = fmaf(t.y, ff, l);
        const uint64_t f = pair2(ff, ff);
        if (!(ok = wait(o_full, j & 1, 0x9f))) break;
        tc_fence_after();
        if (busy) {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint32_t x[16];
            tmem_ld16(trow + 16 * c, x);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 8; ++i)
              acc[8 * c + i] = fma2(pair2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), f, acc[8 * c + i]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) (o_free + (j & 1)).arrive();
        if (end) {
          if (r < rows) {
            // a piece lies by four dims, so that 32 rows are neighbours
            const size_t row0 = (size_t)blockIdx.x * kSH_M + base;
            if (half == 0) a.ml[row0 + r] = make_float2(m_ref, l);
            ulonglong2* to = reinterpret_cast<ulonglong2*>(a.part + row0 * kPG_D + (size_t)half * 128 * rows) + r;
#pragma unroll
            for (int i = 0; i < 64; i += 2) {
              *to = make_ulonglong2(acc[i], acc[i + 1]);
              to += rows;
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0) report_abort(abort, a.err);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Output rows: a block has 32 neighbouring rows of one KV head, in the plan's order (they are neighbours in every piece too), and 16 dims for each of its
// 8 / Split groups of warps; a lane has a row, and the row's pieces (tail, then its runs, CTA by CTA) are dealt to a group's
// Split warps, whose sums are added in order.  The first warp finds where the rows' pieces lie.
constexpr int kSH_MergeDims = 16, kSH_MergeSmem = 23552;       // bytes of static shared memory, at least
template <typename T, int Split>
__global__ void __launch_bounds__(256) paged_merge_kernel(SharedArgs a) {
  constexpr int Groups = 8 / Split, Ways = kSH_Ways;
  __shared__ float s_acc[8][kSH_MergeDims][32];
  __shared__ float2 s_sum[8][32];
  __shared__ int4 s_way[Ways][32];       // first CTA, pieces, rows of a piece, row of it
  __shared__ int s_base[Ways][32], s_out[32];
  wait_for_stream();
  let_next_start();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = warp / Split, split = warp % Split;
  const int d0 = (blockIdx.y * Groups + group) * kSH_MergeDims, g = blockIdx.z;
  const int per_seq = a.t * a.R;
  const long long sr = (long long)blockIdx.x * 32 + lane;
  const bool on = sr < (long long)a.n * per_seq;
  if (warp == 0) {
    const Plan pl(a.plan, a.n, a.plan[0]);
    const int place = on ? (int)(sr / per_seq) : 0, rem = on ? (int)(sr - (long long)place * per_seq) : 0, i = rem / a.R;
    const int4 head = *a.head;
    const int each = head.x, more = head.y, longer = more * (each + 1);
    auto cta_of = [&](int u) { return u < longer ? u / (each + 1) : more + (u - longer) / each; };
#pragma unroll
    for (int k = 0; k < Ways; ++k) {
      const int4* p = reinterpret_cast<const int4*>(a.ways + (size_t)place * Ways + k);
      const int4 x = p[0], y = p[1];
      int4 way = make_int4(0, 0, 1, 0);
      int base = 0;
      if (on && x.w > 0) {
        const int blocks = (x.z + kSH_M - 1) / kSH_M, idx = (place - y.x) * per_seq + rem, rb = idx / kSH_M;
        const int u = x.x + (g * blocks + rb) * (x.w + kSH_Start) + kSH_Start, c0 = cta_of(u);
        way = make_int4(c0, cta_of(u + x.w - 1) - c0 + 1, min(kSH_M, x.z - rb * kSH_M), idx - rb * kSH_M);
        base = x.y + g * x.z + rb * kSH_M;
      }
      s_way[k][lane] = way;
      s_base[k][lane] = base;
    }
    s_out[lane] = (pl.order[place] * a.t + i) * a.H + g * a.R + rem - i * a.R;
  }
  __syncthreads();
  float m = -INFINITY, sum = 0.f, acc[kSH_MergeDims];
#pragma unroll
  for (int k = 0; k < kSH_MergeDims; ++k) acc[k] = 0.f;
  int seen = 0;                            // pieces of the ways before
  for (int k = 0; k < Ways; ++k) {
    const int4 way = s_way[k][lane];
    const int base = s_base[k][lane];
    // a few pieces at a time, the loads of all of them before the first sum
    constexpr int Batch = 3;
    for (int mine = (split - seen) & (Split - 1); mine < way.y; mine += Batch * Split) {
      float v[Batch][kSH_MergeDims];
      float2 ml[Batch];
#pragma unroll
      for (int x = 0; x < Batch; ++x) {
        const size_t row0 = (size_t)(way.x + min(mine + x * Split, way.y - 1)) * kSH_M + base;
        ml[x] = a.ml[row0 + way.w];
        const float4* p = reinterpret_cast<const float4*>(a.part + row0 * kPG_D + (size_t)d0 * way.z) + way.w;
#pragma unroll
        for (int q = 0; q < kSH_MergeDims; q += 4) {
          const float4 y = p[(size_t)(q / 4) * way.z];
          v[x][q] = y.x, v[x][q + 1] = y.y, v[x][q + 2] = y.z, v[x][q + 3] = y.w;
        }
      }
#pragma unroll
      for (int x = 0; x < Batch; ++x) {
        if (mine + x * Split >= way.y) break;
        // a partial without a maximum holds zeros, or NaN to be passed on
        const float mn = fmaxf(m, ml[x].x);
        const float al = m == -INFINITY ? 1.f : ex2_approx(m - mn), f = ml[x].x == -INFINITY ? 1.f : ex2_approx(ml[x].x - mn);
#pragma unroll
        for (int q = 0; q < kSH_MergeDims; ++q) acc[q] = acc[q] * al + v[x][q] * f;
        sum = sum * al + ml[x].y * f;
        m = mn;
      }
    }
    seen += way.y;
  }
#pragma unroll
  for (int k = 0; k < kSH_MergeDims; ++k) s_acc[warp][k][lane] = acc[k];
  s_sum[warp][lane] = make_float2(m, sum);
  __syncthreads();
  // each warp 16 / Split of its group's dims
  constexpr int Dims = kSH_MergeDims / Split;
  const int w0 = group * Split;
  float f[Split], l = 0.f;
  m = -INFINITY;
#pragma unroll
  for (int k = 0; k < Split; ++k) m = fmaxf(m, s_sum[w0 + k][lane].x);
#pragma unroll
  for (int k = 0; k < Split; ++k) {
    const float2 x = s_sum[w0 + k][lane];
    f[k] = x.x == -INFINITY ? 1.f : ex2_approx(x.x - m);
    l = fmaf(x.y, f[k], l);
  }
  if (!on) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;       // nothing seen: zeros
  __align__(16) T out[Dims];
#pragma unroll
  for (int d = 0; d < Dims; ++d) {
    float x = 0.f;
#pragma unroll
    for (int k = 0; k < Split; ++k) x = fmaf(s_acc[w0 + k][split * Dims + d][lane], f[k], x);
    out[d] = (T)(x * inv);
  }
  const int row = s_out[lane];
  T* to = static_cast<T*>(a.o) + (size_t)row * kPG_D + d0 + split * Dims;
#pragma unroll
  for (int d = 0; d < Dims; d += 2) *reinterpret_cast<uint32_t*>(to + d) = *reinterpret_cast<const uint32_t*>(out + d);
  if (a.lse && d0 == 0 && split == 0) {
    const int h = row % a.H, bt = row / a.H, b = bt / a.t;
    a.lse[((size_t)b * a.H + h) * a.t + bt - b * a.t] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
  }
}

template <typename T>
static int launch_shared(const SharedArgs& a, int ctas, cudaStream_t stream) {
  constexpr int Parts = SharedCfg<T>::Parts;
  int rc = ensure_smem_attr((const void*)paged_shared_kernel<T>, SharedSmem<T>::Bytes);
  if (rc) return rc;
  CUtensorMap kmap, vmap, qmap;
  const uint64_t dims[2] = {(uint64_t)kPG_D, (uint64_t)a.p.pages * a.p.heads * a.p.page}, strides[1] = {(uint64_t)kPG_D};
  const uint32_t box[2] = {128, (uint32_t)a.p.page};
  if ((rc = make_tmap(&kmap, a.p.k, kTmapU8, 2, dims, strides, box, true))) return rc;
  if ((rc = make_tmap(&vmap, a.p.v, kTmapU8, 2, dims, strides, box, true))) return rc;
  const uint64_t rows = (uint64_t)a.n * a.t * a.H, qdims[2] = {(uint64_t)Parts * kPG_D, rows}, qstrides[1] = {(uint64_t)Parts * kPG_D};
  const uint32_t qbox[2] = {128, kSH_M};
  if ((rc = make_tmap(&qmap, a.qp, kTmapU8, 2, qdims, qstrides, qbox, true))) return rc;
  const unsigned per_head = (unsigned)(rows / a.p.heads);
  if ((rc = launch_early(paged_queries_kernel<T>, dim3((per_head + 7) / 8, a.p.heads), 256, 0, stream, a))) return rc;
  if ((rc = launch_early(paged_shared_kernel<T>, dim3(ctas), kSH_Threads, SharedSmem<T>::Bytes, stream, kmap, vmap, qmap, a))) return rc;
  // a row's pieces are dealt to so many warps that there are 600 to 1200 of them: with few rows the pieces' way is what takes time (whole call, in bursts at 1965 MHz, 16 x 24 rows of
  // 37 pieces each: 100, 90, 85 and 86 us over 1, 2, 4 and 8), with many the blocks (64 x 24 rows of 13: 48, 52, 53 and 62)
  const unsigned blocks = (per_head + 31) / 32, warps = blocks * a.p.heads * (kPG_D / kSH_MergeDims);
  // Its CTAs come as those of the kernel before them leave their SMs: each takes so much shared memory that no SM has more than its share of them, or the
  // first SMs that are free would take them all (16 x 131072, in bursts: 84 us against 93).
  auto merge = [&](auto kernel, int split) {
    const unsigned ctas_y = kPG_D / kSH_MergeDims * split / 8, each = (blocks * ctas_y * a.p.heads + ctas - 1) / ctas;
    const int idle = each < 8 ? (232448 / (int)each - 1024) / 1024 * 1024 - kSH_MergeSmem : 0;
    const int e = ensure_smem_attr((const void*)kernel, 232448 - 1024 - kSH_MergeSmem);
    return e ? e : launch_early(kernel, dim3(blocks, ctas_y, a.p.heads), 256, idle, stream, a);
  };
  if (warps >= 576) return merge(paged_merge_kernel<T, 1>, 1);
  if (warps >= 288) return merge(paged_merge_kernel<T, 2>, 2);
  if (warps >= 144) return merge(paged_merge_kernel<T, 4>, 4);
  return merge(paged_merge_kernel<T, 8>, 8);
}

// the workspace: its bytes, and the arrays in it
static size_t shared_layout(SharedArgs& a, int n, int t, int H, int parts, uint8_t* ws) {
  size_t at = 0;
  auto take = [&](size_t bytes) {
    uint8_t* p = ws ? ws + at : nullptr;
    at += (bytes + 15) / 16 * 16;
    return p;
  };
  const size_t heads_rows = (size_t)n * t * H, rows = (size_t)kSH_MaxCtas * kSH_M + (kPS_Depth + 1) * heads_rows;
  a.head = reinterpret_cast<int4*>(take(sizeof(int4)));
  a.ways = reinterpret_cast<SharedWay*>(take((size_t)n * kSH_Ways * sizeof(SharedWay)));
  a.qs = reinterpret_cast<float*>(take(heads_rows * 4));
  a.qp = take(heads_rows * parts * kPG_D);
  a.ml = reinterpret_cast<float2*>(take(rows * sizeof(float2)));
  a.part = reinterpret_cast<float*>(take(rows * kPG_D * 4));
  return at;
}

}  // namespace bfb

using namespace bfb;

extern "C" {

size_t bf_paged_attend_shared_workspace(int n, int t, int H, int G, int D) {
  if (n <= 0 || t <= 0 || H <= 0 || G <= 0 || H % G || H / G > kSH_MaxGroup || D != kPG_D) return 0;
  SharedArgs a{};
  return shared_layout(a, n, t, H, 3, nullptr);
}

int bf_paged_attend_shared(const bf_page_pool* pool, int layer, const void* q, long long q_sb, long long q_st, long long q_sh, const int32_t* plan,
                           int n, int t, int H, int dtype, float scale, void* o, float* lse, void* ws, size_t ws_bytes, bf_stream_t stream) {
  SharedArgs a{};
  int rc = page_pool(pool, layer, &a.p);
  if (rc) return rc;
  if (n < 0 || t < 0 || H <= 0 || H % a.p.heads || !(scale > 0.f) || scale > 3e38f) return BF_ERR_INVALID_ARGUMENT;
  if ((dtype != BF_BF16 && dtype != BF_F16) || H / a.p.heads > kSH_MaxGroup) return BF_ERR_UNSUPPORTED;
  if (n == 0 || t == 0) return BF_OK;
  if (!q || !o || !plan) return BF_ERR_INVALID_ARGUMENT;
  if (!aligned16(q) || !aligned16(o) || !aligned16(plan) || ((q_sb | q_st | q_sh) & 7)) return BF_ERR_ALIGNMENT;
  // units and rows are counted in 32 bits: a sequence's stretches cover its table's pages once
  const long long rows = (long long)n * t * H, tiles = (long long)a.p.width * a.p.page / kSH_N + (kPS_Depth + 1) * (kSH_Start + 1);
  if ((kPS_Depth + 1) * rows + (long long)kSH_MaxCtas * kSH_M > 0x7fffffffLL || (rows / kSH_M + 2ll * n * a.p.heads) * tiles > 0x7fffffffLL)
    return BF_ERR_UNSUPPORTED;
  if (!ws || ws_bytes < shared_layout(a, n, t, H, 3, nullptr)) return BF_ERR_WORKSPACE;
  if (!aligned16(ws)) return BF_ERR_ALIGNMENT;
  DeviceState st;
  if ((rc = device_state(&st))) return rc;
  shared_layout(a, n, t, H, 3, static_cast<uint8_t*>(ws));
  a.q = q;
  a.q_sb = q_sb; a.q_st = q_st; a.q_sh = q_sh;
  a.plan = plan;
  a.n = n; a.t = t; a.H = H; a.R = H / a.p.heads;
  a.page_log = a.p.page == 16 ? 4 : a.p.page == 32 ? 5 : a.p.page == 64 ? 6 : 7;
  a.cap = (int)((long long)a.p.width * a.p.page < 0x7fffff00LL ? (long long)a.p.width * a.p.page : 0x7fffff00LL);
  a.c2 = scale * kLog2e;
  a.o = o;
  a.lse = lse;
  a.err = st.err;
  const int ctas = st.sm_count < kSH_MaxCtas ? st.sm_count : kSH_MaxCtas;
  return dtype == BF_BF16 ? launch_shared<__nv_bfloat16>(a, ctas, stream) : launch_shared<__half>(a, ctas, stream);
}

}  // extern "C"
