// Causal attention of packed prompts (sequences of different lengths in one call) with grouped query heads.
//
//   o_i = sum_j p_ij v_j,  p_i = softmax_j(scale q_i . k_j),  keys j <= i + nk - nq of the query's own sequence.
//
// Bound by the tensor core: 4 D flops per visible (query, key, head) against 2 D bytes per key.  With D = 256 an output tile of
// 128 rows takes half of TMEM, so an SM works on one tile of 128 queries; fed by one CTA alone, a 128-key tile is 128 KB
// from L2 per 1.5 us and SM, as much as L2 delivers.  So two CTAs form a pair (cta_group::2, M = 256): each holds its own 128
// query rows and half of the keys' rows and of the values' columns, 64 KB per key tile and SM, which leaves room for two stages
// of each.  The pair's two row tiles are two query heads of one KV head on the same 128 tokens (the same keys, the same causal
// edge), or, with an odd number of heads per KV head, two neighbouring tiles of 128 tokens of one head.
//   S_j = Q K_j^T    M256 N128 K256 (A and B in shared memory)                        -> TMEM S buffer (tile parity)
//   O  += P_j V_j    M256 N256 K128 (A = P_j in TMEM over S_j, B = V_j as it lies: N-major)
//   TMEM of each CTA: S/P buffers at columns 0 and 128, O at 256..511.
// P is rounded to the inputs' type, which moves a weight by half a step of the type at most: as much as the output's own rounding,
// and it averages over the keys.  Its sum is taken before.  Scores are in the log2 domain; O is rescaled only when a row's
// maximum grows by more than 2^8.  In fp16 that leaves 2^7 of the type's range above the weights, so they enter 2^7 times as large:
// fp16 is exact to half a step of the weight only down to 2^-14, thus down to 2^-21 of the row's reference, and below that to 2^-32
// of it (without the factor 2^-25: a key of weight 2^-20 beside one of nearly 1 was off by 2^-6 of itself).
//
// Work items are (token block, KV head, head pair or head), one cluster of the grid each, those with the most key tiles first.
// A cluster that has done its own item asks the hardware for one that has not started (cluster launch control) and goes on with
// that: the start of a CTA pair (barriers, TMEM, the first loads) costs about 9 us, and the next item's loads and first products
// run under the end of the last one.
// Warps (512 threads): 0 Q and K loads; 1 MMA (in the first CTA of the pair); 2 V loads; 3 the next items (the first CTA asks and
// passes the answer on); 4-11 softmax, two warpgroups, every other tile each; 12-15 the outputs, while the next item's products run.
//
// Measured (24 query heads, 4 KV heads, bf16), repeated on one input: 32768 tokens 9.13 ms = 1446 TFLOP/s on one GPU, 9.3 to 9.6 ms on
// others and with other inputs in every pass (1375 to 1420; the library product's rate under the power limit is 1406, its burst
// 1666); 8192 tokens 538 us = 1534 before the power limit sets in, 600 in a longer loop; 2300 cycles per key tile against the tensor core's
// 2048.  Between items 3700 cycles are lost, most of them for the next item's queries, 64 KB that only fit once the last product has
// read the ones before: eight prompts of 1 to 4095 tokens run at 1274.
#include "bifrost_b200.h"
#include "capi_internal.h"
#include "common.cuh"
#include "launch_early.h"
#include "tmap.h"

namespace bfb {

constexpr int kPR_D = 256;
constexpr int kPR_M = 128;        // query rows per CTA
constexpr int kPR_N = 128;        // keys per tile
constexpr int kPR_Threads = 512;
// register split (setmaxnreg) of the 128 per thread at launch
constexpr uint32_t kPR_RegsCtl = 96, kPR_RegsSoftmax = 168, kPR_RegsEpi = 80;
static_assert(128 * kPR_RegsCtl + 256 * kPR_RegsSoftmax + 128 * kPR_RegsEpi == kPR_Threads * 128, "register split");
constexpr int kPR_SmemQ = kPR_M * kPR_D * 2;          // 64 KB
constexpr int kPR_SmemK = kPR_N / 2 * kPR_D * 2;      // 32 KB: this CTA's half of the keys
constexpr int kPR_SmemV = kPR_N * kPR_D / 2 * 2;      // 32 KB: this CTA's half of the columns
constexpr int kPR_Tiles = kPR_SmemQ + 2 * kPR_SmemK + 2 * kPR_SmemV;
constexpr int kPR_Items = 3;      // items known ahead
constexpr int kPR_Ask = 4;        // the next item is asked for this many key tiles before the loads of the last one end
constexpr int kPR_Parts = 1024;   // parts whose first rows and keys fit into shared memory
// Limits: the waits give up after about a second, an item of 2^25 keys takes a third of that, and the first look through 2^20 sequences
// a few hundredths
constexpr int kPR_MaxKeys = 1 << 25, kPR_MaxSeqs = 1 << 20;
constexpr int kPR_Smem = kPR_Tiles + 640 + 5120 + 8192 + 4 * 2048 + 1024;
constexpr uint32_t kPR_TmO = 256;
constexpr float kPR_Rescale = 8.0f;
// log2 of what P is multiplied by: the largest weight, 2^kPR_Rescale times that, has to stay below fp16's 65504
template <typename T>
__device__ __forceinline__ constexpr float prompt_up() { return __is_same(T, __half) ? 7.f : 0.f; }

struct PromptArgs {
  const int32_t *cu_q, *cu_k;
  int n_seq, T, Tk, H, G;
  int qb, qlog;           // tokens per block: 128 (two heads) or 256 (two tiles of one head), and its log2
  int nblk, hsplit;       // blocks, items per (block, KV head)
  int step_log;
  float c2;               // scale * log2(e)
  void* o;
  float* lse;
  unsigned int* err;
};

// the block's sequence: tokens q0 .. q0 + nq - 1, keys k0 .. k0 + nk - 1, the block's first token i0 in it
struct PromptBlock {
  int q0, nq, k0, nk, i0;
};

// What a CTA has to do for an item: its rows of q and o (row0 and up, `rows` of them stored), keys k0 and up of which nk are the
// sequence's, n key tiles (-1: no more items), row r of the tile sees keys up to lim + r
struct __align__(16) PromptItem {
  int row0, rows, k0, nk, n, lim, h, g;
};

// The rows are cut into n_seq + 2 parts: those before the first sequence, the sequences, those behind the last; the first and the
// last part have no keys.  Cumulative lengths are clamped into [previous, T] and [previous, Tk].  Lane's part c + lane, given the
// greatest entries before part c:
struct PromptPart {
  int q0, nq, k0, nk;
};
__device__ __forceinline__ PromptPart prompt_part(const PromptArgs& a, int c, int lane, int& carry_q, int& carry_k) {
  const int p = c + lane;
  const bool from = p >= 1 && p <= a.n_seq + 1 && a.cu_q, to = p <= a.n_seq && a.cu_q;
  int q = from ? min(max(a.cu_q[p - 1], 0), a.T) : 0, k = from ? min(max(a.cu_k[p - 1], 0), a.Tk) : 0;
  int qn = to ? min(max(a.cu_q[p], 0), a.T) : a.T, kn = to ? min(max(a.cu_k[p], 0), a.Tk) : 0;
  q = max(q, carry_q);
  k = max(k, carry_k);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, q, o), y = __shfl_up_sync(0xffffffffu, k, o);
    if (lane >= o) {
      q = max(q, x);
      k = max(k, y);
    }
  }
  qn = max(q, qn);
  kn = p >= 1 && to ? max(k, kn) : k;
  carry_q = __shfl_sync(0xffffffffu, q, 31);
  carry_k = __shfl_sync(0xffffffffu, k, 31);
  return PromptPart{q, qn - q, k, kn - k};
}
__device__ __forceinline__ PromptBlock prompt_of_lane(const PromptPart& p, int i0, int at) {
  return PromptBlock{__shfl_sync(0xffffffffu, p.q0, at), __shfl_sync(0xffffffffu, p.nq, at), __shfl_sync(0xffffffffu, p.k0, at),
                     __shfl_sync(0xffffffffu, p.nk, at), __shfl_sync(0xffffffffu, i0, at)};
}

// The block of rank `rank` by key tiles, the most first.  With a part per lane (up to 30 sequences): the largest number of tiles t
// that more than `rank` blocks have at least, by bisection; of a part with nb blocks those with t tiles or more are its last ones.
// The last blocks to start decide how long the call takes: chunks of 512 tokens after 8192, 1000, 2048 and 4096 earlier ones
// took 164 us in the order of the sequences.
// With more parts than lanes: in the reverse order of the rows; part p owns the block numbers q0 / qb + p and up, at least as many as
// it has blocks, and is found by bisection in shared memory, where starts holds the first row and key of every 2^step_log-th part (of
// each one, if they fit), and by going through the parts from that one on.
__device__ __forceinline__ bool prompt_few(const PromptArgs& a) { return a.n_seq + 2 <= 32; }
__device__ __forceinline__ PromptBlock prompt_block(const PromptArgs& a, const PromptPart& first, const int2* starts, int rank, int lane) {
  if (prompt_few(a)) {
    const PromptPart p = first;
    const int qlog = a.qlog, nb = lane < a.n_seq + 2 ? (p.nq + a.qb - 1) >> qlog : 0, off = p.nk - p.nq;
    auto at_least = [&](int t) {      // blocks of this part with t tiles or more
      const int key = (t - 1) * kPR_N;                       // the first key of the last tile
      if (t <= 0 || nb == 0) return nb;
      if (p.nk <= key) return 0;
      return nb - min(max(((key + 1 - off + a.qb - 1) >> qlog) - 1, 0), nb - 1);
    };
    auto sum = [](int x) { return (int)__reduce_add_sync(0xffffffffu, (unsigned)x); };
    int lo = 0, hi = (int)__reduce_max_sync(0xffffffffu, nb ? (unsigned)((p.nk + kPR_N - 1) / kPR_N) : 0u);
    if (sum(nb) <= rank) return PromptBlock{0, 0, 0, 0, 0};
    while (lo < hi) {                  // the answer is in [lo, hi]
      const int mid = (lo + hi + 1) >> 1;
      if (sum(at_least(mid)) > rank) lo = mid; else hi = mid - 1;
    }
    const int more = at_least(lo + 1), here = at_least(lo) - more;
    int incl = here;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    const int idx = rank - sum(more);
    const int at = __ffs(__ballot_sync(0xffffffffu, incl > idx)) - 1;
    return prompt_of_lane(p, (nb - more - here + idx - (incl - here)) * a.qb, at);
  }
  PromptBlock r{0, 0, 0, 0, 0};
  const int blk = a.nblk - 1 - rank;
  int lo = 0, hi = (a.n_seq + 1) >> a.step_log;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((starts[mid].x >> a.qlog) + (mid << a.step_log) <= blk) lo = mid; else hi = mid - 1;
  }
  int carry_q = starts[lo].x, carry_k = starts[lo].y;
  for (int c = lo << a.step_log; c < a.n_seq + 2; c += 32) {
    const PromptPart p = prompt_part(a, c, lane, carry_q, carry_k);
    const int base = (p.q0 >> a.qlog) + c + lane;
    const unsigned ok = __ballot_sync(0xffffffffu, c + lane < a.n_seq + 2 && base <= blk);
    if (ok == 0u) break;
    const int at = 31 - __clz(ok);
    r = prompt_of_lane(p, (blk - base) * a.qb, at);
    if (at < 31) break;
  }
  return r;
}

template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPR_Threads, 1)
    prompt_attn_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap, PromptArgs a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                        // [4 atoms][128 rows][128 B]
  uint8_t* sK = sQ + kPR_SmemQ;              // [2][4 atoms][64 keys][128 B]
  uint8_t* sV = sK + 2 * kPR_SmemK;          // [2][2 atoms][128 keys][128 B]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kPR_Tiles);
  // in the first CTA, for both: one arrival and the bytes of each CTA, or one arrival per warp of both
  uint64_t *q_full = bars, *k_full = bars + 1 /*[2]*/, *v_full = bars + 3 /*[2]*/, *p_full = bars + 5 /*[2]*/, *o_free = bars + 7;
  // in each CTA, by commits of the first
  uint64_t *q_free = bars + 8, *k_empty = bars + 9 /*[2]*/, *v_empty = bars + 11 /*[2]*/, *s_full = bars + 13 /*[2]*/, *o_fin = bars + 15;
  // within a CTA
  uint64_t *mref = bars + 46 /*[2][4]*/, *stats = bars + 20 /*[2]*/, *sfree = bars + 22 /*[2]*/, *v_own = bars + 24;
  uint64_t *item_full = bars + 25 /*[3]*/, *item_free = bars + 28 /*[3]*/, *clc = bars + 31, *msg_full = bars + 32, *msg_free = bars + 33,
           *ask = bars + 39;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 34);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 35);
  uint8_t* answer = reinterpret_cast<uint8_t*>(bars + 36);                         // 16 bytes
  volatile int* msg = reinterpret_cast<volatile int*>(bars + 38);
  PromptItem* s_items = reinterpret_cast<PromptItem*>(bars + 54);                  // [kPR_Items]
  static_assert(54 * 8 + kPR_Items * sizeof(PromptItem) <= 640, "barriers and items");
  float* xch = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + 640);   // [2 tile parities][128] references
  float* xl = xch + 256;                                                           // [2 slots][2 warpgroups][128] row sums
  float* xmx = xl + 512;                                                           // [2 slots][2 warpgroups][128] their references
  int2* s_starts = reinterpret_cast<int2*>(reinterpret_cast<uint8_t*>(bars) + 640 + 5120);   // [kPR_Parts], one warp's
  uint8_t* s_out = reinterpret_cast<uint8_t*>(bars) + 640 + 5120 + 8192;          // [4 output warps][32 rows][128 B]

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const uint32_t rank = cluster_rank();
  const int R = a.H / a.G, two = a.qb == kPR_M;            // two: the pair's tiles are two heads
  // item `it`, by one lane (lanes = 1) or a whole warp; false when there are no more, or a wait gave up
  auto item = [&](int it, bool whole_warp, PromptItem& x) -> bool {
    const int s = it % kPR_Items;
    const bool ok = whole_warp ? mbar_wait_warp_small(item_full + s, (it / kPR_Items) & 1, abort_flag, 0x90)
                               : mbar_wait_small(item_full + s, (it / kPR_Items) & 1, abort_flag, 0x90);
    if (!ok) return false;
    x = s_items[s];
    if (whole_warp) __syncwarp();
    if (!whole_warp || lane == 0) mbar_arrive(item_free + s);
    return x.n >= 0;
  };

  if (tid == 0) {
    mbar_init(q_full, 2);
    mbar_init(o_free, 8);
    mbar_init(q_free, 1);
    mbar_init(o_fin, 1);
    mbar_init(v_own, 1);
    mbar_init(clc, 1);
    mbar_init(ask, 1);
    mbar_init(msg_full, 1);
    mbar_init(msg_free, 1);
    for (int i = 0; i < kPR_Items; ++i) {
      mbar_init(item_full + i, 1);
      mbar_init(item_free + i, rank == 0 ? 15 : 14);       // Q and K, V, softmax 8, outputs 4, and the products
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(k_full + i, 2);
      mbar_init(v_full + i, 2);
      mbar_init(p_full + i, 8);
      mbar_init(k_empty + i, 1);
      mbar_init(v_empty + i, 1);
      mbar_init(s_full + i, 1);
      mbar_init(stats + i, 8);
      mbar_init(sfree + i, 4);
    }
    for (int i = 0; i < 8; ++i) mbar_init(mref + i, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  wait_for_stream();

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPR_RegsCtl));
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------------- Q and K
      tma_prefetch(&qmap);
      tma_prefetch(&kmap);
      const uint32_t qf = cluster_addr(q_full, 0), kf[2] = {cluster_addr(k_full, 0), cluster_addr(k_full + 1, 0)};
      int t = 0;
      bool ok = true;
      PromptItem x;
      for (int it = 0; ok && item(it, false, x); ++it) {
        if (it >= 1 && !(ok = mbar_wait_small(q_free, (it - 1) & 1, abort_flag, 0x80))) break;
        mbar_expect_tx_cluster(qf, kPR_SmemQ);
        tma_load_4d_pair(sQ, &qmap, qf, 0, x.row0, 0, x.h);
        if (x.n == 0 && rank == 0) mbar_arrive(ask);
        for (int j = 0; j < x.n; ++j, ++t) {
          const int s = t & 1;
          if (j == max(x.n - kPR_Ask, 0) && rank == 0) mbar_arrive(ask);
          if (t >= 2 && !(ok = mbar_wait_small(k_empty + s, ((t >> 1) - 1) & 1, abort_flag, 0x81))) break;
          mbar_expect_tx_cluster(kf[s], kPR_SmemK);
          tma_load_4d_pair(sK + s * kPR_SmemK, &kmap, kf[s], 0, x.k0 + j * kPR_N + (int)rank * (kPR_N / 2), 0, x.g);
        }
      }
    } else if (warp == 2) {
      // ---------------------------------------------------------------- V
      if (lane == 0) tma_prefetch(&vmap);
      const uint32_t vf[2] = {cluster_addr(v_full, 0), cluster_addr(v_full + 1, 0)};
      int t = 0, own = 0;
      bool ok = true;
      PromptItem x;
      for (int it = 0; ok && item(it, true, x); ++it) {
        for (int j = 0; j < x.n; ++j, ++t) {
          const int s = t & 1, rows = x.nk - j * kPR_N;   // rows of the tile that are this sequence's
          if (t >= 2 && !(ok = mbar_wait_warp_small(v_empty + s, ((t >> 1) - 1) & 1, abort_flag, 0x82))) break;
          uint8_t* dst = sV + s * kPR_SmemV;
          const bool whole = rows >= kPR_N;
          if (lane == 0) {
            if (whole) mbar_expect_tx_cluster(vf[s], kPR_SmemV); else mbar_expect_tx(v_own, kPR_SmemV);
            tma_load_4d_pair(dst, &vmap, whole ? vf[s] : smem_u32(v_own), 0, x.k0 + j * kPR_N, 2 * (int)rank, x.g);
          }
          __syncwarp();
          if (!whole) {
            // the rows behind the sequence belong to others: their weights are 0, but 0 times NaN would not be
            if (!(ok = mbar_wait_warp_small(v_own, own & 1, abort_flag, 0x83))) break;
            ++own;
            for (int i = lane; i < (kPR_N - rows) * 8; i += 32) {
              uint4* p = reinterpret_cast<uint4*>(dst + rows * 128) + i;
              p[0] = p[kPR_N * 8] = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(vf[s]);
          }
        }
      }
    } else if (warp == 3) {
      // ---------------------------------------------------------------- items
      const uint32_t peer_msg = cluster_addr((const void*)msg, 1), peer_full = cluster_addr(msg_full, 1), lead_free = cluster_addr(msg_free, 0);
      int it = 0, asked = 0, carry_q = 0, carry_k = 0;
      PromptPart first{0, 0, 0, 0};
      if (prompt_few(a)) {
        first = prompt_part(a, 0, lane, carry_q, carry_k);
      } else {
        for (int c = 0; c < a.n_seq + 2; c += 32) {
          const PromptPart p = prompt_part(a, c, lane, carry_q, carry_k);
          const int at = (c + lane) >> a.step_log;
          if (c + lane < a.n_seq + 2 && at << a.step_log == c + lane) s_starts[at] = make_int2(p.q0, p.k0);
        }
        __syncwarp();
      }
      int cta = (int)(blockIdx.x & ~1u);
      for (bool ok = true; ok;) {
        PromptItem x{0, 0, 0, 0, -1, 0, 0, 0};
        if (cta >= 0) {
          int cl = cta >> 1;
          const int hs = cl % a.hsplit;
          cl /= a.hsplit;
          const PromptBlock b = prompt_block(a, first, s_starts, cl / a.G, lane);
          const int off = b.nk - b.nq;                                // query i sees keys j <= i + off
          const int i0 = b.i0 + (two ? 0 : (int)rank * kPR_M);        // this CTA's first token
          const int last = min(b.i0 + a.qb, b.nq) - 1 + off;          // last key that the pair sees
          x.g = cl % a.G;
          x.h = x.g * R + (two ? 2 * hs + (int)rank : hs);
          x.row0 = b.q0 + i0;
          x.rows = b.nq - i0;
          x.k0 = b.k0;
          x.nk = b.nk;
          x.n = last >= 0 ? last / kPR_N + 1 : 0;
          x.lim = i0 + off;
          if (b.i0 >= b.nq) x.n = -2;                                 // a block number that no sequence uses
        }
        if (x.n != -2) {
          const int s = it % kPR_Items;
          if (it >= kPR_Items && !mbar_wait_warp_small(item_free + s, (it / kPR_Items - 1) & 1, abort_flag, 0x91)) break;
          if (lane == 0) {
            s_items[s] = x;
            mbar_arrive(item_full + s);
            if (it > 0 && x.n > 0) tma_prefetch_tile_4d(&qmap, 0, x.row0, 0, x.h);     // its queries into L2 meanwhile
          }
          __syncwarp();
          ++it;
        }
        if (cta < 0) break;
        // the next one: the first CTA of the pair asks, when the loads of the item before it near their end (a cluster that
        // asked earlier would keep an item waiting that another could start), and tells the other
        if (rank == 0) {
          if (it > 0 && x.n != -2 && !(ok = mbar_wait_warp_small(ask, (it - 1) & 1, abort_flag, 0x95))) break;
          if (lane == 0) {
            mbar_expect_tx(clc, 16);
            clc_try_cancel(answer, clc);
          }
          __syncwarp();
          ok = mbar_wait_warp_small(clc, asked & 1, abort_flag, 0x92);
          if (ok && asked >= 1) ok = mbar_wait_warp_small(msg_free, (asked - 1) & 1, abort_flag, 0x93);
          if (!ok) break;
          cta = clc_answer(answer);
          fence_async_smem();          // the answer has been read before the next one is written over it
          if (lane == 0) st_async_u32(peer_msg, (uint32_t)cta, peer_full);
          __syncwarp();
        } else {
          if (lane == 0) mbar_expect_tx(msg_full, 4);
          __syncwarp();
          if (!(ok = mbar_wait_warp_small(msg_full, asked & 1, abort_flag, 0x94))) break;
          cta = __shfl_sync(0xffffffffu, *msg, 0);
          if (lane == 0) mbar_arrive_cluster(lead_free);       // the word has been read
        }
        ++asked;
      }
    } else if (warp == 1 && rank == 0) {
      // ---------------------------------------------------------------- MMA
      // The warp stays converged and elects the issuing lane, so that descriptors stay in uniform registers: one lane of a diverged
      // warp took 1300 cycles to issue the 16 steps of S and 700 for the 8 of O, longer than the tensor core for them.
      constexpr int is_bf16 = !__is_same(T, __half);
      constexpr uint32_t id_s = idesc_f16(2 * kPR_M, kPR_N, is_bf16), id_o = idesc_f16(2 * kPR_M, kPR_D, is_bf16) | kIdescBMn;
      const uint64_t dq = sdesc_sw128(smem_u32(sQ)), dk0 = sdesc_sw128(smem_u32(sK)), dv0 = sdesc_sw128_mn(smem_u32(sV), kPR_N * 128);
      int t = 0;
      bool ok = true;
      PromptItem x;
#pragma unroll 1
      for (int it = 0; ok && item(it, true, x); ++it) {
        const int n = x.n;
        if (!(ok = mbar_wait_warp_small(q_full, it & 1, abort_flag, 0x84))) break;
        // O += P_j V_j of tile j = jj - 1 follows the issue of S_jj; jj = n closes the item
#pragma unroll 1
        for (int jj = 0; jj <= n; ++jj) {
          if (jj < n) {
            const int tt = t + jj, s = tt & 1;
            if (!(ok = mbar_wait_warp_small(k_full + s, (tt >> 1) & 1, abort_flag, 0x88))) break;
            tc_fence_after();
            if (elect_one()) {
              const uint64_t dk = dk0 + (uint32_t)(s * (kPR_SmemK >> 4));
#pragma unroll
              for (int ks = 0; ks < kPR_D / 16; ++ks)
                umma_f16_ss_pair(tmem + s * kPR_N, dq + ((ks >> 2) * (kPR_M * 128) + (ks & 3) * 32) / 16,
                                 dk + ((ks >> 2) * (kPR_N / 2 * 128) + (ks & 3) * 32) / 16, id_s, ks > 0);
              umma_commit_pair(s_full + s);
              umma_commit_pair(k_empty + s);
              if (jj == n - 1) umma_commit_pair(q_free);
            }
            __syncwarp();
          }
          if (jj >= 1) {
            const int tt = t + jj - 1, s = tt & 1;
            if (!(ok = mbar_wait_warp_small(v_full + s, (tt >> 1) & 1, abort_flag, 0x86))) break;
            if (jj == 1 && it >= 1 && !(ok = mbar_wait_warp_small(o_free, (it - 1) & 1, abort_flag, 0x87))) break;
            if (!(ok = mbar_wait_warp_small(p_full + s, (tt >> 1) & 1, abort_flag, 0x85))) break;
            tc_fence_after();
            if (elect_one()) {
              const uint64_t dv = dv0 + (uint32_t)(s * (kPR_SmemV >> 4));
#pragma unroll
              for (int ks = 0; ks < kPR_N / 16; ++ks)
                umma_f16_ts_pair(tmem + kPR_TmO, tmem + s * kPR_N + ks * 8, dv + ks * (2048 / 16), id_o, (jj > 1 || ks > 0) ? 1u : 0u);
              umma_commit_pair(v_empty + s);
            }
            __syncwarp();
          }
        }
        if (!ok) break;
        // O counts as complete only once the item before has been drained, products or not
        if (n == 0 && it >= 1 && !(ok = mbar_wait_warp_small(o_free, (it - 1) & 1, abort_flag, 0x87))) break;
        if (elect_one()) {
          if (n == 0) umma_commit_pair(q_free);
          umma_commit_pair(o_fin);
        }
        __syncwarp();
        t += n;
      }
    }
  } else if (warp < 12) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPR_RegsSoftmax));
    // ------------------------------------------------------------------ softmax (warps 4..11)
    // Warpgroup w takes the tiles of parity w, thread = row, all 128 keys of it, in 2200 cycles (1400 for the exponentials), so one's
    // exponentials run beside the other's loads and comparisons.  (On the halves of each tile's keys the two would run in step, with
    // an exchange of maxima in between.)  A tile's reference, what O and P are relative to, is the tile before's, unless the tile's
    // maximum exceeds it by more than 2^kPR_Rescale; it is passed on as soon as the maximum is known.
    const int q4 = warp & 3, w = (warp - 4) >> 2;
    const int r = q4 * 32 + lane;                 // row of the tile == TMEM lane
    const uint32_t trow = tmem + ((uint32_t)(q4 * 32) << 16), srow = trow + w * kPR_N;
    const uint32_t pf = cluster_addr(p_full + w, 0);
    bool alive = true;
    int t = 0;
    PromptItem x;
    for (int it = 0; alive && item(it, true, x); ++it) {
      const int n = x.n, lim_all = x.lim, lim = x.lim + r;   // last key that every row of this CTA sees, and this row
      float m_own = -INFINITY, l = 0.f;           // this warpgroup's last reference (log2 domain), its sum relative to that
      for (int j = (t & 1) ^ w; j < n; j += 2) {
        const int tt = t + j, ph = (tt >> 1) & 1;
        if (!mbar_wait_warp_small(s_full + w, ph, abort_flag, 0x89)) { alive = false; break; }
        tc_fence_after();
        float uu[kPR_N];
        {
          uint32_t(&raw)[4][32] = reinterpret_cast<uint32_t(&)[4][32]>(uu);
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32(srow + c * 32, raw[c]);
          tmem_wait_ld();
        }
        if (j * kPR_N + kPR_N - 1 > lim_all) {
          const int hi = lim - j * kPR_N;
#pragma unroll
          for (int e = 0; e < kPR_N; ++e) uu[e] = e <= hi ? uu[e] : -INFINITY;
        }
        float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
        for (int e = 0; e < kPR_N; e += 8) {
          mx0 = max3(mx0, uu[e], uu[e + 1]);
          mx1 = max3(mx1, uu[e + 2], uu[e + 3]);
          mx2 = max3(mx2, uu[e + 4], uu[e + 5]);
          mx3 = max3(mx3, uu[e + 6], uu[e + 7]);
        }
        const float mt = max3(mx0, mx1, fmaxf(mx2, mx3)) * a.c2;
        // the reference of the tile before (which also says that it has been taken over from there)
        if (tt >= 1 && !mbar_wait_warp_small(mref + (1 - w) * 4 + q4, ((tt - 1) >> 1) & 1, abort_flag, 0x8a)) { alive = false; break; }
        const float prev = j >= 1 ? xch[(1 - w) * 128 + r] : -INFINITY;
        // (in fp16 less may be left standing where the scores are so large that their own last bit is a power of two or more)
        const float leave = prompt_up<T>() > 0.f ? fmaxf(fmaf(fabsf(mt), -0x1p-20f, kPR_Rescale), 0.f) : kPR_Rescale;
        const bool grown = prev != -INFINITY && mt > prev + leave;
        const float m = prev == -INFINITY || grown ? mt : prev;
        xch[w * 128 + r] = m;
        __syncwarp();
        if (lane == 0) mbar_arrive(mref + w * 4 + q4);
        l *= m_own == -INFINITY ? 1.f : ex2_approx(m_own - m);
        m_own = m;
        // O rescale (warp-collective), from the item's second tile on: after O += P_{j-1} V_{j-1} has finished
        if (j >= 1 && __any_sync(0xffffffffu, grown)) {
          if (!mbar_wait_warp_small(v_empty + ((tt - 1) & 1), ((tt - 1) >> 1) & 1, abort_flag, 0x8b)) { alive = false; break; }
          tc_fence_after();
          const float factor = grown ? ex2_approx(prev - m) : 1.f;
#pragma unroll 1
          for (int c = 0; c < kPR_D; c += 16) {
            uint32_t ow[16];
            tmem_ld16(trow + kPR_TmO + c, ow);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) ow[e] = __float_as_uint(__uint_as_float(ow[e]) * factor);
            tmem_st16(trow + kPR_TmO + c, ow);
          }
        }
        // a row that has seen nothing: scores of -inf against 0 give weights of 0, and a NaN stays one
        const float nm = m == -INFINITY ? 0.f : prompt_up<T>() - m;
        float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kPR_N; c += 32) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float e0 = ex2_approx(fmaf(uu[c + e], a.c2, nm)), e1 = ex2_approx(fmaf(uu[c + e + 1], a.c2, nm));
            ls[(e >> 1) & 3] += e0 + e1;
            pk[e / 2] = pack16<T>(e0, e1);
          }
          tmem_st16(srow + c / 2, pk);
        }
        l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(pf);
      }
      if (!alive) break;
      t += n;
      // the row's statistics for the output warps (slot it & 1, free once they read item it - 2's)
      const int slot = it & 1;
      if (it >= 2 && !(alive = mbar_wait_warp_small(&sfree[slot], ((it >> 1) - 1) & 1, abort_flag, 0x8c))) break;
      xl[slot * 256 + w * 128 + r] = l;
      xmx[slot * 256 + w * 128 + r] = m_own;
      __syncwarp();
      if (lane == 0) mbar_arrive(&stats[slot]);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPR_RegsEpi));
    // ------------------------------------------------------------------ outputs (warps 12..15)
    const int q4 = warp & 3, r = q4 * 32 + lane;
    const uint32_t trow = tmem + ((uint32_t)(q4 * 32) << 16);
    const uint32_t of = cluster_addr(o_free, 0);
    PromptItem x;
    for (int it = 0; item(it, true, x); ++it) {
      const bool store = r < x.rows;
      const int n = x.n;
      if (!mbar_wait_warp_small(o_fin, it & 1, abort_flag, 0x8d)) break;
      const int slot = it & 1;
      if (!mbar_wait_warp_small(&stats[slot], (it >> 1) & 1, abort_flag, 0x8e)) break;
      // the warpgroups' sums on the later reference, which is the greater
      const float m0 = xmx[slot * 256 + r], m1 = xmx[slot * 256 + 128 + r], m = fmaxf(m0, m1);
      const float l = xl[slot * 256 + r] * (m0 == -INFINITY ? 1.f : ex2_approx(m0 - m)) +
                      xl[slot * 256 + 128 + r] * (m1 == -INFINITY ? 1.f : ex2_approx(m1 - m));
      __syncwarp();
      if (lane == 0) mbar_arrive(&sfree[slot]);
      tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;        // nothing seen: zeros
      const int h = x.h;
      const size_t row = (size_t)x.row0 + r;
      if (store && a.lse) a.lse[(size_t)h * a.T + row] = l == 0.f ? -INFINITY : (m - prompt_up<T>() + log2f(l)) * kLn2;
      // 32 columns at a time through shared memory (16-byte chunks, swizzled by the row), so that a store instruction writes whole
      // 64-byte pieces of eight rows instead of 16 bytes of 32
      uint8_t* stage = s_out + (warp - 12) * 2048;
      const int r8 = lane >> 2, chunk = lane & 3;
      T* out = static_cast<T*>(a.o) + ((size_t)(x.row0 + q4 * 32) * a.H + h) * kPR_D + chunk * 8;
#pragma unroll 1
      for (int c = 0; c < kPR_D; c += 32) {
        uint32_t ow[32];
        if (n > 0) {
          tmem_ld32(trow + kPR_TmO + c, ow);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) ow[e] = 0u;
        }
        if (c + 32 == kPR_D) {           // O is free as soon as the last of it is in registers
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(of);
        }
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = pack16<T>(__uint_as_float(ow[8 * e + 2 * i]) * inv, __uint_as_float(ow[8 * e + 2 * i + 1]) * inv);
          *reinterpret_cast<uint4*>(stage + lane * 64 + ((e ^ ((lane >> 1) & 3)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int rr = 8 * i + r8;
          if (q4 * 32 + rr < x.rows)
            *reinterpret_cast<uint4*>(out + (size_t)rr * a.H * kPR_D + c) =
                *reinterpret_cast<const uint4*>(stage + rr * 64 + ((chunk ^ ((rr >> 1) & 3)) << 4));
        }
      }
    }
  }
  // neither CTA leaves while the other's products may read its shared memory or arrive on its barriers
  tc_fence_before();
  __syncthreads();
  if (tid == 0) report_abort(abort_flag, a.err);
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

template <typename T>
static int launch_prompt(const CUtensorMap& qmap, const CUtensorMap& kmap, const CUtensorMap& vmap, const PromptArgs& a,
                         long long clusters, cudaStream_t stream) {
  const int rc = ensure_smem_attr((const void*)prompt_attn_kernel<T>, kPR_Smem);
  if (rc) return rc;
  return launch_early(prompt_attn_kernel<T>, dim3((unsigned)(2 * clusters)), kPR_Threads, kPR_Smem, stream, qmap, kmap, vmap, a);
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
  if (D != kPR_D || (dtype != BF_BF16 && dtype != BF_F16)) return BF_ERR_UNSUPPORTED;
  if (Tk > kPR_MaxKeys || n_seq > kPR_MaxSeqs) return BF_ERR_UNSUPPORTED;
  if (T == 0) return BF_OK;
  if (!q || !o || (Tk > 0 && (!k || !v)) || (n_seq > 0 && !cu_q)) return BF_ERR_INVALID_ARGUMENT;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || ((q_st | q_sh | k_st | k_sh | v_st | v_sh) & 7))
    return BF_ERR_ALIGNMENT;
  if ((T > 1 && q_st <= 0) || (H > 1 && q_sh <= 0) || (Tk > 1 && (k_st <= 0 || v_st <= 0)) || (G > 1 && (k_sh <= 0 || v_sh <= 0)))
    return BF_ERR_INVALID_ARGUMENT;
  DeviceState st;
  int rc = device_state(&st);
  if (rc) return rc;
  PromptArgs a{};
  a.cu_q = cu_q;
  a.cu_k = cu_k ? cu_k : cu_q;
  a.n_seq = n_seq; a.T = T; a.Tk = Tk; a.H = H; a.G = G;
  a.c2 = scale * kLog2e;
  a.o = o;
  a.lse = lse;
  a.err = st.err;
  const int R = H / G;
  a.qb = R % 2 == 0 ? kPR_M : 2 * kPR_M;
  const long long nblk = (long long)T / a.qb + n_seq + 2;
  if (nblk > 0x7fffffffLL) return BF_ERR_UNSUPPORTED;
  a.nblk = (int)nblk;
  a.qlog = a.qb == kPR_M ? 7 : 8;
  a.hsplit = R % 2 == 0 ? R / 2 : R;
  while ((n_seq + 1) >> a.step_log >= kPR_Parts) ++a.step_log;
  const long long clusters = nblk * G * a.hsplit;
  if (clusters > 0x3fffffffLL) return BF_ERR_UNSUPPORTED;
  // (64 dims, tokens, 4 groups of 64 dims, heads); a stride of a dimension of one means nothing, and the encoder wants a positive one
  auto map = [&](CUtensorMap* m, const void* x, int rows, int heads, long long st_, long long sh_, uint32_t box_rows, uint32_t atoms) {
    const uint64_t dims[4] = {64, (uint64_t)rows, 4, (uint64_t)heads};
    const uint64_t str[3] = {(uint64_t)(st_ > 0 ? st_ : kPR_D) * 2, 128, (uint64_t)(sh_ > 0 ? sh_ : kPR_D) * 2};
    const uint32_t box[4] = {64, box_rows, atoms, 1};
    return make_tmap(m, x, dtype, 4, dims, str, box, true);
  };
  CUtensorMap qmap, kmap, vmap;
  if ((rc = map(&qmap, q, T, H, q_st, q_sh, kPR_M, 4))) return rc;
  // without a key no tile is loaded: any map will do
  if ((rc = map(&kmap, Tk ? k : q, Tk ? Tk : T, Tk ? G : H, Tk ? k_st : q_st, Tk ? k_sh : q_sh, kPR_N / 2, 4))) return rc;
  if ((rc = map(&vmap, Tk ? v : q, Tk ? Tk : T, Tk ? G : H, Tk ? v_st : q_st, Tk ? v_sh : q_sh, kPR_N, 2))) return rc;
  return dtype == BF_BF16 ? launch_prompt<__nv_bfloat16>(qmap, kmap, vmap, a, clusters, stream)
                          : launch_prompt<__half>(qmap, kmap, vmap, a, clusters, stream);
}

}  // extern "C"
