// Attention of sequences that have pages in common, each shared page read once for all of them.
//
//   o_b = softmax over [the runs of shared pages on b's way, b's own tail]; every part gives (m, l, acc) for each row, joined as
//   o = sum 2^(m_i - M) acc_i / sum 2^(m_i - M) l_i.
//
// A run of pages that `count` sequences share is met by count * t * R rows of queries per KV head at once, 128 of them to a tile of the
// tensor core.  A tile of 128 tokens is 64 KB from HBM per KV head, 2900 cycles of an SM's share, and with 128 rows 2048 cycles of 8-bit
// products: bound by HBM while a row block is alone with its pages, by the tensor core when several share them through L2.
// The e4m3 codes go untouched from TMA to the products (kind::f8f6f4); the other operands are split into e4m3 parts that add up, x = x0 + x1 (+ x2
// in fp16), so that a product's parts accumulate in one place:
//   S[row, token] = sum_p Q_p K^T     M = 128 rows, N = 128 tokens, K = 256 dims x parts
//   O[row, dim]   = sum_p P_p V       M = 128 rows, N = 2 x 128 dims, K = 128 tokens x parts      (V as it lies: N-major)
// Two parts hold 9 bits, three 13.  A query's row is scaled to [128, 256), a weight to its row's largest in the tile = 256: the parts end at 2^-9
// of that scale, so a component is off by at most 2^-17 of its row's largest, a weight by 2^-18 of the tile's largest (weights beside a
// heavy token of another tile keep their bits: every tile's O is scaled for itself and added up in registers, in fp32).
// V's power-of-two scales join the exponents: w = 2^(s + log2 sv - m) with m their largest, and the sum of weights takes 1 / sv back.
//
// Work: the tiles of all (run, KV head, row block) in one line, cut into equal runs, one per CTA, one CTA per SM; an item's start counts as kSH_Start tiles.
// Every piece writes its rows' partial, and paged_merge_kernel adds them and the tails (paged_attn.cu) in a fixed order.
// Warps: 0 TMA of K and the tiles' scales, 1 the products S, 2 TMA of V, 3 the products O; a warpgroup of softmax (thread = row), two of
// accumulators (thread = row and half of the dims); these three also make an item's query parts.
#include "bifrost_b200.h"
#include "common.cuh"
#include "launch_early.h"
#include "paged_attn.h"
#include "tmap.h"

namespace bfb {

constexpr int kSH_M = 128, kSH_N = 128;              // rows, tokens of a tile
constexpr int kSH_Unit = 128 * 128;                  // bytes of half a K or V tile: 128 tokens, 128 dims
constexpr int kSH_Threads = 512;
constexpr int kSH_Start = 2;
// register split (setmaxnreg) of the 128 per thread at launch
constexpr uint32_t kSH_RegsCtl = 80, kSH_RegsSoftmax = 112, kSH_RegsAcc = 160;
static_assert(128 * kSH_RegsCtl + 128 * kSH_RegsSoftmax + 256 * kSH_RegsAcc <= kSH_Threads * 128, "register split");

template <typename T>
struct SharedCfg {
  static constexpr int Parts = 3;
  static constexpr int NK = 2, NV = 2;               // half tiles that fit beside Q and P
};
template <>
struct SharedCfg<__nv_bfloat16> {
  static constexpr int Parts = 2;
  static constexpr int NK = 4, NV = 3;
};
template <typename T>
struct SharedSmem {
  using C = SharedCfg<T>;
  static constexpr int Q = C::Parts * 2 * kSH_M * 128, P = C::Parts * kSH_M * 128;
  static constexpr int Tiles = (C::NK + C::NV) * kSH_Unit + Q + P;
  static constexpr int Bytes = Tiles + 512 + 4 * 32 * 4 + 2 * 128 * 8 + 128 * 4 + 1024;
};

struct SharedArgs {
  PagePool p;
  const void* q;
  long long q_sb, q_st, q_sh;
  const int32_t* plan;
  int n, t, H, R;
  int page_log;
  float c2;             // scale * log2(e)
  int4* head;           // units per CTA, CTAs with one more, -, -
  int2* at;             // [runs] the run's first unit, rows before it
  float* part;          // [CTAs * 128 + rows][256], a piece's rows x dims transposed
  float2* ml;           // [CTAs * 128 + rows] maximum, sum
  // the tails, and the result
  PagedTail tail;
  void* o;
  float* lse;
  unsigned int* err;
};

// the plan's arrays
struct Plan {
  const int32_t *slots, *order, *place, *last, *skip, *runs;
  int n_runs;
  __device__ __forceinline__ Plan(const int32_t* p, int n)
      : slots(p + kPS_Head), order(slots + n), place(order + n), last(place + n), skip(last + n), runs(skip + n), n_runs(min(max(p[0], 0), n)) {}
};

// the line of work: run by run, KV head by KV head, row block by row block, tile by tile
struct SharedWalk {
  int run, g, rb, tile;
  int ntiles, blocks, rows, first, page0, page1;      // of the run: tiles, row blocks, rows, first place, pages
  int base;                                           // rows of the items before this one
  __device__ __forceinline__ void enter(const SharedArgs& a, const Plan& pl) {
    const int32_t* r = pl.runs + (size_t)run * kPS_Run;
    first = r[0];
    rows = r[1] * a.t * a.R;
    page0 = r[2];
    page1 = r[3];
    blocks = (rows + kSH_M - 1) / kSH_M;
    ntiles = max(1, (int)((((long long)(page1 - page0) << a.page_log) + kSH_N - 1) / kSH_N));
  }
  __device__ __forceinline__ int block_rows() const { return min(kSH_M, rows - rb * kSH_M); }
  __device__ __forceinline__ bool last_tile() const { return tile + 1 == ntiles; }
  __device__ __forceinline__ void next(const SharedArgs& a, const Plan& pl) {
    if (++tile < ntiles) return;
    tile = 0;
    base += block_rows();
    if (++rb < blocks) return;
    rb = 0;
    if (++g < a.p.heads) return;
    g = 0;
    if (++run < pl.n_runs) enter(a, pl);
  }
};
__device__ __forceinline__ int run_units(const SharedArgs& a, const int32_t* r, int* rows) {
  *rows = r[1] * a.t * a.R;
  const int ntiles = max(1, (int)((((long long)(r[3] - r[2]) << a.page_log) + kSH_N - 1) / kSH_N));
  const int units = a.p.heads * ((*rows + kSH_M - 1) / kSH_M) * (ntiles + kSH_Start);
  *rows *= a.p.heads;
  return units;
}

// two values as e4m3 parts that add up; each remainder is exact in fp16
template <int Parts>
__device__ __forceinline__ void split_sum(__half2 x, uint16_t (&part)[Parts]) {
#pragma unroll
  for (int i = 0; i < Parts; ++i) {
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(part[i]) : "r"(*reinterpret_cast<uint32_t*>(&x)));
    if (i + 1 < Parts) {
      uint32_t f;
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(f) : "h"(part[i]));
      x = __hsub2(x, *reinterpret_cast<__half2*>(&f));
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kSH_Threads, 1)
    paged_shared_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, SharedArgs a) {
  using C = SharedCfg<T>;
  constexpr int Parts = C::Parts, NK = C::NK, NV = C::NV;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));   // K's half tiles, then V's
  uint8_t* sQ = ring + (NK + NV) * kSH_Unit;           // [parts][2 atoms][128 rows][128]
  uint8_t* sP = sQ + SharedSmem<T>::Q;                 // [parts][128 rows][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sP + SharedSmem<T>::P);
  uint64_t *k_full = bars, *k_empty = bars + 4, *v_full = bars + 8, *v_empty = bars + 12, *s_full = bars + 16, *s_free = bars + 18,
           *p_full = bars + 20, *o_full = bars + 22, *o_free = bars + 23, *q_full = bars + 24, *q_free = bars + 25, *sc_full = bars + 26,
           *sc_free = bars + 30;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 34);
  volatile int* abort = reinterpret_cast<volatile int*>(bars + 35);
  int* s_sum = reinterpret_cast<int*>(bars + 36);      // [16][2] per-warp totals
  int* s_start = reinterpret_cast<int*>(bars + 52);    // run, unit in it, rows before it
  float* s_sc = reinterpret_cast<float*>(bars + 64);   // [4][32]: a tile's K scales, V exponents, 1 / V scales; 24: which pages are there
  float2* s_fac = reinterpret_cast<float2*>(s_sc + 128);          // [2][128] factors of the accumulators and of the tile's O
  float* s_qs = reinterpret_cast<float*>(s_fac + 256);            // [128] scale of the Q rows
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < 4; ++i) {
      mbar_init(k_full + i, 1);
      mbar_init(k_empty + i, 1);
      mbar_init(v_full + i, 1);
      mbar_init(v_empty + i, 1);
      mbar_init(sc_full + i, 1);
      mbar_init(sc_free + i, 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(s_free + i, 4);
      mbar_init(p_full + i, 4);
    }
    mbar_init(o_full, 1);
    mbar_init(o_free, 8);
    mbar_init(q_full, 12);
    mbar_init(q_free, 1);
    *abort = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) tma_prefetch(&kmap);
  if (warp == 2 && lane == 0) tma_prefetch(&vmap);
  wait_for_stream();
  let_next_start();
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  // this CTA's part of the line: the runs' units summed over the block, thread i holding `per` consecutive runs
  const Plan pl(a.plan, a.n);
  const int per = (pl.n_runs + kSH_Threads - 1) / kSH_Threads;
  int2 mine = make_int2(0, 0);
  for (int i = 0; i < per; ++i) {
    const int r = tid * per + i;
    if (r < pl.n_runs) {
      int rows;
      mine.x += run_units(a, pl.runs + (size_t)r * kPS_Run, &rows);
      mine.y += rows;
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
  if (lane == 31) {
    s_sum[2 * warp] = incl.x;
    s_sum[2 * warp + 1] = incl.y;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  int total = lane < 16 ? s_sum[2 * lane] : 0;
  const int rows_w = lane < 16 ? s_sum[2 * lane + 1] : 0;
  int2 before = make_int2(lane < warp ? total : 0, lane < warp ? rows_w : 0);
  total = (int)__reduce_add_sync(0xffffffffu, (unsigned)total);
  before.x = (int)__reduce_add_sync(0xffffffffu, (unsigned)before.x) + incl.x - mine.x;
  before.y = (int)__reduce_add_sync(0xffffffffu, (unsigned)before.y) + incl.y - mine.y;
  const int ctas = max(1, min(total, (int)gridDim.x)), each = total / ctas, more = total - each * ctas;
  const int u0 = min((int)blockIdx.x, ctas) * each + min((int)blockIdx.x, more);
  const int u1 = u0 + ((int)blockIdx.x < ctas ? each + ((int)blockIdx.x < more ? 1 : 0) : 0);
  {
    int2 at = before;
    for (int i = 0; i < per; ++i) {
      const int r = tid * per + i;
      if (r >= pl.n_runs) break;
      int rows;
      const int units = run_units(a, pl.runs + (size_t)r * kPS_Run, &rows);
      if (blockIdx.x == 0) a.at[r] = at;
      if (u0 < u1 && at.x <= u0 && u0 < at.x + units) {
        s_start[0] = r;
        s_start[1] = u0 - at.x;
        s_start[2] = at.y;
      }
      at.x += units;
      at.y += rows;
    }
    if (blockIdx.x == 0 && tid == 0) *a.head = make_int4(each, more, 0, 0);
  }
  __syncthreads();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  SharedWalk w{};
  int count = 0;                  // tiles of this CTA
  if (u0 < u1) {
    w.run = s_start[0];
    w.enter(a, pl);
    const int len = w.ntiles + kSH_Start, item = s_start[1] / len, in = s_start[1] - item * len;
    w.g = item / w.blocks;
    w.rb = item - w.g * w.blocks;
    w.base = s_start[2] + w.g * w.rows + w.rb * kSH_M;
    w.tile = max(in - kSH_Start, 0);
    SharedWalk x = w;
    for (int u = u0 - in; u < u1;) {
      count += max(min(u + kSH_Start + x.ntiles, u1) - max(u + kSH_Start, u0), 0);
      u += x.ntiles + kSH_Start;
      x.tile = x.ntiles - 1;
      x.next(a, pl);
    }
  }
  count = __shfl_sync(0xffffffffu, count, 0);
  const int L = a.p.page, ppt = kSH_N >> a.page_log;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kSH_RegsCtl));
    if (warp == 0 || warp == 2) {
      // ---------------------------------------------------------------- codes: K (warp 0, with the scales), V (warp 2)
      const bool is_v = warp == 2;
      const void* map = is_v ? &vmap : &kmap;
      uint64_t *full = is_v ? v_full : k_full, *empty = is_v ? v_empty : k_empty;
      uint8_t* base = ring + (is_v ? NK * kSH_Unit : 0);
      const int units = is_v ? NV : NK;
      int u = 0, uphase = 1, used = 0;
      bool ok = true;
#pragma unroll 1
      for (int j = 0; j < count && ok; ++j) {
        // lane i: the tile's page i; where the run has none, its last one, whose tokens nobody sees twice (no code may stay from another tile:
        // a weight of 0 times NaN would be NaN)
        const int slot = pl.slots[pl.order[w.first]];
        const int pages = w.page1 - w.page0, pi = min(w.tile * ppt + lane, pages - 1);
        int page = -1;
        if (lane < ppt && slot >= 0 && slot < a.p.slots && w.page0 + pi < a.p.width) page = a.p.table[(size_t)slot * a.p.width + w.page0 + pi];
        const bool there = page >= 0 && page < a.p.pages;
        page = there ? page : 0;
        const int row = (page * a.p.heads + w.g) * L;
        if (!is_v) {
          const int s = j & 3;
          float ks = 1.f;
          int e = 0;
          if (lane < ppt && there) {
            ks = a.p.ks[(size_t)page * a.p.heads + w.g];
            e = (int)(__float_as_uint(a.p.vs[(size_t)page * a.p.heads + w.g]) >> 23) - 127;      // scales are powers of two
            e = max(e, -120);
          }
          const unsigned have = __ballot_sync(0xffffffffu, lane < ppt && there && w.tile * ppt + lane < pages);
          if (j >= 4 && !(ok = mbar_wait_warp_small(sc_free + s, ((j >> 2) - 1) & 1, abort, 0x90))) break;
          if (lane < 8) {
            s_sc[s * 32 + lane] = ks;
            s_sc[s * 32 + 8 + lane] = (float)e;
            s_sc[s * 32 + 16 + lane] = __uint_as_float((uint32_t)(127 - e) << 23);
          }
          if (lane == 0) s_sc[s * 32 + 24] = __uint_as_float(have);
          __syncwarp();
          if (lane == 0) mbar_arrive(sc_full + s);
        }
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          if (used >= units && !(ok = mbar_wait_warp_small(empty + u, uphase, abort, 0x91))) break;
          if (lane == 0) mbar_expect_tx(full + u, kSH_Unit);
          __syncwarp();
#pragma unroll 1
          for (int i = 0; i < ppt; ++i) {
            const int r = __shfl_sync(0xffffffffu, row, i);
            if (elect_one()) tma_load_2d(base + u * kSH_Unit + i * L * 128, map, full + u, 128 * half, r);
            __syncwarp();
          }
          ++used;
          if (++u == units) {
            u = 0;
            uphase ^= 1;
          }
        }
        w.next(a, pl);
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- S = sum_p Q_p K^T
      constexpr uint32_t id = idesc_e4m3(kSH_M, kSH_N);
      const uint64_t dk0 = sdesc_sw128(smem_u32(ring)), dq0 = sdesc_sw128(smem_u32(sQ));
      int u = 0, uphase = 0, item = 0;
      bool first = true;
#pragma unroll 1
      for (int j = 0; j < count; ++j) {
        const int s = j & 1;
        if (first && !mbar_wait_warp_small(q_full, item & 1, abort, 0x92)) break;
        if (j >= 2 && !mbar_wait_warp_small(s_free + s, ((j >> 1) - 1) & 1, abort, 0x93)) break;
        const bool end = w.last_tile() || j + 1 == count;
        bool ok = true;
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          if (!(ok = mbar_wait_warp_small(k_full + u, uphase, abort, 0x94))) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t dk = dk0 + (uint32_t)(u * (kSH_Unit >> 4));
#pragma unroll
            for (int p = 0; p < Parts; ++p)
#pragma unroll
              for (int ks = 0; ks < 4; ++ks)
                umma_f8_ss(tmem + s * kSH_N, dq0 + (uint32_t)((p * 2 + half) * (kSH_Unit >> 4) + ks * 2), dk + ks * 2, id, half > 0 || p > 0 || ks > 0);
            umma_commit(k_empty + u);
            if (half) {
              umma_commit(s_full + s);
              if (end) umma_commit(q_free);
            }
          }
          __syncwarp();
          if (++u == NK) {
            u = 0;
            uphase ^= 1;
          }
        }
        if (!ok) break;
        item += end;
        first = end;
        w.next(a, pl);
      }
    } else {
      // ---------------------------------------------------------------- O = sum_p P_p V
      constexpr uint32_t id = idesc_e4m3(kSH_M, 128) | kIdescBMn;
      const uint64_t dv0 = sdesc_sw128_mn(smem_u32(ring + NK * kSH_Unit), 16384), dp0 = sdesc_sw128(smem_u32(sP));
      int u = 0, uphase = 0;
#pragma unroll 1
      for (int j = 0; j < count; ++j) {
        if (!mbar_wait_warp_small(p_full + (j & 1), (j >> 1) & 1, abort, 0x95)) break;
        if (j >= 1 && !mbar_wait_warp_small(o_free, (j - 1) & 1, abort, 0x96)) break;
        bool ok = true;
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          if (!(ok = mbar_wait_warp_small(v_full + u, uphase, abort, 0x97))) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t dv = dv0 + (uint32_t)(u * (kSH_Unit >> 4));
#pragma unroll
            for (int p = 0; p < Parts; ++p)
#pragma unroll
              for (int ks = 0; ks < 4; ++ks)
                umma_f8_ss(tmem + 256 + half * 128, dp0 + (uint32_t)(p * (kSH_Unit >> 4) + ks * 2), dv + ks * (4096 >> 4), id, p > 0 || ks > 0);
            umma_commit(v_empty + u);
            if (half) umma_commit(o_full);
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
    // a row of the block: its sequence's place, token and head
    const int per_seq = a.t * a.R;
    auto row_of = [&](const SharedWalk& x, int r, int& b, int& i, int& h) {
      const int idx = x.rb * kSH_M + r, k = idx / per_seq, rem = idx - k * per_seq;
      b = pl.order[x.first + k];
      i = rem / a.R;
      h = x.g * a.R + rem - i * a.R;
    };
    // an item's query parts: warp w of 12 takes the rows w, w + 12, ..., lane l dims 8 l .. 8 l + 7.  Lane k finds where the warp's row k lies.
    auto queries = [&](const SharedWalk& x) {
      const int rows = x.block_rows(), w12 = warp - 4;
      long long at = 0;
      if (w12 + 12 * lane < rows) {
        int b, i, h;
        row_of(x, w12 + 12 * lane, b, i, h);
        at = b * a.q_sb + i * a.q_st + h * a.q_sh;
        const T* p = static_cast<const T*>(a.q) + at;
#pragma unroll
        for (int k = 0; k < 4; ++k) prefetch_l2(p + 64 * k);
      }
#pragma unroll 1
      for (int k0 = 0; w12 + 12 * k0 < rows; k0 += 4) {
        uint4 raw[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const long long from = __shfl_sync(0xffffffffu, at, k0 + k);
          if (w12 + 12 * (k0 + k) < rows) raw[k] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + from + 8 * lane));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = w12 + 12 * (k0 + k);
          if (r >= rows) break;
          const uint32_t v[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
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
          for (int e2 = 0; e2 < 4; ++e2) {
            const T* e = reinterpret_cast<const T*>(&v[e2]);
            split_sum<Parts>(__floats2half2_rn(fin ? (float)e[0] * up : 0.f, fin ? (float)e[1] * up : 0.f), c[e2]);
          }
          uint8_t* dst = sQ + (lane >> 4) * kSH_Unit + r * 128 + ((((lane & 15) >> 1) ^ (r & 7)) << 4) + (lane & 1) * 8;
#pragma unroll
          for (int p = 0; p < Parts; ++p)
            *reinterpret_cast<uint2*>(dst + p * 2 * kSH_Unit) = make_uint2(c[0][p] | ((uint32_t)c[1][p] << 16), c[2][p] | ((uint32_t)c[3][p] << 16));
          // a row with a value that is not finite has no finite scores
          if (lane == 0) s_qs[r] = fin ? __uint_as_float((uint32_t)(ex - 7) << 23) * a.c2 : NAN;
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    };
    const int wq = warp & 3, r = wq * 32 + lane;      // this thread's row
    int item = 0;
    bool ok = true, first = true;
    if (warp < 8) {
      // ---------------------------------------------------------------- softmax: thread = row
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kSH_RegsSoftmax));
      const uint32_t trow = tmem + ((uint32_t)(wq * 32) << 16);
      float m_run = -INFINITY, l = 0.f, qs = 0.f;
      int limit = -1, rows = 0;            // the last position that the row sees
#pragma unroll 1
      for (int j = 0; j < count; ++j) {
        const int s = j & 1;
        if (first) {
          if (item && !(ok = mbar_wait_warp_small(q_free, (item - 1) & 1, abort, 0x98))) break;
          queries(w);
          if (!(ok = mbar_wait_warp_small(q_full, item & 1, abort, 0x99))) break;
          rows = w.block_rows();
          m_run = -INFINITY;
          l = 0.f;
          limit = -1;
          if (r < rows) {
            int b, i, h;
            row_of(w, r, b, i, h);
            const int slot = pl.slots[b];
            if (slot >= 0 && slot < a.p.slots) limit = a.p.lens[slot] - a.t + i;
            qs = s_qs[r];
          }
        }
        const bool end = w.last_tile() || j + 1 == count, busy = wq * 32 < rows;
        if (!(ok = mbar_wait_warp_small(sc_full + (j & 3), (j >> 2) & 1, abort, 0x9a))) break;
        if (!(ok = mbar_wait_warp_small(s_full + s, (j >> 1) & 1, abort, 0x9b))) break;
        tc_fence_after();
        const float* sc = s_sc + (j & 3) * 32;
        const unsigned have = __float_as_uint(sc[24]);
        // the tokens of the tile that the row sees are its first `vis`, of pages that are there
        const long long pos0 = ((long long)w.page0 << a.page_log) + w.tile * kSH_N;
        const int vis = (int)max(min((long long)limit - pos0 + 1, (long long)kSH_N), 0ll);
        const bool all = have == (ppt == 32 ? ~0u : (1u << ppt) - 1u) && __all_sync(0xffffffffu, vis == kSH_N || r >= rows);
        float mt = -INFINITY, lt = 0.f;
        if (busy) {
          // two ways through the row's scores (they do not fit the registers): its largest, then the weights
#pragma unroll 1
          for (int c = 0; c < kSH_N; c += 32) {
            uint32_t x[32];
            tmem_ld32(trow + s * kSH_N + c, x);
            tmem_wait_ld();
            if (!all) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (c + i >= vis || !((have >> ((c + i) >> a.page_log)) & 1u)) x[i] = 0xff800000u;
            }
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              float mx = __uint_as_float(x[16 * q]);
#pragma unroll
              for (int i = 1; i < 16; ++i) mx = fmaxf(mx, __uint_as_float(x[16 * q + i]));
              const int pi = (c + 16 * q) >> a.page_log;
              mt = fmaxf(mt, fmaf(mx, sc[pi] * qs, sc[8 + pi]));
            }
          }
        }
        // tile j - 1's products have read P
        if (j >= 1 && !(ok = mbar_wait_warp_small(o_full, (j - 1) & 1, abort, 0x9c))) break;
        if (busy) {
          const float ref = mt == -INFINITY ? 0.f : mt;
#pragma unroll 1
          for (int c = 0; c < kSH_N; c += 32) {
            uint32_t x[32];
            tmem_ld32(trow + s * kSH_N + c, x);
            tmem_wait_ld();
            if (!all) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (c + i >= vis || !((have >> ((c + i) >> a.page_log)) & 1u)) x[i] = 0xff800000u;
            }
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int pi = (c + 16 * q) >> a.page_log;
              const float f = sc[pi] * qs, off = sc[8 + pi] - ref;
              float sum = 0.f;
              uint32_t out[Parts][4];
#pragma unroll
              for (int i = 0; i < 16; i += 2) {
                const float w0 = ex2_approx(fmaf(__uint_as_float(x[16 * q + i]), f, off)), w1 = ex2_approx(fmaf(__uint_as_float(x[16 * q + i + 1]), f, off));
                sum += w0 + w1;
                uint16_t pt[Parts];
                split_sum<Parts>(__floats2half2_rn(w0 * 256.f, w1 * 256.f), pt);
#pragma unroll
                for (int p = 0; p < Parts; ++p) out[p][i >> 2] = (i & 2) ? out[p][i >> 2] | ((uint32_t)pt[p] << 16) : pt[p];
              }
              lt = fmaf(sum, sc[16 + pi], lt);
              uint8_t* dst = sP + r * 128 + ((((c >> 4) + q) ^ (r & 7)) << 4);
#pragma unroll
              for (int p = 0; p < Parts; ++p) *reinterpret_cast<uint4*>(dst + p * kSH_Unit) = make_uint4(out[p][0], out[p][1], out[p][2], out[p][3]);
            }
          }
        }
        tc_fence_before();
        const float mn = fmaxf(m_run, mt);
        const float al = m_run == -INFINITY ? 0.f : ex2_approx(m_run - mn), f = mt == -INFINITY ? 0.f : ex2_approx(mt - mn);
        l = mt == -INFINITY && !(lt != lt) ? l * (m_run == -INFINITY ? 1.f : al) : l * al + lt * (lt != lt ? 1.f : f);
        m_run = mn;
        s_fac[s * kSH_M + r] = make_float2(al, mt == -INFINITY ? (1.f / 256.f) : f * (1.f / 256.f));
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(s_free + s);
          mbar_arrive(sc_free + (j & 3));
          mbar_arrive(p_full + s);
        }
        if (end) {
          if (r < rows) a.ml[(size_t)blockIdx.x * kSH_M + w.base + r] = make_float2(m_run, l);
          ++item;
        }
        first = end;
        w.next(a, pl);
      }
    } else {
      // ---------------------------------------------------------------- accumulators: thread = row, half of the dims
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSH_RegsAcc));
      const int half = (warp - 8) >> 2;
      const uint32_t trow = tmem + 256 + half * 128 + ((uint32_t)(wq * 32) << 16);
      uint64_t acc[64];
      int rows = 0;
#pragma unroll 1
      for (int j = 0; j < count; ++j) {
        if (first) {
          if (item && !(ok = mbar_wait_warp_small(q_free, (item - 1) & 1, abort, 0x9d))) break;
          queries(w);
          rows = w.block_rows();
#pragma unroll
          for (int i = 0; i < 64; ++i) acc[i] = 0;
        }
        const bool end = w.last_tile() || j + 1 == count, busy = wq * 32 < rows;
        if (!(ok = mbar_wait_warp_small(p_full + (j & 1), (j >> 1) & 1, abort, 0x9e))) break;      // the factors
        if (!(ok = mbar_wait_warp_small(o_full, j & 1, abort, 0x9f))) break;
        tc_fence_after();
        if (busy) {
          const float2 fac = s_fac[(j & 1) * kSH_M + r];
          const uint64_t al = pair2(fac.x, fac.x), f = pair2(fac.y, fac.y);
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint32_t x[16];
            tmem_ld16(trow + 16 * c, x);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              uint64_t y;
              asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(acc[8 * c + i]), "l"(al));
              acc[8 * c + i] = fma2(pair2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), f, y);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(o_free);
        if (end) {
          if (r < rows) {
            // a piece lies dim by dim, so that 32 rows are neighbours
            float* to = a.part + ((size_t)blockIdx.x * kSH_M + w.base) * kPG_D + (size_t)half * 128 * rows + r;
#pragma unroll
            for (int i = 0; i < 64; ++i) {
              to[(size_t)(2 * i) * rows] = lo_hi(acc[i], 0);
              to[(size_t)(2 * i + 1) * rows] = lo_hi(acc[i], 1);
            }
          }
          ++item;
        }
        first = end;
        w.next(a, pl);
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

// Output rows: a warp has 32 neighbouring rows of one KV head, in the plan's order (they are neighbours in every piece too), and 16 dims; a lane adds its
// row's pieces run by run from the last one up, CTA by CTA, then the tail.
template <typename T>
__global__ void __launch_bounds__(256) paged_merge_kernel(SharedArgs a) {
  wait_for_stream();
  let_next_start();
  const int lane = threadIdx.x & 31, d0 = (blockIdx.y * 8 + (threadIdx.x >> 5)) * 16, g = blockIdx.z;
  const Plan pl(a.plan, a.n);
  const int per_seq = a.t * a.R;
  const long long sr = (long long)blockIdx.x * 32 + lane;
  const bool on = sr < (long long)a.n * per_seq;
  const int place = on ? (int)(sr / per_seq) : 0, rem = on ? (int)(sr - (long long)place * per_seq) : 0, i = rem / a.R, hh = rem - i * a.R;
  if (!on) return;
  const int b = pl.order[place], h = g * a.R + hh;
  const int4 head = *a.head;
  const int each = head.x, more = head.y, longer = more * (each + 1);
  auto cta_of = [&](int u) { return u < longer ? u / (each + 1) : more + (u - longer) / each; };
  float m = -INFINITY, sum = 0.f, acc[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) acc[k] = 0.f;
  auto add = [&](float2 ml, const float (&v)[16]) {
    // a partial without a maximum holds zeros, or NaN to be passed on
    const float mn = fmaxf(m, ml.x);
    const float al = m == -INFINITY ? 1.f : ex2_approx(m - mn), f = ml.x == -INFINITY ? 1.f : ex2_approx(ml.x - mn);
#pragma unroll
    for (int k = 0; k < 16; ++k) acc[k] = acc[k] * al + v[k] * f;
    sum = sum * al + ml.y * f;
    m = mn;
  };
  for (int run = pl.last[b], guard = 0; run >= 0 && run < pl.n_runs && guard < kPS_Depth; ++guard) {
    const int32_t* r = pl.runs + (size_t)run * kPS_Run;
    const int rows = r[1] * per_seq, blocks = (rows + kSH_M - 1) / kSH_M, idx = (place - r[0]) * per_seq + rem, rb = idx / kSH_M, in = idx - rb * kSH_M;
    const int ntiles = max(1, (int)((((long long)(r[3] - r[2]) << a.page_log) + kSH_N - 1) / kSH_N)), block_rows = min(kSH_M, rows - rb * kSH_M);
    const int2 at = a.at[run];
    const int u = at.x + (g * blocks + rb) * (ntiles + kSH_Start) + kSH_Start;
    const size_t base = (size_t)at.y + (size_t)g * rows + rb * kSH_M;
    const int c1 = cta_of(u + ntiles - 1);
    for (int c = cta_of(u); c <= c1; c += 2) {
      float v[2][16];
      float2 ml[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const size_t row0 = (size_t)min(c + x, c1) * kSH_M + base;
        ml[x] = a.ml[row0 + in];
        const float* p = a.part + row0 * kPG_D + (size_t)d0 * block_rows + in;
#pragma unroll
        for (int k = 0; k < 16; ++k) v[x][k] = p[(size_t)k * block_rows];
      }
      add(ml[0], v[0]);
      if (c < c1) add(ml[1], v[1]);
    }
    run = r[4];
  }
  {
    const int chunk = i / a.tail.tc;
    const int2 seg = a.tail.seg[((size_t)b * a.tail.nqc + chunk) * a.p.heads + g];
    const int rr = (i - chunk * a.tail.tc) * a.R + hh;
    auto piece = [&](const float* p) {
      float v[16];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float4 x = *reinterpret_cast<const float4*>(p + d0 + 4 * k);
        v[4 * k] = x.x, v[4 * k + 1] = x.y, v[4 * k + 2] = x.z, v[4 * k + 3] = x.w;
      }
      add(*reinterpret_cast<const float2*>(p + kPG_D), v);
    };
    if (seg.x < 0) {
      piece(a.tail.tail + (((size_t)b * a.t + i) * a.H + h) * kPA_Part);
    } else {
      for (int c = seg.x; c <= min(seg.y, kPA_MaxCtas - 1); ++c)
        piece(a.tail.part + (((size_t)c * 2 + (c == seg.x ? 1 : 0)) * a.tail.rp + rr) * kPA_Part);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;       // nothing seen: zeros
  uint4 out[2];
  T* o = reinterpret_cast<T*>(out);
#pragma unroll
  for (int k = 0; k < 16; ++k) o[k] = (T)(acc[k] * inv);
  uint4* to = reinterpret_cast<uint4*>(static_cast<T*>(a.o) + (((size_t)b * a.t + i) * a.H + h) * kPG_D + d0);
  to[0] = out[0];
  to[1] = out[1];
  if (a.lse && d0 == 0) a.lse[((size_t)b * a.H + h) * a.t + i] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * kLn2;
}

template <typename T>
static int launch_shared(const SharedArgs& a, const CUtensorMap& kmap, const CUtensorMap& vmap, int ctas, cudaStream_t stream) {
  const int rc = ensure_smem_attr((const void*)paged_shared_kernel<T>, SharedSmem<T>::Bytes);
  return rc ? rc : launch_early(paged_shared_kernel<T>, dim3(ctas), kSH_Threads, SharedSmem<T>::Bytes, stream, kmap, vmap, a);
}

struct SharedLayout {
  size_t at, ml, part, tail, bytes;
};
static SharedLayout shared_layout(int n, int t, int H, int G) {
  SharedLayout x;
  const size_t rows = (size_t)kPA_MaxCtas * kSH_M + (size_t)kPS_Depth * n * t * H;
  x.at = 16;
  x.ml = x.at + ((size_t)n * sizeof(int2) + 15) / 16 * 16;
  x.part = x.ml + rows * sizeof(float2);
  x.tail = x.part + rows * kPG_D * 4;
  x.bytes = x.tail + paged_tail_workspace(n, t, H, G);
  return x;
}

}  // namespace bfb

using namespace bfb;

extern "C" {

size_t bf_paged_attend_shared_workspace(int n, int t, int H, int G, int D) {
  if (n <= 0 || t <= 0 || H <= 0 || G <= 0 || H % G || H / G > kPA_MaxGroup || D != kPG_D) return 0;
  return shared_layout(n, t, H, G).bytes;
}

int bf_paged_attend_shared(const bf_page_pool* pool, int layer, const void* q, long long q_sb, long long q_st, long long q_sh, const int32_t* plan,
                           int n, int t, int H, int dtype, float scale, void* o, float* lse, void* ws, size_t ws_bytes, bf_stream_t stream) {
  SharedArgs a{};
  int rc = page_pool(pool, layer, &a.p);
  if (rc) return rc;
  if (n < 0 || t < 0 || H <= 0 || H % a.p.heads || !(scale > 0.f) || scale > 3e38f) return BF_ERR_INVALID_ARGUMENT;
  if ((dtype != BF_BF16 && dtype != BF_F16) || H / a.p.heads > kPA_MaxGroup) return BF_ERR_UNSUPPORTED;
  if (n == 0 || t == 0) return BF_OK;
  if (!q || !o || !plan) return BF_ERR_INVALID_ARGUMENT;
  if (!aligned16(q) || !aligned16(o) || !aligned16(plan) || ((q_sb | q_st | q_sh) & 7)) return BF_ERR_ALIGNMENT;
  // units and rows are counted in 32 bits: every sequence's runs cover its table's pages once at most
  const long long rows = (long long)n * t * H, tiles = (long long)a.p.width * a.p.page / kSH_N + kPS_Depth * (kSH_Start + 1);
  if (kPS_Depth * rows + (long long)kPA_MaxCtas * kSH_M > 0x7fffffffLL || (rows / kSH_M + (long long)n * a.p.heads) * tiles > 0x7fffffffLL)
    return BF_ERR_UNSUPPORTED;
  const SharedLayout x = shared_layout(n, t, H, a.p.heads);
  if (!ws || ws_bytes < x.bytes) return BF_ERR_WORKSPACE;
  if (!aligned16(ws)) return BF_ERR_ALIGNMENT;
  DeviceState st;
  if ((rc = device_state(&st))) return rc;
  uint8_t* at = static_cast<uint8_t*>(ws);
  a.q = q;
  a.q_sb = q_sb; a.q_st = q_st; a.q_sh = q_sh;
  a.plan = plan;
  a.n = n; a.t = t; a.H = H; a.R = H / a.p.heads;
  a.page_log = a.p.page == 16 ? 4 : a.p.page == 32 ? 5 : a.p.page == 64 ? 6 : 7;
  a.c2 = scale * kLog2e;
  a.head = reinterpret_cast<int4*>(at);
  a.at = reinterpret_cast<int2*>(at + x.at);
  a.ml = reinterpret_cast<float2*>(at + x.ml);
  a.part = reinterpret_cast<float*>(at + x.part);
  a.o = o;
  a.lse = lse;
  a.err = st.err;
  CUtensorMap kmap, vmap;
  if ((rc = paged_maps(a.p, &kmap, &vmap))) return rc;
  const int ctas = st.sm_count < kPA_MaxCtas ? st.sm_count : kPA_MaxCtas;
  rc = dtype == BF_BF16 ? launch_shared<__nv_bfloat16>(a, kmap, vmap, ctas, stream) : launch_shared<__half>(a, kmap, vmap, ctas, stream);
  if (rc) return rc;
  const int32_t* slots = plan + kPS_Head;
  rc = paged_tail(a.p, q, q_sb, q_st, q_sh, slots, slots + 4 * (size_t)n, n, t, H, dtype, scale, at + x.tail, st, stream, &a.tail);
  if (rc) return rc;
  const dim3 grid((unsigned)(((long long)n * t * a.R + 31) / 32), 2, a.p.heads);
  return dtype == BF_BF16 ? launch_early(paged_merge_kernel<__nv_bfloat16>, grid, 256, 0, stream, a)
                          : launch_early(paged_merge_kernel<__half>, grid, 256, 0, stream, a);
}

}  // extern "C"
