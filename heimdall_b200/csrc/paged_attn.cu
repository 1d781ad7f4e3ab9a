// Attention of the last t tokens of each sequence over its 8-bit pages.
//
//   o = sum_j p_j sv_j c^v_j,  p = softmax_j(scale sk_j q . c^k_j)  over the positions j <= the token's own that have a page,
//   with the e4m3 codes c and the scales sk, sv of each (page, KV head).
//
// A decode step reads every code once and computes little with it, so what bounds it is HBM: 512 bytes per (token, KV
// head).  Turning the codes into 16-bit operands in registers would cost two conversions and a shared-memory round trip
// per byte pair; instead the codes go from HBM by TMA into shared memory and from there, untouched, into the 5th-gen
// tensor core (kind::f8f6f4).  The other operand of each product, which is small, is split into three e4m3 parts of 4
// significant bits each (x = (x0 + x1 / 16 + x2 / 256) / 2^k, every part scaled into the code's upper range), each part a column of
// its own:
//   S^T[token, part x row] = K Q^T    M = 128 tokens, N = 3 RP, K = 256 dims   (a query component is exact in three parts while it is not
//                                     far below its row's largest, and off by at most 2^-25 of the largest: the parts end there)
//   O^T[dim, part x row]   = V^T P^T  M = 2 x 128 dims, N = 3 RP, K = 128 tokens (P is rounded to fp16's 11 bits, which the parts
//                                     hold: off by at most 2^-11 of itself, or 2^-26 of the tile's largest weight)
// with a row = (token of the call, query head of the KV head's group), RP rows at a time.  P is taken relative to its own
// tile's maximum, so that a tile of small weights keeps its bits, and the tile's O^T leaves TMEM for fp32 registers that
// carry the running maximum: nothing is rescaled in TMEM.  V's scales go into P (as their ratio to the tile's largest).
//
// Work: the tiles of 128 tokens of all (sequence, token chunk, KV head) segments in one line, cut into equal runs, one per CTA
// (one CTA per SM), whatever the lengths; a segment's start counts as one or two tiles, as its queries and its output take about
// that long.  A segment inside one run is finished there; of a cut one each CTA writes its partial (at most two per CTA), and
// paged_combine_kernel merges them in order, so results do not depend on timing.
// Warps: 0 and 2 TMA of the codes (K and V, each its own ring of 32 KB units), 0 also the tiles' scales; 1 the products S; 3 the
// products O; then two (24 rows: three) warpgroups of softmax (thread = token and every second, or third, row), which at the start of
// a segment also make the next one's Q parts (loaded a segment before; a warp of its own for them took 9000 cycles for 24 rows);
// the last two warpgroups the accumulators (thread = dim) and the output.
// A tile has 2900 cycles at HBM's rate, so what counts is each role's chain of instructions.  With one softmax warp per scheduler a
// tile took 6100 cycles; the rows are therefore dealt to several warpgroups, and what is the same for all tokens (a row's maximum
// and its two factors) is computed by one lane per row and passed by shuffles.  The products are small, so issuing them is what
// costs: one thread of a diverged warp took 4400 cycles per tile for both (every descriptor on its way through vector registers); two
// warps that stay converged and elect the issuing lane do not bound it.  The roles together have to stay in the instruction
// cache: waits and loops are written for few instructions (106 KB of code took a third longer than 72 KB).
// Measured (24 query heads, 4 KV heads, pages of 64): 64 sequences of 16384 tokens 326 us, 6.6 TB/s (the measured rate of a copy, which
// also writes, is 6.5; 16 of 131072 take 622 us repeated, 676 to 734 with other passes in between); 64 of 1 to 16384 tokens 48 us
// (floor 36); one of 777 tokens 9.6 us.  24 rows (four tokens): 3550 cycles a tile, bound by the softmax warps' way through a tile: 32
// sequences of 16384 tokens 225 us (floor 166), with pages of 16 tokens 247 (eight copies per tile and half).  There 80 registers per
// thread are all there are, and what does not fit costs: 244 us with 28 bytes spilled.
// (Taking a tile's scores before the weights of the one before, so that nobody waits for the maxima, made it 267 us.)
#include "bifrost_b200.h"
#include "capi_internal.h"
#include "common.cuh"
#include "launch_early.h"
#include "paged_kv.h"
#include "tmap.h"

namespace bfb {

constexpr int kPA_Tile = 128;                        // tokens per tile
constexpr int kPA_Unit = kPA_Tile * kPG_D;           // bytes of one K or V tile
constexpr int kPA_MaxCtas = 160;
constexpr int kPA_MaxRows = 24;
constexpr int kPA_Part = kPG_D + 4;                  // floats of a row's partial: accumulator, maximum, sum, two to keep it aligned

struct PagedAttnArgs {
  PagePool p;
  const void* q;
  long long q_sb, q_st, q_sh;
  const int32_t* slots;
  int B, t, H, R;
  int tc, nqc;          // tokens per chunk, chunks
  int cap;              // tokens that the table has room for
  int page_log;         // log2 of the page's tokens
  unsigned by_r;        // 2^16 / R, rounded up: r / R = r * by_r >> 16 for rows r < 24
  float c2;             // scale * log2(e)
  void* o;
  float* lse;
  int4* desc;           // [ctas] (first CTA of the cut segment that ends here or -1, b, chunk, KV head)
  float* part;          // [ctas][2][RP][kPA_Part]
  unsigned int* err;
};

template <int RP>
struct PagedCfg {
  static constexpr int NP = (3 * RP + 15) / 16 * 16;       // MMA N: three parts of RP rows, padded to 16
  static constexpr int Groups = RP == 24 ? 3 : 2;          // softmax warpgroups: row r is of group r % Groups
  static constexpr int Threads = (4 + 4 * Groups + 8) * 32;
  static constexpr int KUnits = 3, VUnits = RP == 8 ? 3 : 2;   // ring units that fit beside Q and P
  static constexpr int Units = KUnits + VUnits;
  // what a segment's start counts, in tiles.  64 sequences of 1 to 16384 tokens, 8 rows: 60, 48 and 51 us with 0, 1 and 2, 64 of 700: 56 to
  // 57 with each; 32 of 4 to 32768 tokens, 24 rows: 95, 88 and 90 us with 1, 2 and 3, 64 of 100 to 3000, 16 rows: 59, 57 and 58
  static constexpr int Start = RP == 8 ? 1 : 2;
  static constexpr int TmemCols = 6 * NP <= 256 ? 256 : 512;   // S[2], O[2][2 halves]
  static constexpr int QBytes = NP * kPG_D, PBytes = NP * kPA_Tile;
  static constexpr int Smem = Units * kPA_Unit + 2 * QBytes + 2 * PBytes + 5120 + 1024;
};

// slot (-1: none) and visible length of sequence b
__device__ __forceinline__ int2 paged_seq(const PagedAttnArgs& a, int b) {
  const int slot = a.slots ? a.slots[b] : b;
  const bool ok = slot >= 0 && slot < a.p.slots;
  return make_int2(ok ? slot : -1, ok ? max(0, min(a.p.lens[slot], a.cap)) : 0);
}
// tiles of a sequence: at least one, so that a segment that sees nothing has a CTA that writes its zeros
__device__ __forceinline__ int paged_tiles(int len) { return max(1, (len + kPA_Tile - 1) / kPA_Tile); }

// a row's token of the chunk and its query head of the group
__device__ __forceinline__ int2 paged_row(const PagedAttnArgs& a, int r) {
  const int i = (int)(r * a.by_r >> 16);
  return make_int2(i, r - i * a.R);
}

// a CTA's walk over its run of tiles; the run's first kPA_Seqs sequences are in shared memory, a load from L2 on every warp's
// way to the next sequence would cost as much as half a tile
constexpr int kPA_Seqs = 192;
struct PagedWalk {
  int b, c, g, tile, ntiles, len, slot;
  int b0;
  const int2* seqs;      // (slot, length) of sequences b0, b0 + 1, ...
  __device__ __forceinline__ void enter(const PagedAttnArgs& a) {
    const int2 x = b - b0 < kPA_Seqs ? seqs[b - b0] : paged_seq(a, b);
    slot = x.x;
    len = x.y;
    ntiles = paged_tiles(len);
  }
  __device__ __forceinline__ void next(const PagedAttnArgs& a) {
    if (++tile < ntiles) return;
    tile = 0;
    if (++g < a.p.heads) return;
    g = 0;
    if (++c < a.nqc) return;
    c = 0;
    if (++b < a.B) enter(a);
  }
  // on to the next segment; returns this one's tiles from `tile` on
  __device__ __forceinline__ int skip(const PagedAttnArgs& a) {
    const int n = ntiles - tile;
    tile = ntiles - 1;
    next(a);
    return n;
  }
};

// x = (x0 + x1 / 16 + x2 / 256) with e4m3 parts, for |x| <= 256; two values at a time.  x is first rounded to fp16, whose 11
// bits the parts hold exactly; the remainders are exact in fp16.
__device__ __forceinline__ uint16_t to_e4m3x2(uint32_t h2) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(h2));
  return r;
}
__device__ __forceinline__ void split3(float a, float b, uint16_t (&part)[3]) {
  const __half2 m16 = __floats2half2_rn(-16.f, -16.f), p16 = __floats2half2_rn(16.f, 16.f);
  __half2 x = __floats2half2_rn(a, b);
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    part[i] = to_e4m3x2(*reinterpret_cast<uint32_t*>(&x));
    if (i < 2) {
      uint32_t f;
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(f) : "h"(part[i]));
      x = __hfma2(*reinterpret_cast<__half2*>(&f), m16, __hmul2(x, p16));   // 16 (x - part)
    }
  }
}
// the RP rows lie group by group of the softmax warps: row r in column row_col(r) of each part
template <int RP>
__device__ __forceinline__ constexpr int row_col(int r) { return r % PagedCfg<RP>::Groups * (RP / PagedCfg<RP>::Groups) + r / PagedCfg<RP>::Groups; }
template <int RP>
__device__ __forceinline__ constexpr int col_row(int c) {
  constexpr int n = RP / PagedCfg<RP>::Groups;
  return c % n * PagedCfg<RP>::Groups + c / n;
}

template <typename T, int RP>
__global__ void __launch_bounds__(PagedCfg<RP>::Threads, 1)
    paged_attn_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, PagedAttnArgs a) {
  using C = PagedCfg<RP>;
  constexpr int NP = C::NP, NU = C::Units, NK = C::KUnits, NV = C::VUnits, SG = C::Groups;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem;
  uint8_t* sQ = ring + NU * kPA_Unit;          // [2][2 atoms][NP][128]
  uint8_t* sP = sQ + 2 * C::QBytes;            // [2][NP][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sP + 2 * C::PBytes);
  uint64_t *full = bars, *empty = bars + 6, *s_full = bars + 12, *s_free = bars + 14, *p_full = bars + 16, *o_full = bars + 18,
           *o_free = bars + 20, *q_full = bars + 22, *q_free = bars + 24, *sc_full = bars + 26, *sc_free = bars + 30, *red = bars + 34,
           *seg_full = bars + 37, *seg_free = bars + 39;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 41);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 42);
  int* s_sum = reinterpret_cast<int*>(bars + 43);                   // [24] per-warp totals of the unit count
  int* s_start = reinterpret_cast<int*>(bars + 56);                 // b, segment of it, tile of that
  float* s_qs = reinterpret_cast<float*>(bars + 66);                // [2][RP] scale of the Q rows
  float* s_fac = s_qs + 2 * kPA_MaxRows;                            // [2][RP][2] factors of the tile's O^T and the accumulators
  float* s_red = s_fac + 4 * kPA_MaxRows;                           // [2][4][RP] the warps' maxima
  float* s_seg = s_red + 8 * kPA_MaxRows;                           // [2][5][RP] a segment's sums per warp, its maximum
  float* s_sc = s_seg + 10 * kPA_MaxRows;                           // [4][20] scales of a tile's pages: 8 K, 8 V ratios, V's largest, mask
  int2* s_seqs = reinterpret_cast<int2*>(s_sc + 80);                 // [kPA_Seqs]
  static_assert(66 * 8 + (2 + 4 + 8 + 10) * kPA_MaxRows * 4 + 80 * 4 + kPA_Seqs * 8 <= 5120, "barriers and exchanges");

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < NU; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(s_free + i, 4 * SG);
      mbar_init(p_full + i, 4 * SG);
      mbar_init(o_full + i, 1);
      mbar_init(o_free + i, 8);
      mbar_init(q_full + i, 4 * SG);
      mbar_init(q_free + i, 4 * SG + 1);
      mbar_init(seg_full + i, 4 * SG);
      mbar_init(seg_free + i, 8);
    }
    for (int i = 0; i < SG; ++i) mbar_init(red + i, 4);
    for (int i = 0; i < 4; ++i) {
      mbar_init(sc_full + i, 1);
      mbar_init(sc_free + i, 4 * SG);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  let_next_start();
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::TmemCols);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) tma_prefetch(&kmap);
  if (warp == 2 && lane == 0) tma_prefetch(&vmap);
  wait_for_stream();
  // this CTA's run: every segment is Start units and one for each of its tiles.  The sequences' units are summed over the block,
  // thread i holding `per` consecutive sequences (the caller has made sure that 32 bits hold the sum)
  const int per = (a.B + C::Threads - 1) / C::Threads;
  const int segs = a.nqc * a.p.heads;
  const bool known = a.B <= kPA_Seqs;          // all sequences fit into s_seqs
  int mine = 0;
  for (int i = 0; i < per; ++i) {
    const int b = tid * per + i;
    if (b < a.B) {
      const int2 q = paged_seq(a, b);
      mine += (paged_tiles(q.y) + C::Start) * segs;
      if (known) s_seqs[b] = q;
    }
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) s_sum[warp] = incl;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  int total = lane < C::Threads / 32 ? s_sum[lane] : 0, before = lane < warp ? total : 0;
  total = (int)__reduce_add_sync(0xffffffffu, (unsigned)total);
  before = (int)__reduce_add_sync(0xffffffffu, (unsigned)before) + incl - mine;
  // with fewer units than CTAs the first `total` CTAs take one each; the first `more` runs are one unit longer than the others
  const int ctas = min(total, (int)gridDim.x), each = total / ctas, more = total - each * ctas;
  const int u0 = min((int)blockIdx.x, ctas) * each + min((int)blockIdx.x, more);
  const int u1 = u0 + ((int)blockIdx.x < ctas ? each + ((int)blockIdx.x < more ? 1 : 0) : 0);
  // the sequence, segment and tile of the first unit u0, and how many of the run's units are tiles
  if (u0 < u1 && before <= u0 && u0 < before + mine) {
    int at = before;
    for (int b = tid * per;; ++b) {
      const int n = paged_tiles(known ? s_seqs[b].y : paged_seq(a, b).y) + C::Start;
      if (u0 < at + n * segs) {
        s_start[0] = b;
        s_start[1] = (u0 - at) / n;
        s_start[2] = (u0 - at) - s_start[1] * n;
        break;
      }
      at += n * segs;
    }
  }
  __syncthreads();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  PagedWalk w{};
  int count = 0;                  // tiles of the run
  if (!known) {
    for (int i = tid; u0 < u1 && i < kPA_Seqs && s_start[0] + i < a.B; i += C::Threads) s_seqs[i] = paged_seq(a, s_start[0] + i);
    __syncthreads();
  }
  if (u0 < u1) {
    w.seqs = s_seqs;
    w.b = s_start[0];
    w.b0 = known ? 0 : w.b;
    w.c = s_start[1] / a.p.heads;
    w.g = s_start[1] % a.p.heads;
    w.enter(a);
    w.tile = max(s_start[2] - C::Start, 0);
    // walk the run's segments: the units of each that are tiles
    PagedWalk x = w;
    for (int u = u0 - s_start[2]; u < u1;) {
      count += max(min(u + C::Start + x.ntiles, u1) - max(u + C::Start, u0), 0);
      u += x.ntiles + C::Start;
      x.tile = x.ntiles - 1;
      x.next(a);
    }
  }
  count = __shfl_sync(0xffffffffu, count, 0);
  const int L = a.p.page, ppt = kPA_Tile >> a.page_log;       // pages per tile
  // the page of this tile's page number `i`, -1 where there is none
  auto page_of = [&](const PagedWalk& x, int i) -> int {
    const int j = x.tile * ppt + i;
    if (i >= ppt || (long long)j * L >= x.len) return -1;
    const int page = a.p.table[(size_t)x.slot * a.p.width + j];
    return page >= 0 && page < a.p.pages ? page : -1;
  };

  if (warp == 0 || warp == 2) {
    // ------------------------------------------------------------------ codes: K (warp 0), V (warp 2)
    const bool is_v = warp == 2;
    const void* map = is_v ? &vmap : &kmap;
    // each ring has one producer, which waits for its slots' rounds one by one (with K and V in one ring of an odd number of slots, a
    // producer could meet a slot two rounds behind and take the parity of the round before for its own)
    const int units = is_v ? NV : NK, base = is_v ? NK : 0;
    int u = 0, uphase = 1;                // the unit's slot of the ring; the parity of the round before
    bool ok = true;
    // each lane a page of the tile: page numbers are loaded two tiles ahead, scales one, so that no load is waited for here
    int now = -1, next = -1, g = 0, g_next = 0, ahead = 0;
    float ks_next = 0.f, vs_next = 0.f;
    auto step = [&]() {                   // the walk's next tile into (next, g_next)
      next = -1;
      if (ahead < count) {
        g_next = w.g;
        next = page_of(w, lane);
        w.next(a);
      }
      ++ahead;
    };
    auto scales = [&]() {
      ks_next = vs_next = 0.f;
      if (now >= 0 && !is_v) {
        ks_next = a.p.ks[(size_t)now * a.p.heads + g];
        vs_next = a.p.vs[(size_t)now * a.p.heads + g];
      }
    };
    step();
    now = next;
    g = g_next;
    step();
    scales();
#pragma unroll 1
    for (int j = 0; j < count; ++j) {
      const float ks = ks_next, vs = vs_next;
      const int page = now, head = g;
      now = next;
      g = g_next;
      step();
      scales();
      const unsigned have = __ballot_sync(0xffffffffu, page >= 0);
      const int first_row = page >= 0 ? (page * a.p.heads + head) * L : 0;
      if (j >= units && !(ok = mbar_wait_warp_small(empty + base + u, uphase, abort_flag, 0x60))) break;
      if (lane == 0) {
        if (have) mbar_expect_tx(full + base + u, (uint32_t)__popc(have) * L * kPG_D); else mbar_arrive(full + base + u);
      }
      __syncwarp();
      // page by page with operands that all lanes agree on: eight lanes issuing their own pages took 150 cycles per copy
#pragma unroll 1
      for (int i = 0; i < ppt; ++i) {
        const int row = __shfl_sync(0xffffffffu, first_row, i);
        if (((have >> i) & 1u) && elect_one()) {
          uint8_t* dst = ring + (base + u) * kPA_Unit + i * L * 128;
          tma_load_2d(dst, map, full + base + u, 0, row);
          tma_load_2d(dst + kPA_Tile * 128, map, full + base + u, 128, row);
        }
        __syncwarp();
      }
      if (++u == units) {
        u = 0;
        uphase ^= 1;
      }
      if (is_v) continue;
      // the tile's scales, their loads as old as its TMA's
      const int s = j & 3;
      const float top = warp_max(vs);
      if (j >= 4 && !(ok = mbar_wait_warp_small(sc_free + s, ((j >> 2) - 1) & 1, abort_flag, 0x69))) break;
      if (lane < 8) {
        s_sc[s * 20 + lane] = ks;
        s_sc[s * 20 + 8 + lane] = top > 0.f ? vs / top : 0.f;      // powers of two: exact
      }
      if (lane == 0) {
        s_sc[s * 20 + 16] = top;
        s_sc[s * 20 + 17] = __uint_as_float(have);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(sc_full + s);
    }
    // every load issued has landed before the CTA may exit: the products have read it, or, with a wait that gave up, report_abort
    // gives it time
  } else if (warp == 1) {
    // ------------------------------------------------------------------ S = K Q^T
    constexpr uint32_t id_s = idesc_e4m3(kPA_Tile, NP);
    const uint64_t dk0 = sdesc_sw128(smem_u32(ring)), dq0 = sdesc_sw128(smem_u32(sQ));
    int seg = 0, u = 0, uphase = 0;
    bool first = true;
#pragma unroll 1
    for (int j = 0; j < count; ++j) {
      const int s = j & 1;
      if (first && !mbar_wait_warp_small(q_full + (seg & 1), (seg >> 1) & 1, abort_flag, 0x65)) break;
      if (!mbar_wait_warp_small(full + u, uphase, abort_flag, 0x66)) break;
      if (j >= 2 && !mbar_wait_warp_small(s_free + s, ((j >> 1) - 1) & 1, abort_flag, 0x67)) break;
      // the accumulators have taken over tile j - 2, so its P, its factors and its O may be written over once S of this tile is there:
      // waited for here, where it costs nothing, and not again on the way of the softmax warps and of O
      if (j >= 2 && !mbar_wait_warp_small(o_free + s, ((j >> 1) - 1) & 1, abort_flag, 0x64)) break;
      tc_fence_after();
      first = w.tile + 1 == w.ntiles;
      const bool end = first || j + 1 == count;
      if (elect_one()) {
        const uint64_t dk = dk0 + (uint32_t)(u * (kPA_Unit >> 4)), dq = dq0 + (uint32_t)((seg & 1) * (C::QBytes >> 4));
#pragma unroll
        for (int ks = 0; ks < kPG_D / 32; ++ks)
          umma_f8_ss(tmem + s * NP, dk + ((ks >> 2) * (kPA_Tile * 128) + (ks & 3) * 32) / 16,
                     dq + ((ks >> 2) * (NP * 128) + (ks & 3) * 32) / 16, id_s, ks > 0);
        umma_commit(s_full + s);
        umma_commit(empty + u);
        if (end) umma_commit(q_free + (seg & 1));
      }
      __syncwarp();
      seg += end;
      w.next(a);
      if (++u == NK) {
        u = 0;
        uphase ^= 1;
      }
    }
  } else if (warp == 3) {
    // ------------------------------------------------------------------ O = V^T P^T
    constexpr uint32_t id_o = idesc_e4m3(128, NP) | kIdescAMn;
    const uint64_t dv0 = sdesc_sw128_mn(smem_u32(ring), 16384), dp0 = sdesc_sw128(smem_u32(sP));
    int u = 0, uphase = 0;
#pragma unroll 1
    for (int j = 0; j < count; ++j) {
      const int s = j & 1;
      if (!mbar_wait_warp_small(full + NK + u, uphase, abort_flag, 0x63)) break;
      if (!mbar_wait_warp_small(p_full + s, (j >> 1) & 1, abort_flag, 0x62)) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t dv = dv0 + (uint32_t)((NK + u) * (kPA_Unit >> 4)), dp = dp0 + (uint32_t)(s * (C::PBytes >> 4));
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            umma_f8_ss(tmem + 2 * NP + (2 * s + half) * NP, dv + (half * 16384 + ks * 4096) / 16, dp + ks * 32 / 16, id_o, ks > 0);
        umma_commit(o_full + s);
        umma_commit(empty + NK + u);
      }
      __syncwarp();
      if (++u == NV) {
        u = 0;
        uphase ^= 1;
      }
    }
  } else if (warp < 4 + 4 * SG) {
    // ------------------------------------------------------------------ softmax: thread = token of the tile, rows SG i + hh
    constexpr int RH = RP / SG;
    const int wq = warp & 3, hh = (warp - 4) >> 2, tok = wq * 32 + lane;
    const uint32_t trow = tmem + ((uint32_t)(wq * 32) << 16) + hh * RH;
    float l[RH];
    int rows = 0, first_pos = 0;         // of the chunk; the position of its first token
    float m_run = -INFINITY;             // of row SG lane + hh, in lanes < RH
    bool ok = true, first = true;
    int seg = 0;
    // the queries: warp w of the 4 SG takes rows w, w + 4 SG, ..., lane l dims 8 l .. 8 l + 7
    constexpr int QW = 4 * SG;
    uint4 qraw[RP / QW];
    auto q_load = [&](const PagedWalk& nx) {
      const int i0 = nx.c * a.tc, nx_rows = min(a.tc, a.t - i0) * a.R;
#pragma unroll
      for (int i = 0; i < RP / QW; ++i) {
        const int r = warp - 4 + QW * i;
        const int2 ih = paged_row(a, r);
        if (r < nx_rows)
          qraw[i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + nx.b * a.q_sb + (long long)(i0 + ih.x) * a.q_st +
                                                         (long long)(nx.g * a.R + ih.y) * a.q_sh + 8 * lane));
      }
    };
    // the queries in qraw, of segment nx, which begins with tile `at` of the run; then nx and qraw are the next segment's.  Rows from
    // nx_rows on stay as they are, nothing reads their scores
    auto q_store = [&](PagedWalk& nx, int& at, int buf) {
      const int nx_rows = min(a.tc, a.t - nx.c * a.tc) * a.R;
      uint8_t* dst = sQ + buf * C::QBytes + (lane >> 4) * (NP * 128) + (lane & 1) * 8;
#pragma unroll
      for (int i = 0; i < RP / QW; ++i) {
        const int r = warp - 4 + QW * i;
        if (r >= nx_rows) break;
        const uint32_t u[4] = {qraw[i].x, qraw[i].y, qraw[i].z, qraw[i].w};
        // the largest value of the row, as 16-bit patterns without their sign
        const uint32_t m2 = __vmaxu2(__vmaxu2(u[0] & 0x7fff7fffu, u[1] & 0x7fff7fffu), __vmaxu2(u[2] & 0x7fff7fffu, u[3] & 0x7fff7fffu));
        const uint32_t m = __reduce_max_sync(0xffffffffu, max(m2 & 0xffffu, m2 >> 16));
        const uint16_t m16 = (uint16_t)m;
        const float mf = (float)*reinterpret_cast<const T*>(&m16);
        const bool fin = mf < INFINITY;          // false for NaN too
        // to [128, 256): x * 2^k, k = 7 - exponent
        const int ex = mf > 0.f ? max((int)(__float_as_uint(mf) >> 23), 16) : 127;
        const float up = fin ? __uint_as_float((uint32_t)(254 + 7 - ex) << 23) : 0.f;
        uint16_t c[4][3];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const T* e = reinterpret_cast<const T*>(&u[q]);
          split3(fin ? (float)e[0] * up : 0.f, fin ? (float)e[1] * up : 0.f, c[q]);
        }
#pragma unroll
        for (int part = 0; part < 3; ++part) {
          const int n = part * RP + row_col<RP>(r);
          *reinterpret_cast<uint2*>(dst + n * 128 + ((((lane & 15) >> 1) ^ (n & 7)) << 4)) =
              make_uint2(c[0][part] | ((uint32_t)c[1][part] << 16), c[2][part] | ((uint32_t)c[3][part] << 16));
        }
        // a row with a value that is not finite has no finite scores
        if (lane == 0) s_qs[buf * RP + row_col<RP>(r)] = fin ? __uint_as_float((uint32_t)(ex - 7) << 23) * a.c2 : NAN;
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full + buf);
      at += nx.skip(a);
      if (at < count) q_load(nx);
    };
    if (count > 0) q_load(w);
#pragma unroll 1
    for (int j = 0; j < count; ++j) {
      const int s = j & 1;
      if (first) {
        // store the next segment's queries (and, at the run's start, this one's before them)
        PagedWalk nx = w;
        int at = j;
        if (j) at += nx.skip(a);
#pragma unroll 1
        for (int k = j ? 1 : 0; k < 2 && ok; ++k) {
          if (k) {
            if (!(ok = mbar_wait_warp_small(q_full + (seg & 1), (seg >> 1) & 1, abort_flag, 0x6a))) break;
            rows = min(a.tc, a.t - w.c * a.tc) * a.R;
            first_pos = w.len - a.t + w.c * a.tc;
            m_run = -INFINITY;
#pragma unroll
            for (int i = 0; i < RH; ++i) l[i] = 0.f;
          }
          if (at < count) {
            if (k && seg >= 1 && !(ok = mbar_wait_warp_small(q_free + ((seg + 1) & 1), (((seg + 1) >> 1) - 1) & 1, abort_flag, 0x68))) break;
            q_store(nx, at, (seg + k) & 1);
          }
        }
        if (!ok) break;
      }
      const bool last = w.tile + 1 == w.ntiles, end = last || j + 1 == count;
      // the scores, four rows at a time (more registers there are not for 24 rows), the first of them on their way while the mask is made
      if (!(ok = mbar_wait_warp_small(s_full + s, (j >> 1) & 1, abort_flag, 0x6c))) break;
      tc_fence_after();
      uint32_t raw[12];
      auto load4 = [&](int c) {
#pragma unroll
        for (int part = 0; part < 3; ++part) tmem_ld4(trow + s * NP + part * RP + c, raw + part * 4);
      };
      load4(0);
      if (!(ok = mbar_wait_warp_small(sc_full + (j & 3), (j >> 2) & 1, abort_flag, 0x6b))) break;
      const float* sc = s_sc + (j & 3) * 20;
      const int pi = tok >> a.page_log;
      const float ks = sc[pi], vr = sc[8 + pi] * 256.f, top = sc[16];
      const bool there = (__float_as_uint(sc[17]) >> pi) & 1u;
      const int pos = w.tile * kPA_Tile + tok;
      const bool valid = there && pos < w.len;
      // bit r: row r's token is at or behind this position (the first of them is that many tokens into the chunk)
      const unsigned later = (unsigned)min(max(pos - first_pos, 0) * a.R, 31);
      const unsigned sees = valid ? (((1u << rows) - 1u) >> later << later) >> hh : 0u;
      float x[RH], mine = -INFINITY;
      const float* qs = s_qs + (seg & 1) * RP + hh * RH;
      float* rd = s_red + s * 4 * RP + hh * RH;
#pragma unroll
      for (int c = 0; c < RH; c += 4) {
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float d = __uint_as_float(raw[i]) + (__uint_as_float(raw[4 + i]) + __uint_as_float(raw[8 + i]) * 0.0625f) * 0.0625f;
          x[c + i] = (sees >> (SG * (c + i))) & 1u ? d * (ks * qs[c + i]) : -INFINITY;
        }
        if (c + 4 < RH) load4(c + 4);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(s_free + s);
        mbar_arrive(sc_free + (j & 3));
        if (end) mbar_arrive(q_free + (seg & 1));
      }
#pragma unroll
      for (int i = 0; i < RH; ++i) {
        float mx;
        asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(mx) : "f"(x[i]));
        if (lane == i) mine = mx;
      }
      if (lane < RH) rd[wq * RP + lane] = mine;
      __syncwarp();
      if (lane == 0) mbar_arrive(red + hh);
      if (!(ok = mbar_wait_warp_small(red + hh, j & 1, abort_flag, 0x6d))) break;
      // lane i: row SG i + hh's maximum of the tile, and the factors of what was before and of this tile
      float mt = -INFINITY;
      if (lane < RH) mt = fmaxf(fmaxf(rd[lane], rd[RP + lane]), fmaxf(rd[2 * RP + lane], rd[3 * RP + lane]));
      const float mn = fmaxf(m_run, mt);
      const float al = m_run == -INFINITY ? 0.f : ex2_approx(m_run - mn);
      const float f = mt == -INFINITY ? 0.f : ex2_approx(mt - mn);
      m_run = mn;
      mt = mt == -INFINITY ? 0.f : mt;
      if (wq == 0 && lane < RH)
        *reinterpret_cast<float2*>(s_fac + (s * RP + hh * RH + lane) * 2) = make_float2(al, f * top * (1.f / 256.f));
      uint8_t* pd = sP + s * C::PBytes;
#pragma unroll
      for (int i = 0; i < RH; i += 2) {
        float y[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // masked scores are -inf and give 0; a NaN stays one, whatever the others are
          const float p = ex2_approx(x[i + e] - __shfl_sync(0xffffffffu, mt, i + e));
          const float fi = __shfl_sync(0xffffffffu, f, i + e);
          l[i + e] = fmaf(l[i + e], __shfl_sync(0xffffffffu, al, i + e), p * fi);
          y[e] = p * vr;
        }
        uint16_t c[3];
        split3(y[0], y[1], c);
#pragma unroll
        for (int part = 0; part < 3; ++part) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int n7 = (part * RP + hh * RH + i + e) & 7, n = part * RP + hh * RH + i + e;
            pd[n * 128 + (tok ^ (n7 << 4))] = (uint8_t)(c[part] >> (8 * e));
          }
        }
      }
      if (__any_sync(0xffffffffu, !valid)) {
        // the values of tokens that are not there may be anything (a weight of 0 times NaN would be NaN): zeros
        const int u = NK + j % NV;
        if (!(ok = mbar_wait_warp_small(full + u, (j / NV) & 1, abort_flag, 0x6f))) break;
        if (!valid && hh < 2) {
          uint4* row = reinterpret_cast<uint4*>(ring + u * kPA_Unit + hh * (kPA_Tile * 128) + tok * 128);
#pragma unroll
          for (int i = 0; i < 8; ++i) row[(i + tok) & 7] = make_uint4(0u, 0u, 0u, 0u);     // a chunk per lane: rows are as long as all banks
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + s);
      if (end) {
        if (seg >= 2 && !(ok = mbar_wait_warp_small(seg_free + (seg & 1), ((seg >> 1) - 1) & 1, abort_flag, 0x70))) break;
        float* sg = s_seg + (seg & 1) * 5 * RP + hh * RH;
#pragma unroll
        for (int i = 0; i < RH; ++i) {
          const float sum = warp_sum(l[i]);
          if (lane == 0) sg[wq * RP + i] = sum;
        }
        if (wq == 0 && lane < RH) sg[4 * RP + lane] = m_run;
        __syncwarp();
        if (lane == 0) mbar_arrive(seg_full + (seg & 1));
        ++seg;
      }
      first = last;
      w.next(a);
    }
  } else {
    // ------------------------------------------------------------------ accumulators: thread = dim d of every row
    const int wq = warp & 3, half = (warp - 4 - 4 * SG) >> 2, d = half * 128 + wq * 32 + lane;
    const uint32_t trow = tmem + ((uint32_t)(wq * 32) << 16) + (2 + half) * NP;
    float acc[RP];
    bool ok = true, from_start = w.tile == 0;
    int seg = 0;
    int unit = count > 0 ? u0 + max(C::Start - s_start[2], 0) : 0;      // the tile's
    int4 desc = make_int4(-1, 0, 0, 0);
#pragma unroll
    for (int c = 0; c < RP; ++c) acc[c] = 0.f;
#pragma unroll 1
    for (int j = 0; j < count; ++j) {
      const int s = j & 1;
      if (!(ok = mbar_wait_warp_small(p_full + s, (j >> 1) & 1, abort_flag, 0x73))) break;   // the factors
      if (!(ok = mbar_wait_warp_small(o_full + s, (j >> 1) & 1, abort_flag, 0x71))) break;
      tc_fence_after();
      // eight rows at a time (all of RP = 24 at once would not fit the registers)
#pragma unroll
      for (int c0 = 0; c0 < RP; c0 += 8) {
        uint32_t raw[24];
#pragma unroll
        for (int part = 0; part < 3; ++part) tmem_ld8(trow + 2 * s * NP + part * RP + c0, raw + part * 8);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 fac = *reinterpret_cast<const float2*>(s_fac + (s * RP + c0 + i) * 2);
          const float x = __uint_as_float(raw[i]) + (__uint_as_float(raw[8 + i]) + __uint_as_float(raw[16 + i]) * 0.0625f) * 0.0625f;
          acc[c0 + i] = acc[c0 + i] * fac.x + x * fac.y;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free + s);
      const bool last = w.tile + 1 == w.ntiles;
      if (last || j + 1 == count) {
        if (!(ok = mbar_wait_warp_small(seg_full + (seg & 1), (seg >> 1) & 1, abort_flag, 0x72))) break;
        const float* sg = s_seg + (seg & 1) * 5 * RP;
        const int i0 = w.c * a.tc, rows = min(a.tc, a.t - i0) * a.R;
        const bool whole = from_start && last;
        float* part = a.part + ((size_t)blockIdx.x * 2 + (from_start ? 1 : 0)) * RP * kPA_Part;
        // lane c: row of column c, its sum, maximum and place in the output
        const int rc = col_row<RP>(min(lane, RP - 1));
        const int2 ih = paged_row(a, rc);
        const bool mine_row = lane < RP && rc < rows;
        float sum = 0.f, m = -INFINITY;
        if (mine_row) {
          sum = (sg[lane] + sg[RP + lane]) + (sg[2 * RP + lane] + sg[3 * RP + lane]);
          m = sg[4 * RP + lane];
        }
        const int row = ((w.b * a.t + i0 + ih.x) * a.H) + w.g * a.R + ih.y;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;       // nothing seen: zeros
        if (mine_row && warp == 4 + 4 * SG) {
          if (!whole)
            *reinterpret_cast<float2*>(part + rc * kPA_Part + kPG_D) = make_float2(m, sum);
          else if (a.lse)
            a.lse[((size_t)w.b * a.H + w.g * a.R + ih.y) * a.t + i0 + ih.x] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * kLn2;
        }
        // one copy of the code for all rows: the accumulators move up by one per row
        T* out = static_cast<T*>(a.o) + d;
#pragma unroll 1
        for (int c = 0; c < RP; ++c) {
          const float f = __shfl_sync(0xffffffffu, inv, c);
          const int to = __shfl_sync(0xffffffffu, row, c), r = __shfl_sync(0xffffffffu, rc, c);
          if (r < rows) {
            if (whole) out[(size_t)to * kPG_D] = (T)(acc[0] * f); else part[r * kPA_Part + d] = acc[0];
          }
#pragma unroll
          for (int k = 0; k + 1 < RP; ++k) acc[k] = acc[k + 1];
          acc[RP - 1] = 0.f;
        }
        // a cut segment that ends here: the CTA that holds its first tile
        if (last && !from_start) {
          const int t0 = unit - (w.ntiles - 1), longer = more * (each + 1);
          desc = make_int4(t0 < longer ? t0 / (each + 1) : more + (t0 - longer) / each, w.b, w.c, w.g);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(seg_free + (seg & 1));
        ++seg;
        from_start = true;
        unit += C::Start;
      }
      ++unit;
      w.next(a);
    }
    if (d == 0) a.desc[blockIdx.x] = ok ? desc : make_int4(-1, 0, 0, 0);
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0) report_abort(abort_flag, a.err);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TmemCols);
  }
}

// Block (x, y): a quarter of the rows and dims of the cut segment that ends in CTA x, if there is one: the partials of the CTAs
// first .. x, added in order, four dims per thread.  Up to eight partials are loaded at once; more are dealt to the block's eight warps,
// whose results are added in order.  (One block per row and 64 dims took 12 us for 8 rows and 32 us for 24, most of it block starts.)
template <typename T, int RP>
__global__ void __launch_bounds__(256) paged_combine_kernel(PagedAttnArgs a) {
  __shared__ float4 s_acc[8][32];
  __shared__ float2 s_ml[8][32];
  let_next_start();
  wait_for_stream();
  const int x = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int4 desc = a.desc[x];
  if (desc.x < 0) return;
  const int i0 = desc.z * a.tc, items = min(a.tc, a.t - i0) * a.R * (kPG_D / 4);
  const int n = x - desc.x + 1, lo = (int)((long long)items * blockIdx.y / gridDim.y), hi = (int)((long long)items * (blockIdx.y + 1) / gridDim.y);
  const bool few = n <= 8;
  const int each = few ? n : (n + 7) / 8, c_lo = few ? 0 : min(warp * each, n), c_hi = few ? n : min(c_lo + each, n);
  for (int it0 = lo; it0 < hi; it0 += few ? 256 : 32) {
    const int it = it0 + (few ? tid : lane), r = min(it, hi - 1) / (kPG_D / 4), d = (min(it, hi - 1) % (kPG_D / 4)) * 4;
    float m = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    // a partial without a maximum holds zeros, or NaN to be passed on
    auto add = [&](float mv, float lv, const float4& v) {
      const float mn = fmaxf(m, mv);
      const float al = m == -INFINITY ? 1.f : ex2_approx(m - mn), f = mv == -INFINITY ? 1.f : ex2_approx(mv - mn);
      acc.x = acc.x * al + v.x * f;
      acc.y = acc.y * al + v.y * f;
      acc.z = acc.z * al + v.z * f;
      acc.w = acc.w * al + v.w * f;
      sum = sum * al + lv * f;
      m = mn;
    };
    for (int c0 = c_lo; c0 < c_hi; c0 += 8) {
      float4 v[8];
      float2 ml[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = desc.x + min(c0 + i, c_hi - 1);
        const float* p = a.part + (((size_t)c * 2 + (c == desc.x ? 1 : 0)) * RP + r) * kPA_Part;
        v[i] = *reinterpret_cast<const float4*>(p + d);
        ml[i] = *reinterpret_cast<const float2*>(p + kPG_D);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c0 + i < c_hi) add(ml[i].x, ml[i].y, v[i]);
    }
    if (!few) {
      __syncthreads();
      s_acc[warp][lane] = acc;
      s_ml[warp][lane] = make_float2(m, sum);
      __syncthreads();
      if (warp == 0) {
#pragma unroll
        for (int k = 1; k < 8; ++k) add(s_ml[k][lane].x, s_ml[k][lane].y, s_acc[k][lane]);
      }
    }
    if (it < hi && (few || warp == 0)) {
      const int2 ih = paged_row(a, r);
      const int i = i0 + ih.x, h = desc.w * a.R + ih.y;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      T o[4] = {(T)(acc.x * inv), (T)(acc.y * inv), (T)(acc.z * inv), (T)(acc.w * inv)};
      *reinterpret_cast<uint2*>(static_cast<T*>(a.o) + (((size_t)desc.y * a.t + i) * a.H + h) * kPG_D + d) = *reinterpret_cast<uint2*>(o);
      if (a.lse && d == 0) a.lse[((size_t)desc.y * a.H + h) * a.t + i] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * kLn2;
    }
  }
}

// rows at a time for t tokens of R query heads: as many whole tokens as 24 rows hold, in equal chunks
static void paged_chunks(int t, int R, int* tc, int* nqc, int* rp) {
  const int most = t < kPA_MaxRows / R ? t : kPA_MaxRows / R;
  *nqc = (t + most - 1) / most;
  *tc = (t + *nqc - 1) / *nqc;
  *rp = (*tc * R + 7) / 8 * 8;
}

template <typename T, int RP>
static int launch_paged(const CUtensorMap& kmap, const CUtensorMap& vmap, const PagedAttnArgs& a, int ctas, cudaStream_t stream) {
  int rc = ensure_smem_attr((const void*)paged_attn_kernel<T, RP>, PagedCfg<RP>::Smem);
  if (rc) return rc;
  rc = launch_early(paged_attn_kernel<T, RP>, dim3(ctas), PagedCfg<RP>::Threads, PagedCfg<RP>::Smem, stream, kmap, vmap, a);
  return rc ? rc : launch_early(paged_combine_kernel<T, RP>, dim3(ctas, 4), 256, 0, stream, a);
}

}  // namespace bfb

using namespace bfb;

extern "C" {

size_t bf_paged_attend_workspace(int B, int t, int H, int G, int D) {
  if (B <= 0 || t <= 0 || H <= 0 || G <= 0 || H % G || H / G > kPA_MaxRows || D != kPG_D) return 0;
  int tc, nqc, rp;
  paged_chunks(t, H / G, &tc, &nqc, &rp);
  return (size_t)kPA_MaxCtas * (sizeof(int4) + (size_t)2 * rp * kPA_Part * 4);
}

int bf_paged_attend(const bf_page_pool* pool, int layer, const void* q, long long q_sb, long long q_st, long long q_sh,
                    const int32_t* slots, int B, int t, int H, int dtype, float scale, void* o, float* lse, void* ws,
                    size_t ws_bytes, bf_stream_t stream) {
  PagedAttnArgs a{};
  int rc = page_pool(pool, layer, &a.p);
  if (rc) return rc;
  if (B < 0 || t < 0 || H <= 0 || H % a.p.heads || (!slots && B > a.p.slots) || !(scale > 0.f) || scale > 3e38f)
    return BF_ERR_INVALID_ARGUMENT;
  if ((dtype != BF_BF16 && dtype != BF_F16) || H / a.p.heads > kPA_MaxRows) return BF_ERR_UNSUPPORTED;
  if (B == 0 || t == 0) return BF_OK;
  if (!q || !o) return BF_ERR_INVALID_ARGUMENT;
  if (!aligned16(q) || !aligned16(o) || ((q_sb | q_st | q_sh) & 7)) return BF_ERR_ALIGNMENT;
  if (!ws || ws_bytes < bf_paged_attend_workspace(B, t, H, a.p.heads, kPG_D)) return BF_ERR_WORKSPACE;
  if (!aligned16(ws)) return BF_ERR_ALIGNMENT;
  DeviceState st;
  if ((rc = device_state(&st))) return rc;
  a.q = q;
  a.q_sb = q_sb; a.q_st = q_st; a.q_sh = q_sh;
  a.slots = slots;
  a.B = B; a.t = t; a.H = H; a.R = H / a.p.heads;
  int rp;
  paged_chunks(t, a.R, &a.tc, &a.nqc, &rp);
  a.page_log = a.p.page == 16 ? 4 : a.p.page == 32 ? 5 : a.p.page == 64 ? 6 : 7;
  a.cap = (int)((long long)a.p.width * a.p.page < 0x7fffff00LL ? (long long)a.p.width * a.p.page : 0x7fffff00LL);
  a.by_r = (65536u + a.R - 1) / a.R;
  // the tiles of all segments are counted, and the output's rows numbered, in 32 bits
  if ((long long)B * a.nqc * a.p.heads * (a.cap / kPA_Tile + 4) > 0x7fffffffLL || (long long)B * t * H > 0x7fffffffLL)
    return BF_ERR_UNSUPPORTED;
  a.c2 = scale * kLog2e;
  a.o = o;
  a.lse = lse;
  a.desc = static_cast<int4*>(ws);
  a.part = reinterpret_cast<float*>(a.desc + kPA_MaxCtas);
  a.err = st.err;
  CUtensorMap kmap, vmap;
  const uint64_t dims[2] = {(uint64_t)kPG_D, (uint64_t)a.p.pages * a.p.heads * a.p.page}, strides[1] = {(uint64_t)kPG_D};
  const uint32_t box[2] = {128, (uint32_t)a.p.page};
  if ((rc = make_tmap(&kmap, a.p.k, kTmapU8, 2, dims, strides, box, true))) return rc;
  if ((rc = make_tmap(&vmap, a.p.v, kTmapU8, 2, dims, strides, box, true))) return rc;
  const int ctas = st.sm_count < kPA_MaxCtas ? st.sm_count : kPA_MaxCtas;
  if (dtype == BF_BF16) {
    if (rp == 8) return launch_paged<__nv_bfloat16, 8>(kmap, vmap, a, ctas, stream);
    if (rp == 16) return launch_paged<__nv_bfloat16, 16>(kmap, vmap, a, ctas, stream);
    return launch_paged<__nv_bfloat16, 24>(kmap, vmap, a, ctas, stream);
  }
  if (rp == 8) return launch_paged<__half, 8>(kmap, vmap, a, ctas, stream);
  if (rp == 16) return launch_paged<__half, 16>(kmap, vmap, a, ctas, stream);
  return launch_paged<__half, 24>(kmap, vmap, a, ctas, stream);
}

}  // extern "C"
