// The attention of cache_attn.cu for many query rows per KV head (chunks of prompts, long drafts under large groups):
// tiles of 128 rows on tcgen05. At these sizes a page's codes are used for 128 rows at once and arithmetic bounds it:
// 2 x 128 x 64 x D products, 128 x 64 exponentials (one SM makes 16 a clock: 512 clocks, as long as the products) and
// the conversion of 128 D codes per page.
//
// The page list, its cut into ranges and the joining of split units are those of cache_attn.cu, a CTA being a worker. Per
// page: K and V codes come in by bulk copies; two warps convert them to FP16 (exact) in the 128-byte-swizzled layout of the
// MMA's B operand (K [token][dim], V [dim][token]: both K-major as the cache keeps them); S = Q K^T with Q in tensor
// memory as the A operand; two threads per row turn 32 of its scores each into weights, which go back to tensor memory as
// the A operand of O' = P V; another thread per row adds O' to its sums in registers, scaled in FP32 by the page's exponent
// and by what the row's reference has moved. S, P and O' are double-buffered in tensor memory (64 + 2 x 64 + 2 x 32 + 2 x 128
// columns at D = 128), so the products of one page run under the exponentials of another.
//
// Measured (chunk of 2 x 512 tokens against 4096, 32 query and 8 KV heads, D = 128; with the join): 141 us, 458
// TFLOP/s; a page takes a CTA about 2000 clocks, whatever the rows of a tile: 32 sequences of 4000 with 5 drafts (20 rows) take
// 124 us, with 4 (16 rows, the other kernel) 73. At 128 registers the D = 128 form spills 138 bytes. What it is short of is instructions: some 3500 per page on four schedulers,
// and their fetching. With every loop written out the kernel was 183 KB of code, missed the instruction cache on 4 of 10
// fetches and took 349 us; loops over MMAs kept as loops and masks out of the way 220 and 176; FP32 operations two at a time
// and a row split over two threads (so that its scores stay in registers) 138. Tried and slower: four warps that convert
// (20 warps, 145 us), one for K and one for V (213), even and odd pages on different softmax warps (180).
//
// Roles: warp 0 looks pages up and copies, warp 1 issues MMAs, warps 2 and 3 convert, warps 4..11 softmax, warps 12..15
// sums and output. All waits are bounded.
#include "cache_attn.cuh"

namespace muse {

constexpr int TC_ROWS = 128;
constexpr int TC_THREADS = 512;
constexpr int TC_RAW = 8;              // ring slots of raw codes (K and V of a page are one each)
constexpr int TC_UNITS = 16;           // ring of unit records: no role is that many pages behind another
constexpr int TC_PAGES = 64;           // ring of page records
constexpr float TC_LIFT = 7.f, TC_UNLIFT = 0.0078125f;   // the lift of weights up to 2^8 (their reference lags behind): FP16 holds them down to 2^-31 of it
__host__ __device__ constexpr int tc_raw_bytes(int D) { return ATTN_PAGE * D; }
__host__ __device__ constexpr int tc_f16_bytes(int D) { return ATTN_PAGE * D * 2; }
__host__ __device__ constexpr int tc_smem_bytes(int D) { return 4 * tc_f16_bytes(D) + TC_RAW * tc_raw_bytes(D) + 1024; }
constexpr int TC_MIN_SMEM = 120 * 1024;   // one CTA per SM: it takes all of tensor memory

// The last page of a unit's share of the range, of the range; some row does not see some token; there is a page at all.
enum : int { PAGE_SEG_LAST = 1, PAGE_RANGE_LAST = 2, PAGE_EDGE = 4, PAGE_LIVE = 8 };
struct __align__(16) PageRec {
  int bits;      // exponents k | v << 8, PAGE_* << 16
  int p0;        // position of the page's first token
  int seen;      // first | last << 8: the page's tokens that some row of the tile sees
};
struct UnitRec {
  int first, row0, rows, pos;   // as in AttnEntry
  int h, whole;
  int slot;
};

__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// FP16 x FP16 -> FP32, both K-major.
__host__ __device__ constexpr uint32_t umma_idesc_f16(int M, int N) {
  return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
      "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void sts16(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// Two FP32 operations in one instruction: issue slots are what the softmax and the sums are short of.
__device__ __forceinline__ unsigned long long pack2(float lo, float hi) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(unsigned long long x, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x)); }
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Sixteen codes to FP16.
__device__ __forceinline__ void to_half16(const uint4& x, uint32_t (&o)[8]) {
  const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    o[2 * i] = fp8_to_half2(static_cast<uint16_t>(u[i] & 0xffffu));
    o[2 * i + 1] = fp8_to_half2(static_cast<uint16_t>(u[i] >> 16));
  }
}
// A page's V for one thread of the converters when some row does not see some token (or there is no page): of the thread's
// sixteen tokens those outside [lo, hi], which no row sees and which may hold anything, become zero, and so do NaN that only
// some rows see; those are noted, a bit per token, in `nan` (of dimensions 16 apart), and whether there are any comes back.
template <int D>
__device__ __forceinline__ int convert_v_edge(uint32_t src, uint32_t dst, bool live, int lo, int hi, unsigned short* nan) {
  uint32_t any = 0;
#pragma unroll 1
  for (int k = 0; k < D / 16; ++k) {
    const uint4 x = live ? lds16(src + k * 1024) : make_uint4(0u, 0u, 0u, 0u);
    uint32_t u[4] = {x.x, x.y, x.z, x.w}, noted = 0, o[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int from = max(lo - 4 * i, 0), to = min(hi - 4 * i, 3);
      u[i] &= from > 3 || to < from ? 0u : (0xffffffffu << (8 * from)) & (0xffffffffu >> (8 * (3 - to)));
      const uint32_t bad = ((u[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
      u[i] &= ~((bad >> 7) * 0xffu);
      noted |= ((bad >> 7 & 1u) | (bad >> 14 & 2u) | (bad >> 21 & 4u) | (bad >> 28 & 8u)) << (4 * i);
    }
    nan[k * 16 * 4] = static_cast<unsigned short>(noted);
    any |= noted;
    to_half16(make_uint4(u[0], u[1], u[2], u[3]), o);
    sts16(dst + k * 2048, o[0], o[1], o[2], o[3]);
    sts16((dst + k * 2048) ^ 16u, o[4], o[5], o[6], o[7]);
  }
  return __any_sync(0xffffffffu, any != 0);
}

// More registers for the sums, fewer for the others: 96 + 2 x 112 + 192 = 512 is what the launch has, 128 each.
template <int N>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <int D>
__global__ void __launch_bounds__(TC_THREADS, 1) cache_attn_tc_kernel(const __grid_constant__ AttnArgs a) {
  constexpr uint32_t RAW = ATTN_PAGE * D, F16 = ATTN_PAGE * D * 2;
  // tensor memory columns
  constexpr uint32_t COL_Q = 0, COL_S = D / 2, COL_P = COL_S + 2 * ATTN_PAGE, COL_O = COL_P + ATTN_PAGE;
  static_assert(COL_O + 2 * D <= 512, "tensor memory");
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t raw_full[TC_RAW], raw_empty[TC_RAW], unit_full[TC_UNITS], kf_full[2], vf_full[2], qk_done[2], pv_done[2], s_empty[2],
      p_full[2], o_empty[2], q_full, fin_full[8], pair_full[4];
  __shared__ PageRec s_page[TC_PAGES];
  __shared__ UnitRec s_unit[TC_UNITS];
  __shared__ float2 s_alpha[4][TC_ROWS];   // what a row's sums so far are scaled by, and what its page's sum is
  __shared__ float s_fin[8][3][TC_ROWS], s_max[2][2][TC_ROWS];
  __shared__ __align__(8) unsigned short s_nan[4][D][4];      // edge pages: the tokens of each dimension that hold NaN
  __shared__ int s_has_nan[4][2];
  __shared__ int s_sum[TC_THREADS / 32];
  __shared__ int s_entry;
  __shared__ int s_start;
  __shared__ uint32_t tmem_slot;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = a.group, entries = a.batch * a.tiles;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t k16 = smem_base, v16 = k16 + 2 * F16, raw = v16 + 2 * F16;

  if (tid == 0) {
    for (int i = 0; i < TC_RAW; ++i) {
      mbar_init(smem_u32(&raw_full[i]), 1);
      mbar_init(smem_u32(&raw_empty[i]), 2);
    }
    for (int i = 0; i < TC_UNITS; ++i) mbar_init(smem_u32(&unit_full[i]), 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&kf_full[i]), 2);
      mbar_init(smem_u32(&vf_full[i]), 2);
      mbar_init(smem_u32(&qk_done[i]), 1);
      mbar_init(smem_u32(&pv_done[i]), 1);
      mbar_init(smem_u32(&s_empty[i]), 8);
      mbar_init(smem_u32(&p_full[i]), 8);
      mbar_init(smem_u32(&o_empty[i]), 4);
    }
    mbar_init(smem_u32(&q_full), 8);
    for (int i = 0; i < 8; ++i) mbar_init(smem_u32(&fin_full[i]), 8);
    for (int i = 0; i < 4; ++i) mbar_init(smem_u32(&pair_full[i]), 2);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_slot), 512);
    tmem_relinquish();
  }
  griddep_wait();

  // The list of items, as in cache_attn_kernel.
  const int per = (entries + TC_THREADS - 1) / TC_THREADS;
  const int e0 = min(tid * per, entries), e1 = min(e0 + per, entries);
  auto items_of = [&](int e) { return attn_items(attn_entry_of(a, e, group, TC_ROWS)) * a.hk; };
  int mine = 0;
  for (int e = e0; e < e1; ++e) {
    mine += items_of(e);
    if (blockIdx.x == 0) attn_report_bad(a, e);
  }
  int incl = mine;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, s);
    if (lane >= s) incl += up;
  }
  if (lane == 31) s_sum[warp] = incl;
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  griddep_launch_dependents();   // behind the wait, as in cache_attn_kernel, and behind the allocation: who comes in may want tensor memory
  const uint32_t tmem = tmem_slot;
  int base = 0, total = 0;
  for (int w = 0; w < TC_THREADS / 32; ++w) {
    if (w < warp) base += s_sum[w];
    total += s_sum[w];
  }
  const int begin = base + incl - mine, end = base + incl;
  const AttnDeal deal = attn_deal(total, static_cast<int>(gridDim.x));
  const int worker = blockIdx.x;
  const int f0 = worker < deal.workers ? attn_range(deal, worker) : 0;
  const int items = worker < deal.workers ? attn_range(deal, worker + 1) - f0 : 0;
  if (items > 0 && f0 >= begin && f0 < end) {
    int at = begin;
    int e = e0;
    for (; e + 1 < e1; ++e) {
      const int next = at + items_of(e);
      if (f0 < next) break;
      at = next;
    }
    s_entry = e;
    s_start = at;
  }
  if (blockIdx.x == 0) {
    int at = begin;
    for (int e = e0; e < e1; ++e) {
      a.prefix[e] = at;
      if (e + 1 < e1) at += items_of(e);
    }
    if (tid == 0) a.prefix[entries] = total;
  }
  __syncthreads();

  // (A range of head items alone has no page: beside the first, no role has anything to wait for.)
  const bool pages = items > 0 && items > ATTN_HEAD - (f0 - s_start) % attn_items(attn_entry_of(a, s_entry, group, TC_ROWS));
  bool ok = true;
  // (A barrier of which no phase is complete yet lets a wait for the parity before the first pass: that is how the two
  // buffers' first uses find them free.)
  // A wait of the whole warp: all lanes come back with the same answer, and together.
  // (Several at once: their first looks are in flight together, a look takes a hundred clocks or two.)
  auto warp_wait = [&](uint64_t& bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar), parity)) != 0; };
  auto warp_wait2 = [&](uint64_t& bar0, uint32_t p0, uint64_t& bar1, uint32_t p1) {
    const bool r0 = mbar_try_wait(smem_u32(&bar0), p0), r1 = mbar_try_wait(smem_u32(&bar1), p1);
    if (__all_sync(0xffffffffu, r0 && r1)) return true;
    return warp_wait(bar0, p0) && warp_wait(bar1, p1);
  };
  auto warp_wait3 = [&](uint64_t& bar0, uint32_t p0, uint64_t& bar1, uint32_t p1, uint64_t& bar2, uint32_t p2) {
    const bool r0 = mbar_try_wait(smem_u32(&bar0), p0), r1 = mbar_try_wait(smem_u32(&bar1), p1), r2 = mbar_try_wait(smem_u32(&bar2), p2);
    if (__all_sync(0xffffffffu, r0 && r1 && r2)) return true;
    return warp_wait(bar0, p0) && warp_wait(bar1, p1) && warp_wait(bar2, p2);
  };
  if (warp < 4) {
    regs_down<96>();
    if (warp == 0 && items > 0) {
      // ---- looks pages up, describes them, and copies their codes
      EntryCache cache;
      cache.base = -64;
      Cursor c;
      c.e = s_entry;
      c.en = attn_entry_cached(a, cache, c.e, entries, group, TC_ROWS);
      const int off0 = f0 - s_start, per_unit = attn_items(c.en);
      c.h = off0 / per_unit;
      c.i = off0 % per_unit - ATTN_HEAD;
      int unit0 = s_start + c.h * per_unit;
      int left = items, n = 0, unit = 0, issued = 0;
      bool in_unit = false;
      // how many pages of the range lie in the unit that c stands in, and whether any page follows
      while (left > 0 && ok) {
        if (c.i < 0) {
          const int skip = min(-c.i, left);
          c.i += skip;
          left -= skip;
          continue;
        }
        // pages of this unit in the range, up to 32 at a time, one per lane
        const int in_range = min(c.en.pages - c.i, left), take = min(in_range, 32);
        if (!in_unit) {
          in_unit = true;
          if (lane == 0) {
            UnitRec& u = s_unit[unit & (TC_UNITS - 1)];
            u.first = c.en.first; u.row0 = c.en.row0; u.rows = c.en.rows; u.pos = c.en.pos;
            u.h = c.h;
            u.whole = c.i == 0 && in_range == c.en.pages;
            u.slot = attn_slot_of(deal, worker, unit0 + ATTN_HEAD);
            mbar_arrive(smem_u32(&unit_full[unit & (TC_UNITS - 1)]));   // releases the record
          }
          ++unit;
        }
        int tile = -1, exps = 127 | 127 << 8;
        if (lane < take && c.en.last >= 0) {
          const int b = a.tiles == 1 ? c.e : c.e / a.tiles;
          const int p = __ldcg(a.page_table + static_cast<size_t>(b) * a.width + c.en.page0 + c.i + lane);
          if (p >= 0 && p < a.pages) {
            tile = p * a.hk + c.h;
            exps = __ldcg(a.k_exp + tile) | __ldcg(a.v_exp + tile) << 8;
          } else {
            atomicOr(a.status, ST_BAD_PAGE);
          }
        }
        const int p_first = c.en.pos + div_group(a, c.en.row0), p_last = c.en.pos + div_group(a, c.en.row0 + c.en.rows - 1);
        const bool follows = [&] {   // does a page follow this unit's share of the range?
          int rest = left - in_range;
          if (rest <= 0) return false;
          return rest > ATTN_HEAD;   // the next unit's head items come first
        }();
        for (int j = 0; j < take && ok; ++j) {
          const int t = __shfl_sync(0xffffffffu, tile, j), ex = __shfl_sync(0xffffffffu, exps, j);
          const int p0 = (c.en.page0 + c.i + j) * ATTN_PAGE;
          const bool seg_last = j + 1 == take && take == in_range;
          // K, then V; the record is written ahead of the K slot's arrival
          for (int half = 0; half < 2 && ok; ++half) {
            const int slot = issued % TC_RAW, turn = issued / TC_RAW;
            if (turn > 0 && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&raw_empty[slot]), (turn - 1) & 1))) {
              ok = false;
              break;
            }
            if (lane == 0) {
              if (half == 0) {
                PageRec r;
                const bool edge = p_first < p0 + ATTN_PAGE - 1 || (a.window > 0 && p_last - a.window + 1 > p0);
                r.bits = ex | ((seg_last ? PAGE_SEG_LAST : 0) | (seg_last && !follows ? PAGE_RANGE_LAST : 0) |
                               (edge ? PAGE_EDGE : 0) | (t >= 0 ? PAGE_LIVE : 0)) << 16;
                r.p0 = p0;
                const int lo = a.window > 0 ? max(p_first - a.window + 1 - p0, 0) : 0, hi = min(p_last - p0, ATTN_PAGE - 1);
                r.seen = (lo > 63 ? 63 : lo) | max(hi, 0) << 8;
                s_page[n & (TC_PAGES - 1)] = r;
              }
              const uint32_t bar = smem_u32(&raw_full[slot]);
              if (t >= 0) {
                mbar_expect_tx(bar, RAW);
                bulk_load_1d(raw + static_cast<uint32_t>(slot) * RAW, (half ? a.v : a.k) + static_cast<size_t>(t) * RAW, RAW, bar);
              } else {
                mbar_arrive(bar);
              }
            }
            __syncwarp();
            ++issued;
          }
          ++n;
        }
        c.i += take;
        left -= take;
        if (take == in_range) {
          in_unit = false;
          if (left > 0) {
            unit0 += attn_items(c.en);
            c.i = -ATTN_HEAD;
            if (++c.h == a.hk) {
              c.h = 0;
              do {
                if (++c.e >= entries) {
                  left = 0;
                  break;
                }
                c.en = attn_entry_cached(a, cache, c.e, entries, group, TC_ROWS);
              } while (c.en.pages == 0);
            }
          }
        }
      }
      if (!ok) {
        for (int i = issued > TC_RAW ? issued - TC_RAW : 0; i < issued; ++i) mbar_wait(smem_u32(&raw_full[i % TC_RAW]), (i / TC_RAW) & 1);
      }
    } else if (warp == 1 && pages) {
      // ---- MMA. The whole warp walks along and one elected lane issues: what is the same in all lanes is then known to be
      // (an MMA's operands are uniform registers; out of a branch of one lane each would be moved there first, which
      // took three times as long as the MMA itself).
      constexpr uint32_t id_s = umma_idesc_f16(TC_ROWS, ATTN_PAGE), id_o = umma_idesc_f16(TC_ROWS, D);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      int unit = 0;
      bool fresh = true, last = false;
      // S of page n, then O' of page n - 1, whose weights were made meanwhile
      for (int n = 0; ok; ++n) {
        const uint32_t b = n & 1, ph = (n >> 1) & 1;
        const bool done = last;
        if (!done) {
          if (fresh) ok = warp_wait(q_full, unit++ & 1);   // the unit's q is in tensor memory
          ok = ok && warp_wait2(kf_full[b], ph, s_empty[b], ph ^ 1u);
          if (!ok) break;
          tc_fence_after_sync();
          const uint64_t kd = umma_desc_k_sw128(k16 + b * F16);
          const uint32_t ds = tm + COL_S + b * ATTN_PAGE;
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < D / 16; ++k)   // the next 64 dimensions are a swizzle atom of their own
              umma_f16_ts(ds, tm + COL_Q + 8 * k, kd + (k / 4) * (ATTN_PAGE * 128 / 16) + 2 * (k % 4), id_s, k > 0 ? 1u : 0u);
            umma_commit(smem_u32(&qk_done[b]));
          }
          __syncwarp();
          const int bits = __shfl_sync(0xffffffffu, s_page[n & (TC_PAGES - 1)].bits >> 16, 0);   // visible: kf_full was waited for
          last = bits & PAGE_RANGE_LAST;
          fresh = bits & PAGE_SEG_LAST;
        }
        if (n > 0) {
          const uint32_t b1 = b ^ 1u, ph1 = ((n - 1) >> 1) & 1;
          ok = warp_wait3(p_full[b1], ph1, vf_full[b1], ph1, o_empty[b1], ph1 ^ 1u);
          if (!ok) break;
          tc_fence_after_sync();
          const uint64_t vd = umma_desc_k_sw128(v16 + b1 * F16);
          const uint32_t dd = tm + COL_O + b1 * D, da = tm + COL_P + b1 * (ATTN_PAGE / 2);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < ATTN_PAGE / 16; ++k) umma_f16_ts(dd, da + 8 * k, vd + 2 * k, id_o, k > 0 ? 1u : 0u);
            umma_commit(smem_u32(&pv_done[b1]));
          }
          __syncwarp();
        }
        if (done) break;
      }
    } else if (warp >= 2 && pages) {
      // ---- codes to FP16, two warps: a thread takes 16 codes (32 bytes of FP16) at a time
      const int ct = tid - 64;
      constexpr int PIECES = D / 16;   // 16-code pieces of a token
      // Where the thread's piece of a token's K row goes: chunks j and j + 1 of its half's 128 bytes, swizzled.
      const int piece = ct % PIECES, tok0 = ct / PIECES;
      const uint32_t k_at = static_cast<uint32_t>(piece / 4) * (ATTN_PAGE * 128) + static_cast<uint32_t>(tok0) * 128 +
                            ((((piece % 4) * 2) ^ (tok0 & 7)) << 4);
      // and 16 tokens of a V row (a dimension)
      const int vp = ct & 3, dim0 = ct >> 2;
      const uint32_t v_at = static_cast<uint32_t>(dim0) * 128 + (((2 * vp) ^ (dim0 & 7)) << 4);
      bool last = false;
      int used = 0;
      for (int n = 0; ok && !last; ++n) {
        const int b = n & 1;
        const uint32_t ph = (n >> 1) & 1;
        int slot = used % TC_RAW;
        ok = warp_wait2(raw_full[slot], (used / TC_RAW) & 1, qk_done[b], ph ^ 1u);
        if (!ok) break;
        const PageRec r = s_page[n & (TC_PAGES - 1)];
        const int bits = r.bits >> 16;
        last = bits & PAGE_RANGE_LAST;
        const bool live = bits & PAGE_LIVE, edge = bits & PAGE_EDGE;
        if (live) {
          // A thread's pieces are 64 / PIECES tokens apart, a multiple of 8: the same place in the swizzle, a fixed stride.
          const uint32_t src = raw + static_cast<uint32_t>(slot) * RAW + static_cast<uint32_t>(ct) * 16;
          const uint32_t dst = k16 + b * F16 + k_at;
          constexpr int N = ATTN_PAGE * PIECES / 64;
          uint4 x[N];
#pragma unroll
          for (int k = 0; k < N; ++k) x[k] = lds16(src + k * 1024);   // all in flight
#pragma unroll
          for (int k = 0; k < N; ++k) {
            uint32_t o[8];
            to_half16(x[k], o);
            // the two halves' lanes write even and odd chunks in turn: no bank twice
            sts16(dst + k * (64 / PIECES) * 128, o[0], o[1], o[2], o[3]);
            sts16((dst + k * (64 / PIECES) * 128) ^ 16u, o[4], o[5], o[6], o[7]);
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&raw_empty[slot]));
          mbar_arrive(smem_u32(&kf_full[b]));
        }
        ++used;
        slot = used % TC_RAW;
        ok = warp_wait2(raw_full[slot], (used / TC_RAW) & 1, pv_done[b], ph ^ 1u);
        if (!ok) break;
        {
          const uint32_t src = raw + static_cast<uint32_t>(slot) * RAW + static_cast<uint32_t>(ct) * 16, dst = v16 + b * F16 + v_at;
          int some = 0;
          if (edge || !live) {
            some = convert_v_edge<D>(src, dst, live, (r.seen & 255) - 16 * vp, (r.seen >> 8) - 16 * vp, &s_nan[n & 3][dim0][vp]);
          } else {
            uint4 x[D / 16];
#pragma unroll
            for (int k = 0; k < D / 16; ++k) x[k] = lds16(src + k * 1024);
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              uint32_t o[8];
              to_half16(x[k], o);
              sts16(dst + k * 2048, o[0], o[1], o[2], o[3]);
              sts16((dst + k * 2048) ^ 16u, o[4], o[5], o[6], o[7]);
            }
          }
          if (lane == 0) s_has_nan[n & 3][warp - 2] = some;
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&raw_empty[slot]));
          mbar_arrive(smem_u32(&vf_full[b]));
        }
        ++used;
      }
    }
  } else if (warp < 12) {
    regs_down<112>();
    if (pages) {
      // ---- softmax: two threads per row, 32 tokens of a page each; warps w and w + 4 share their rows
      const int half = warp >= 8, other = half ^ 1;
      const int row = (warp & 3) * 32 + lane;
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      bool last = false;
      int unit = 0, n = 0;
      while (ok && !last) {
        const int us = unit & (TC_UNITS - 1);
        ok = warp_wait(unit_full[us], (unit / TC_UNITS) & 1);
        if (!ok) break;
        const UnitRec u = s_unit[us];
        const bool there = row < u.rows;
        const int rr = u.row0 + row, tk = div_group(a, rr), pos = u.pos + tk;
        float f_row;
        {   // q to tensor memory: FP16 under a power of two, the row's largest value to [2^9, 2^10)
          const __nv_bfloat16* src = a.q + static_cast<size_t>(u.first + tk) * a.ld_q + static_cast<size_t>(u.h * group + rr - tk * group) * D;
          uint4 w[D / 8];
          float amax = 0.f;
#pragma unroll
          for (int i = 0; i < D / 8; ++i) w[i] = there ? __ldcg(reinterpret_cast<const uint4*>(src) + i) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) amax = fmaxf(amax, fmaxf(finite_abs(bf16lo_f32(x[k])), finite_abs(bf16hi_f32(x[k]))));
          }
          const int e = q_exponent(amax);
          const float down = exp2_byte(127 - e);
          f_row = a.scale_log2 * exp2_byte(127 + e);
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            if (i / (D / 64) != half) continue;   // half the row each
            uint32_t p[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const uint4& v = w[4 * i + k / 4];
              const uint32_t x = (k & 3) == 0 ? v.x : (k & 3) == 1 ? v.y : (k & 3) == 2 ? v.z : v.w;
              p[k] = pack_half2(bf16lo_f32(x) * down, bf16hi_f32(x) * down);
            }
            tmem_st16(tmem + lanes + COL_Q + 16 * i, p);
          }
          tmem_store_wait();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&q_full));
        }
        float mx = -INFINITY, l = 0.f;
        bool seg_last = false;
        for (; ok && !seg_last; ++n) {
          const int b = n & 1;
          const uint32_t ph = (n >> 1) & 1;
          ok = warp_wait(qk_done[b], ph);
          if (!ok) break;
          tc_fence_after_sync();
          const PageRec r = s_page[n & (TC_PAGES - 1)];
          const int bits = r.bits >> 16;
          seg_last = bits & PAGE_SEG_LAST;
          last = bits & PAGE_RANGE_LAST;
          const float f = score_factor(f_row, exp2_byte(r.bits & 255));
          // The thread's scores stay in registers; what the row does not see of them becomes -infinity.
          uint32_t v[32];
          tmem_ld32(tmem + lanes + COL_S + b * ATTN_PAGE + half * 32, v);
          tmem_ld_wait();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&s_empty[b]));
          if (!(bits & PAGE_LIVE) || (bits & PAGE_EDGE)) {
            const int lim = there && (bits & PAGE_LIVE) ? min(pos - r.p0, ATTN_PAGE - 1) : -1, low = a.window > 0 ? max(pos - a.window + 1 - r.p0, 0) : 0;
            const unsigned long long all = lim >= low ? (~0ull >> (63 - lim)) & (~0ull << low) : 0ull;
            const uint32_t sees = static_cast<uint32_t>(all >> (32 * half));
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(sees >> i & 1u)) v[i] = 0xff800000u;
          }
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 32; i += 2) m4[i / 2 & 3] = max3(m4[i / 2 & 3], __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
          const float m_half = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
          s_max[b][half][row] = m_half;
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&pair_full[warp & 3]));
          // (the second: the P buffer's last reader)
          ok = warp_wait2(pair_full[warp & 3], n & 1, pv_done[b], ph ^ 1u);
          if (!ok) break;
          tc_fence_after_sync();
          // The reference of the weights follows the maximum only when that has grown by more than 2^8 (the weights stay below
          // 2^8, and lifted inside FP16): the sums are then hardly ever to be scaled.
          const float m_new = fmaxf(m_half, s_max[b][other][row]) * f, grown = m_new > mx + 8.f || (mx == -INFINITY && m_new > mx) ? m_new : mx;
          const float base2 = grown == -INFINITY ? 0.f : grown, alpha = grown == mx ? 1.f : exp2_fast(mx - base2);
          mx = grown;
          const bool loud = too_loud_to_lift(mx);
          const float lift = loud ? 0.f : TC_LIFT, unlift = loud ? 1.f : TC_UNLIFT;
          if (half == 0) s_alpha[n & 3][row] = make_float2(alpha, unlift);
          const unsigned long long ff = pack2(f, f), bb = pack2(lift - base2, lift - base2);
          unsigned long long l2[2] = {0ull, 0ull};
          uint32_t p[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float e0, e1;
            unpack2(fma2(pack2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), ff, bb), e0, e1);
            e0 = exp2_fast(e0);
            e1 = exp2_fast(e1);
            l2[i / 2 & 1] = add2(l2[i / 2 & 1], pack2(e0, e1));
            p[i >> 1] = pack_half2(e0, e1);
          }
          float l_lo, l_hi;
          unpack2(add2(l2[0], l2[1]), l_lo, l_hi);
          tmem_st16(tmem + lanes + COL_P + b * (ATTN_PAGE / 2) + half * 16, p);
          l = fmaf(l, alpha, (l_lo + l_hi) * unlift);
          if (seg_last) {
            if (half == 0) s_fin[unit & 7][2][row] = mx;
            s_fin[unit & 7][half][row] = l;
          }
          tmem_store_wait();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) {
            if (seg_last) mbar_arrive(smem_u32(&fin_full[unit & 7]));
            mbar_arrive(smem_u32(&p_full[b]));
          }
        }
        ++unit;
      }
    }
  } else {
    regs_up<192>();
    if (pages) {
      // ---- sums and output: a thread per row
      const int row = (warp & 3) * 32 + lane;
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      bool last = false;
      int unit = 0;
      unsigned long long o[D / 2];   // two dimensions each
#pragma unroll
      for (int i = 0; i < D / 2; ++i) o[i] = 0ull;
      for (int n = 0; ok && !last; ++n) {
        const int b = n & 1;
        const uint32_t ph = (n >> 1) & 1;
        ok = warp_wait(pv_done[b], ph);
        if (!ok) break;
        tc_fence_after_sync();
        const PageRec r = s_page[n & (TC_PAGES - 1)];
        const int bits = r.bits >> 16;
        last = bits & PAGE_RANGE_LAST;
        const float2 scale = s_alpha[n & 3][row];
        const float alpha = scale.x, vs = exp2_byte(r.bits >> 8 & 255) * scale.y;
        const unsigned long long vs2 = pack2(vs, vs);
        if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
          for (int i = 0; i < D / 2; ++i) o[i] = fma2(o[i], pack2(alpha, alpha), 0ull);
        }
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          uint32_t v[16], w[16];
          tmem_ld16(tmem + lanes + COL_O + b * D + c, v);
          tmem_ld16(tmem + lanes + COL_O + b * D + c + 16, w);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if (i & 1) continue;
            o[(c + i) / 2] = fma2(pack2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), vs2, o[(c + i) / 2]);
            o[(c + 16 + i) / 2] = fma2(pack2(__uint_as_float(w[i]), __uint_as_float(w[i + 1])), vs2, o[(c + 16 + i) / 2]);
          }
        }
        if ((bits & PAGE_EDGE) && (s_has_nan[n & 3][0] | s_has_nan[n & 3][1])) {
          // rows that see a token with NaN in a dimension have NaN there
          const UnitRec& u = s_unit[unit & (TC_UNITS - 1)];
          const int pos = u.pos + div_group(a, u.row0 + row), lim = min(pos - r.p0, ATTN_PAGE - 1), low = a.window > 0 ? max(pos - a.window + 1 - r.p0, 0) : 0;
          unsigned long long sees = 0;
          if (row < u.rows && lim >= low) sees = (~0ull >> (63 - lim)) & (~0ull << low);
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            uint32_t bad = 0;
#pragma unroll 1
            for (int i = 0; i < 32; ++i)
              bad |= (*reinterpret_cast<const unsigned long long*>(&s_nan[n & 3][c + i][0]) & sees) ? 1u << i : 0u;
            if (__any_sync(0xffffffffu, bad != 0)) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (bad >> i & 1u) o[(c + i) / 2] |= 0x7fffffffull << (32 * (i & 1));
            }
          }
        }
        if (!(bits & PAGE_SEG_LAST)) {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&o_empty[b]));
          continue;
        }
        // The unit's end. The sums go through the page's O' once more: read back from there, the loop over a row's dimensions
        // can stay one.
        const uint32_t to = tmem + lanes + COL_O + b * D;
#pragma unroll
        for (int c = 0; c < D; c += 16) {
          uint32_t v[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = static_cast<uint32_t>(o[(c + i) / 2] >> (32 * (i & 1)));
#pragma unroll
          for (int i = 0; i < 8; ++i) o[c / 2 + i] = 0ull;
          tmem_st16(to + c, v);
        }
        tmem_store_wait();
        ok = warp_wait(fin_full[unit & 7], (unit >> 3) & 1);
        if (!ok) break;
        const UnitRec u = s_unit[unit & (TC_UNITS - 1)];
        const bool there = row < u.rows;
        const float m = s_fin[unit & 7][2][row], l = s_fin[unit & 7][0][row] + s_fin[unit & 7][1][row];
        const float inv = !u.whole ? 1.f : l == 0.f ? 0.f : 1.f / l;   // no token seen: the row is zero
        const int rr = u.row0 + row, tk = div_group(a, rr), col = (u.h * group + rr - tk * group) * D;
        float* part = a.part + static_cast<size_t>(u.slot) * attn_slot_floats(D, TC_ROWS);
        if (there && !u.whole) {
          part[row] = m;
          part[TC_ROWS + row] = l;
        }
        part += 2 * TC_ROWS + static_cast<size_t>(row) * D;
#pragma unroll 1
        for (int c = 0; c < D; c += 8) {
          uint32_t v[8];
          tmem_ld8(to + c, v);
          tmem_ld_wait();
          float x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(v[i]) * inv;
          if (there && u.whole) store8(a, u.first + tk, col + c, x);
          if (there && !u.whole) {
            *reinterpret_cast<float4*>(part + c) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4*>(part + c + 4) = make_float4(x[4], x[5], x[6], x[7]);
          }
          __syncwarp();
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&o_empty[b]));
        ++unit;
      }
    }
  }
  if (!ok && lane == 0) atomicOr(a.status, ST_ATTN_TIMEOUT);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

template <int D>
static cudaError_t tc_launch(const AttnArgs& a, int sms, cudaStream_t stream) {
  const size_t smem = tc_smem_bytes(D) > TC_MIN_SMEM ? tc_smem_bytes(D) : TC_MIN_SMEM;
  static DeviceOnce once;
  const cudaError_t e = once.run([&] { return cudaFuncSetAttribute(cache_attn_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)); });
  if (e != cudaSuccess) return e;
  return launch_dependent(cache_attn_tc_kernel<D>, dim3(sms), dim3(TC_THREADS), smem, stream, a);
}

cudaError_t cache_attn_tc_launch(const AttnArgs& a, int dim, int sms, cudaStream_t stream) {
  return dim == 128 ? tc_launch<128>(a, sms, stream) : tc_launch<64>(a, sms, stream);
}

}  // namespace muse
