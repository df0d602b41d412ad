// Attention of the newest tokens of each sequence over its paged 8-bit cache (rope_append.cu):
//     o[r] = sum over seen tokens p of softmax(q[r] . k[p] / sqrt(D))_p v[p],    then o *= sigmoid(gate)
// in one pass with a running maximum and sum per row (FP32, powers of two). A row sees the tokens up to its own
// position, the last `window` of them where a window is given; a row that sees none is zero.
//
// What bounds it is reading the cache: 2 D bytes per token and KV head, for all query heads that share the head (and a
// sequence's few new tokens) at once: they are the rows of one 16-row MMA tile. The pages of all sequences and heads
// form one list that is cut into equal ranges (attn_sched.cuh), one per warp, whatever the sequences' lengths, so
// that a batch of any shape keeps every SM's loads in flight; a warp brings its pages in with bulk copies (K and V of
// a page and head are 64 D contiguous bytes each) into a ring of its own and waits for nobody else. More than 16
// rows (a chunk of a prompt) take 16 rows per warp and one ring and range per CTA.
//
// Codes become FP16 in registers (exact, as e4m3 is a subset), q becomes FP16 under a power of two per row (exact down
// to 2^-34 of the row's largest value), the scores take both powers in FP32. A lane's 16 bytes of k are 4 k-slots of 4 MMAs; the
// order of slots is free as long as q follows it. The n-index of the score MMAs is a token order of our choosing too:
// lane (g, t) gets tokens 16 t .. 16 t + 15 of the page for row g, which is what the second product wants as its A
// fragment beside V kept [dim, token], so neither operand passes through shared memory again. The probabilities are
// rounded to FP16 (2^-11, values below 2^-14 of the running maximum to 2^-25 of it), a page's sum is scaled by its V
// exponent in FP32.
#include "attn_sched.cuh"
#include "cache8.cuh"
#include "fp8.cuh"

namespace muse {

constexpr int ATTN_TILE = 16;   // rows of one warp's MMA tile
constexpr int ATTN_WARPS = 8;
constexpr int ATTN_THREADS = ATTN_WARPS * 32;

__host__ __device__ constexpr int attn_slots(int D) { return D == 128 ? 3 : 6; }              // ring slots per warp
__host__ __device__ constexpr int attn_ring_bytes(int D) { return ATTN_WARPS * attn_slots(D) * ATTN_PAGE * D; }
// Floats of one partial slot of a tile of `rows` rows: (max, sum) per row, then the rows.
__host__ __device__ constexpr int attn_slot_floats(int D, int rows) { return rows * (D + 2); }

__device__ __forceinline__ void mma_f16_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a));
  return r;
}

__device__ __forceinline__ AttnEntry attn_entry_of(const AttnArgs& a, int e, int group, int tile) {
  const int b = e / a.tiles, rt = e % a.tiles;
  const int c0 = a.cu_q ? __ldcg(a.cu_q + b) : b, c1 = a.cu_q ? __ldcg(a.cu_q + b + 1) : b + 1;
  return attn_entry(c0, c1, __ldcg(a.seq_lens + b), a.m, a.max_q, a.width * ATTN_PAGE, group, tile, rt, a.window);
}

// A place in the list of pages: entry, head, i-th page of the unit.
struct Cursor {
  AttnEntry en;
  int e, h, i;
};

// The rows' state of one 16-row tile in a warp: lane (g, t) holds rows g and g + 8.
template <int D>
struct TileState {
  float o[D / 8][4];
  float mx[2], l[2];   // running maximum (log2 units) and the lane's share of the running sum
};

template <int D>
__device__ __forceinline__ void tile_reset(TileState<D>& s) {
#pragma unroll
  for (int n = 0; n < D / 8; ++n) s.o[n][0] = s.o[n][1] = s.o[n][2] = s.o[n][3] = 0.f;
  s.mx[0] = s.mx[1] = -INFINITY;
  s.l[0] = s.l[1] = 0.f;
}

// q fragments of 16 rows (row0 .. of the unit's rows) as FP16 under a power of two per row; qs = the row's factor for
// the scores in log2 units.
template <int D>
__device__ __forceinline__ void load_q(const AttnArgs& a, const AttnEntry& en, int h, int row0, int rows, int group, uint32_t (&qf)[D / 16][4], float (&qs)[2]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = g + 8 * half;
    uint4 w[D / 32];   // 16 dimensions (two vectors) per 64
    float amax = 0.f;
    const bool live = r < rows;
    const int rr = row0 + r;
    const __nv_bfloat16* src = a.q + static_cast<size_t>(en.first + (live ? rr / group : 0)) * a.ld_q + static_cast<size_t>(h * group + (live ? rr % group : 0)) * D;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      w[c] = live ? __ldcg(reinterpret_cast<const uint4*>(src + 64 * (c >> 1) + 16 * t + 8 * (c & 1))) : make_uint4(0u, 0u, 0u, 0u);
      const uint32_t u[4] = {w[c].x, w[c].y, w[c].z, w[c].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fmaxf(finite_abs(bf16lo_f32(u[i])), finite_abs(bf16hi_f32(u[i]))));
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // largest value to [2^9, 2^10): FP16's smallest step, 2^-24, is then 2^-34 of it
    const int e = max(min(static_cast<int>(__float_as_uint(amax) >> 23) - 127 - 9, 100), -100);
    const float down = exp2_byte(127 - e);
    qs[half] = a.scale_log2 * exp2_byte(127 + e);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const uint32_t u[4] = {w[c].x, w[c].y, w[c].z, w[c].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // word i of vector c holds dimensions 8 (c & 1) + 2 i, + 1 of the lane's 16: MMA 4 (c >> 1) + 2 (c & 1) + (i >> 1)
        const uint32_t hv = pack_half2(bf16lo_f32(u[i]) * down, bf16hi_f32(u[i]) * down);
        qf[4 * (c >> 1) + 2 * (c & 1) + (i >> 1)][2 * (i & 1) + half] = hv;
      }
    }
  }
}

// One page: scores, softmax step, P V. `ks`, `vs`: shared-memory addresses of the page's k [64][D] and v [D][64].
// lim / low: last and first position each of the lane's rows sees, relative to the page's first token.
template <int D>
__device__ __forceinline__ void page_scores(float (&s)[8][4], const uint32_t (&qf)[D / 16][4], uint32_t ks) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
    const uint32_t row = ks + static_cast<uint32_t>(16 * (g >> 1) + 2 * j + (g & 1)) * D + 16 * t;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const uint4 w = lds16(row + 64 * c);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        mma_f16_16816(s[j], qf[4 * c + i][0], qf[4 * c + i][1], qf[4 * c + i][2], qf[4 * c + i][3], fp8_to_half2(static_cast<uint16_t>(u[i] & 0xffffu)),
                      fp8_to_half2(static_cast<uint16_t>(u[i] >> 16)));
    }
  }
}

// Bytes of `w` (four tokens from `tok`) outside [lo, hi] become zero.
__device__ __forceinline__ uint32_t keep_tokens(uint32_t w, int tok, int lo, int hi) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m |= (tok + i >= lo && tok + i <= hi) ? 0xffu << (8 * i) : 0u;
  return w & m;
}
__device__ __forceinline__ bool has_nan_code(uint32_t w) { return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0; }

// o = o * alpha + vscale * P V. Tokens outside [lo, hi] of the page have P = 0, but their codes may stand for NaN.
template <int D, bool EDGE>
__device__ __forceinline__ void page_pv(TileState<D>& st, const uint32_t (&p)[4][4], uint32_t vs, float a0, float a1, float vscale, int lo, int hi) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int n = 0; n < D / 8; ++n) {
    const uint4 w = lds16(vs + static_cast<uint32_t>(8 * n + g) * ATTN_PAGE + 16 * t);
    uint32_t u[4] = {w.x, w.y, w.z, w.w};
    float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (EDGE) u[i] = keep_tokens(u[i], 16 * t + 4 * i, lo, hi);
      mma_f16_16816(c, p[i][0], p[i][1], p[i][2], p[i][3], fp8_to_half2(static_cast<uint16_t>(u[i] & 0xffffu)), fp8_to_half2(static_cast<uint16_t>(u[i] >> 16)));
    }
    st.o[n][0] = fmaf(c[0], vscale, st.o[n][0] * a0);
    st.o[n][1] = fmaf(c[1], vscale, st.o[n][1] * a0);
    st.o[n][2] = fmaf(c[2], vscale, st.o[n][2] * a1);
    st.o[n][3] = fmaf(c[3], vscale, st.o[n][3] * a1);
  }
}

// lim[2], low[2]: first and last token of the page that rows g and g + 8 see; any_lo, any_hi: of any row of the tile,
// all_lo, all_hi: of all of them. `s`: the page's raw scores; they become the weights `p`, and (a0, a1) what the rows' sums so
// far are to be scaled by. Returns whether some row does not see some token.
template <int D>
__device__ __forceinline__ bool page_softmax(TileState<D>& st, float (&s)[8][4], uint32_t (&p)[4][4], float& a0, float& a1, const float (&qs)[2], float kscale,
                                             const int (&low)[2], const int (&lim)[2], int all_lo, int all_hi) {
  const int t = threadIdx.x & 3;
  const float f0 = qs[0] * kscale, f1 = qs[1] * kscale;
  const bool edge = all_lo > 0 || all_hi < ATTN_PAGE - 1;   // warp-uniform
  float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      s[j][c] *= f0;
      s[j][2 + c] *= f1;
      if (edge) {
        const int tok = 16 * t + 2 * j + c;
        if (tok < low[0] || tok > lim[0]) s[j][c] = -INFINITY;
        if (tok < low[1] || tok > lim[1]) s[j][2 + c] = -INFINITY;
      }
      m0 = fmaxf(m0, s[j][c]);
      m1 = fmaxf(m1, s[j][2 + c]);
    }
  }
  m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, 1));
  m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, 2));
  m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, 1));
  m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, 2));
  m0 = fmaxf(m0, st.mx[0]);
  m1 = fmaxf(m1, st.mx[1]);
  const float b0 = m0 == -INFINITY ? 0.f : m0, b1 = m1 == -INFINITY ? 0.f : m1;   // nothing seen yet: every weight is 2^-inf = 0
  a0 = exp2_fast(st.mx[0] - b0);
  a1 = exp2_fast(st.mx[1] - b1);
  st.mx[0] = m0;
  st.mx[1] = m1;
  float l0 = 0.f, l1 = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float e0 = exp2_fast(s[j][0] - b0), e1 = exp2_fast(s[j][1] - b0), e2 = exp2_fast(s[j][2] - b1), e3 = exp2_fast(s[j][3] - b1);
    l0 += e0 + e1;
    l1 += e2 + e3;
    p[j >> 1][2 * (j & 1)] = pack_half2(e0, e1);
    p[j >> 1][2 * (j & 1) + 1] = pack_half2(e2, e3);
  }
  st.l[0] = st.l[0] * a0 + l0;
  st.l[1] = st.l[1] * a1 + l1;
  return edge;
}

// A page that some row does not see all of. Tokens that no row sees (behind the sequence, or left of the window) may hold
// anything: their codes count as zero. A token that only some rows see and that holds NaN must not reach the others
// through 0 * NaN: such a page is multiplied once per distinct bound (rare: looked for in the codes).
template <int D>
__device__ __forceinline__ void page_pv_edge(TileState<D>& st, const uint32_t (&p)[4][4], uint32_t vs, float a0, float a1, float vscale, const int (&low)[2],
                                          const int (&lim)[2], int any_lo, int any_hi) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  bool nan = false;
#pragma unroll 4
  for (int n = 0; n < D / 8; ++n) {
    const uint4 w = lds16(vs + static_cast<uint32_t>(8 * n + g) * ATTN_PAGE + 16 * t);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) nan |= has_nan_code(keep_tokens(u[i], 16 * t + 4 * i, any_lo, any_hi));
  }
  if (!__any_sync(0xffffffffu, nan)) {
    page_pv<D, true>(st, p, vs, a0, a1, vscale, any_lo, any_hi);
    return;
  }
#pragma unroll
  for (int n = 0; n < D / 8; ++n) {
    st.o[n][0] *= a0;
    st.o[n][1] *= a0;
    st.o[n][2] *= a1;
    st.o[n][3] *= a1;
  }
#pragma unroll 1
  for (int r = 0; r < ATTN_TILE; ++r) {
    const int rl = __shfl_sync(0xffffffffu, r < 8 ? low[0] : low[1], (r & 7) * 4), rh = __shfl_sync(0xffffffffu, r < 8 ? lim[0] : lim[1], (r & 7) * 4);
    bool seen_before = false;
    for (int x = 0; x < r; ++x) {
      const int xl = __shfl_sync(0xffffffffu, x < 8 ? low[0] : low[1], (x & 7) * 4), xh = __shfl_sync(0xffffffffu, x < 8 ? lim[0] : lim[1], (x & 7) * 4);
      seen_before |= xl == rl && xh == rh;
    }
    if (seen_before || rl > rh) continue;   // warp-uniform
    const bool u0 = low[0] == rl && lim[0] == rh, u1 = low[1] == rl && lim[1] == rh;
    uint32_t pr[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      pr[i][0] = u0 ? p[i][0] : 0u;
      pr[i][1] = u1 ? p[i][1] : 0u;
      pr[i][2] = u0 ? p[i][2] : 0u;
      pr[i][3] = u1 ? p[i][3] : 0u;
    }
    TileState<D> one;
    tile_reset(one);
    page_pv<D, true>(one, pr, vs, 0.f, 0.f, vscale, max(rl, 0), min(rh, ATTN_PAGE - 1));
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      if (u0) { st.o[n][0] += one.o[n][0]; st.o[n][1] += one.o[n][1]; }
      if (u1) { st.o[n][2] += one.o[n][2]; st.o[n][3] += one.o[n][3]; }
    }
  }
}

__device__ __forceinline__ float sigmoid_f32(float x) { return 1.f / (1.f + __expf(-x)); }

// A finished segment of a unit: the output rows themselves when the segment is the whole unit, else a partial slot.
template <int D>
__device__ __forceinline__ void tile_store(TileState<D>& st, const AttnArgs& a, const AttnEntry& en, int h, int row0, int rows, int group, bool whole, float* slot,
                                           int slot_rows, int slot_row0) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float l = st.l[half];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    const int r = g + 8 * half;
    if (r >= rows) continue;
    if (whole) {
      const float inv = l == 0.f ? 0.f : 1.f / l;   // no token seen: the row is zero
      const int rr = row0 + r;
      const size_t tok = en.first + rr / group;
      const int col = (h * group + rr % group) * D;
      __nv_bfloat16* o = a.out + tok * a.ld_out + col;
      const __nv_bfloat16* gt = a.gate ? a.gate + tok * a.ld_gate + col : nullptr;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        float x = st.o[n][2 * half] * inv, y = st.o[n][2 * half + 1] * inv;
        if (gt) {
          const uint32_t w = __ldcg(reinterpret_cast<const uint32_t*>(gt + 8 * n + 2 * t));
          x *= sigmoid_f32(bf16lo_f32(w));
          y *= sigmoid_f32(bf16hi_f32(w));
        }
        *reinterpret_cast<__nv_bfloat162*>(o + 8 * n + 2 * t) = __floats2bfloat162_rn(x, y);
      }
    } else {
      if (t == 0) {
        slot[slot_row0 + r] = st.mx[half];
        slot[slot_rows + slot_row0 + r] = l;
      }
      float* o = slot + 2 * slot_rows + static_cast<size_t>(slot_row0 + r) * D;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) *reinterpret_cast<float2*>(o + 8 * n + 2 * t) = make_float2(st.o[n][2 * half], st.o[n][2 * half + 1]);
    }
  }
}

// SHARED: the CTA is one worker of 128 rows, all warps on the same pages; else every warp is a worker of 16 rows.
template <int D, bool SHARED>
__global__ void __launch_bounds__(ATTN_THREADS, 1) cache_attn_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int TILE = SHARED ? ATTN_TILE * ATTN_WARPS : ATTN_TILE;
  constexpr int SLOTS = SHARED ? attn_slots(D) * ATTN_WARPS : attn_slots(D);   // ring slots of one worker
  constexpr uint32_t SLOT_BYTES = ATTN_PAGE * D;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bar_full[attn_slots(D) * ATTN_WARPS], bar_empty[attn_slots(D) * ATTN_WARPS];
  __shared__ long long s_sum[ATTN_WARPS + 1];
  __shared__ int s_entry[ATTN_WARPS];
  __shared__ long long s_start[ATTN_WARPS];
  __shared__ int2 s_rec[ATTN_WARPS][64];   // looked-up pages: tile index in the pool, exponents (k | v << 8)
  __shared__ volatile int s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = a.hq / a.hk, entries = a.batch * a.tiles;
  const int ring = SHARED ? 0 : warp;   // this warp's ring
  uint64_t* const full = bar_full + (SHARED ? 0 : warp * attn_slots(D));
  uint64_t* const empty = bar_empty + (SHARED ? 0 : warp * attn_slots(D));
  const uint32_t ring_base = smem_u32(smem) + static_cast<uint32_t>(ring) * attn_slots(D) * SLOT_BYTES;
  if (tid < attn_slots(D) * ATTN_WARPS) {
    mbar_init(smem_u32(&bar_full[tid]), 1);
    mbar_init(smem_u32(&bar_empty[tid]), ATTN_WARPS);   // used by the shared ring only
    fence_mbar_init();
  }
  if (tid == 0) s_abort = 0;
  griddep_launch_dependents();
  griddep_wait();

  // The list of pages: every thread adds up the entries of its share, a scan over the CTA gives the total and where
  // each share begins; the thread whose share holds a worker's first page finds the entry.
  const int per = (entries + ATTN_THREADS - 1) / ATTN_THREADS;
  const int e0 = min(tid * per, entries), e1 = min(e0 + per, entries);
  long long mine = 0;
  for (int e = e0; e < e1; ++e) {
    const AttnEntry en = attn_entry_of(a, e, group, TILE);
    mine += static_cast<long long>(en.pages) * a.hk;
    if (blockIdx.x == 0) {
      const int b = e / a.tiles;
      const int len = __ldcg(a.seq_lens + b);
      bool bad = len < 0 || len > a.width * ATTN_PAGE;
      if (a.cu_q) {
        const int c0 = __ldcg(a.cu_q + b), c1 = __ldcg(a.cu_q + b + 1);
        bad |= c0 < 0 || c1 < c0 || c1 > a.m || c1 - c0 > a.max_q;
      }
      if (bad) atomicOr(a.status, ST_BAD_LENGTH);
    }
  }
  long long incl = mine;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, incl, s);
    if (lane >= s) incl += up;
  }
  if (lane == 31) s_sum[warp] = incl;
  __syncthreads();
  long long base = 0, total = 0;
  for (int w = 0; w < ATTN_WARPS; ++w) {
    if (w < warp) base += s_sum[w];
    total += s_sum[w];
  }
  const long long begin = base + incl - mine, end = base + incl;   // this thread's share of the list
  const AttnDeal deal = attn_deal(total, static_cast<int>(SHARED ? gridDim.x : gridDim.x * ATTN_WARPS));
  // Neighbouring workers sit on different SMs, so that a list with fewer pages than warps is spread over all of them.
  auto worker_of = [&](int w) { return static_cast<int>(SHARED ? blockIdx.x : w * gridDim.x + blockIdx.x); };
  if (total > 0) {
    for (int w = 0; w < (SHARED ? 1 : ATTN_WARPS); ++w) {
      if (worker_of(w) >= deal.workers) break;
      const long long f = attn_range(deal, worker_of(w));
      if (f >= begin && f < end) {
        long long at = begin;
        for (int e = e0; e < e1; ++e) {
          const long long next = at + static_cast<long long>(attn_entry_of(a, e, group, TILE).pages) * a.hk;
          if (f < next) {
            s_entry[w] = e;
            s_start[w] = at;
            break;
          }
          at = next;
        }
      }
    }
    if (blockIdx.x == 0) {   // for the kernel that adds up the partial sums
      long long at = begin;
      for (int e = e0; e < e1; ++e) {
        a.prefix[e] = at;
        at += static_cast<long long>(attn_entry_of(a, e, group, TILE).pages) * a.hk;
      }
    }
  }
  if (blockIdx.x == 0 && tid == 0) a.prefix[entries] = total;
  __syncthreads();
  const int worker = worker_of(warp);
  if (worker >= deal.workers) return;   // SHARED: CTA-uniform; else this warp has no page, and nobody waits for it
  const long long f0 = attn_range(deal, worker);
  const int count = static_cast<int>(attn_range(deal, worker + 1) - f0);   // this worker's pages

  Cursor rd, fill;   // where the warp computes, and up to where it has looked up pages
  {
    const int w = SHARED ? 0 : warp;
    rd.e = s_entry[w];
    rd.en = attn_entry_of(a, rd.e, group, TILE);
    const int off = static_cast<int>(f0 - s_start[w]);
    rd.h = off / rd.en.pages;
    rd.i = off % rd.en.pages;
    fill = rd;
  }
  auto next_unit = [&](Cursor& c) {   // false behind the last entry
    c.i = 0;
    if (++c.h < a.hk) return true;
    c.h = 0;
    do {
      if (++c.e >= entries) return false;
      c.en = attn_entry_of(a, c.e, group, TILE);
    } while (c.en.pages == 0);
    return true;
  };
  // Looks up the next 32 pages of the worker's list, a page per lane: the tile's index in the pool (page * hk + head; -1:
  // not a page of the pool, or nothing is seen) and its two exponents, into the warp's ring of records.
  int filled = 0;
  auto look_up = [&]() {
    int b = -1, h = 0, i = 0, off = 0;
    while (off < 32 && filled + off < count) {
      const int left = fill.en.pages - fill.i, take = min(left, 32 - off);
      if (lane >= off && lane < off + take) {
        b = fill.en.last < 0 ? -1 : fill.e / a.tiles;
        h = fill.h;
        i = fill.en.page0 + fill.i + lane - off;
      }
      off += take;
      fill.i += take;
      if (fill.i == fill.en.pages && !next_unit(fill)) break;
    }
    int2 rec = make_int2(-1, 127 | 127 << 8);
    if (b >= 0 && filled + lane < count) {
      const int p = __ldcg(a.page_table + static_cast<size_t>(b) * a.width + i);
      if (p >= 0 && p < a.pages) {
        rec.x = p * a.hk + h;
        rec.y = __ldcg(a.k_exp + rec.x) | __ldcg(a.v_exp + rec.x) << 8;
      } else {
        atomicOr(a.status, ST_BAD_PAGE);
      }
    }
    s_rec[warp][(filled + lane) & 63] = rec;
    filled += 32;
    __syncwarp();
  };
  look_up();

  int issued = 0, used = 0;               // halves (K, then V of a page) requested and consumed by this worker
  const int halves = 2 * count;
  const bool issuer = !SHARED || warp == 0;
  // Requests the next half; every lane of the issuing warp runs it.
  auto request = [&]() {
    const int slot = issued % SLOTS, turn = issued / SLOTS;
    if (SHARED && turn > 0 && !mbar_wait(smem_u32(&empty[slot]), (turn - 1) & 1)) {
      if (lane == 0) atomicOr(a.status, ST_ATTN_TIMEOUT);
      s_abort = 1;
      return;
    }
    if (lane == 0) {
      const uint32_t bar = smem_u32(&full[slot]);
      const int tile = s_rec[warp][(issued >> 1) & 63].x;
      if (tile >= 0) {
        mbar_expect_tx(bar, SLOT_BYTES);
        bulk_load_1d(ring_base + static_cast<uint32_t>(slot) * SLOT_BYTES, ((issued & 1) ? a.v : a.k) + static_cast<size_t>(tile) * SLOT_BYTES, SLOT_BYTES, bar);
      } else {
        mbar_arrive(bar);   // nothing to bring: the page is masked whole
      }
    }
    ++issued;
  };
  // The warp has read a half: its slot may be filled again.
  auto release = [&]() {
    __syncwarp();
    if (SHARED && lane == 0) mbar_arrive(smem_u32(&empty[used % SLOTS]));
    ++used;
    if (issuer)
      while (issued < halves && issued < used + SLOTS && (issued >> 1) < filled && !(SHARED && s_abort)) request();
  };
  if (issuer)
    while (issued < halves && issued < SLOTS && (issued >> 1) < filled) request();

  TileState<D> st;
  uint32_t qf[D / 16][4];
  float qs[2];
  const int wrow = SHARED ? warp * ATTN_TILE : 0;   // this warp's first row in the worker's tile
  bool fresh = true, first_segment = true;
  int seg_first = 0, my_rows = 0;                   // first page of the segment; rows of this warp
  for (int n = 0; n < count; ++n) {
    if (fresh) {
      my_rows = max(0, min(ATTN_TILE, rd.en.rows - wrow));
      tile_reset(st);
      load_q<D>(a, rd.en, rd.h, rd.en.row0 + wrow, my_rows, group, qf, qs);
      fresh = false;
      seg_first = rd.i;
    }
    // records: looked up 32 at a time, while those of the pages under way stay (the ring of records holds 64)
    if (filled < count && filled - n <= SLOTS / 2 + 2) look_up();
    const int2 rec = s_rec[warp][n & 63];
    const bool live = rec.x >= 0 && my_rows > 0;
    const int ks = used % SLOTS, vsl = (used + 1) % SLOTS, vt = (used + 1) / SLOTS;
    bool ok = mbar_wait(smem_u32(&full[ks]), (used / SLOTS) & 1);
    float s[8][4], a0, a1;
    uint32_t p[4][4];
    int low[2], lim[2], any_lo, any_hi, all_lo, all_hi;   // positions grow with the row
    bool edge = false;
    if (ok && live) page_scores<D>(s, qf, ring_base + static_cast<uint32_t>(ks) * SLOT_BYTES);
    release();
    if (ok && live) {
      const int p0 = (rd.en.page0 + rd.i) * ATTN_PAGE, g = lane >> 2;
      auto bounds = [&](int r, int& lo, int& hi) {   // tokens of the page that row r of the warp's tile sees
        const int pos = rd.en.pos + (rd.en.row0 + wrow + r) / group;
        hi = pos - p0;
        lo = a.window > 0 ? pos - a.window + 1 - p0 : 0;
      };
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        bounds(g + 8 * half, low[half], lim[half]);
        if (g + 8 * half >= my_rows) {   // rows that are not there see nothing
          low[half] = ATTN_PAGE;
          lim[half] = -1;
        }
      }
      bounds(0, any_lo, all_hi);
      bounds(my_rows - 1, all_lo, any_hi);
      edge = page_softmax<D>(st, s, p, a0, a1, qs, exp2_byte(rec.y & 255), low, lim, all_lo, all_hi);
    }
    ok = ok && mbar_wait(smem_u32(&full[vsl]), vt & 1);
    if (!ok || (SHARED && s_abort)) {
      if (lane == 0 && !ok) atomicOr(a.status, ST_ATTN_TIMEOUT);
      s_abort = 1;
      break;
    }
    if (live) {
      const uint32_t vs = ring_base + static_cast<uint32_t>(vsl) * SLOT_BYTES;
      const float vscale = exp2_byte(rec.y >> 8);
      if (edge) page_pv_edge<D>(st, p, vs, a0, a1, vscale, low, lim, any_lo, any_hi);
      else page_pv<D, false>(st, p, vs, a0, a1, vscale, 0, ATTN_PAGE - 1);
    }
    release();
    // end of the unit or of the range: the segment [seg_first, rd.i] is done
    const bool unit_end = rd.i == rd.en.pages - 1;
    if (unit_end || n + 1 == count) {
      const bool whole = unit_end && seg_first == 0;
      // a worker has at most two partial segments: the one it begins inside a unit, and the one it ends inside one
      float* slot = a.part + (2ll * worker + (first_segment ? 0 : 1)) * attn_slot_floats(D, TILE);
      tile_store<D>(st, a, rd.en, rd.h, rd.en.row0 + wrow, my_rows, group, whole, slot, TILE, wrow);
      fresh = true;
      first_segment = false;
    }
    if (n + 1 < count) {
      if (unit_end) next_unit(rd);
      else ++rd.i;
    }
  }
  if (s_abort) {
    // leave no copy in flight behind: each slot's last request is waited for (bounded)
    if (issuer)
      for (int i = issued > SLOTS ? issued - SLOTS : 0; i < issued; ++i) mbar_wait(smem_u32(&full[i % SLOTS]), (i / SLOTS) & 1);
  }
}

// Adds up the partial sums of the units that were split between workers: one warp per row, a unit's segments in page
// order (the same bits in every run).
template <int D, bool SHARED>
__global__ void __launch_bounds__(128) cache_attn_join_kernel(const __grid_constant__ AttnArgs a, int workers) {
  constexpr int TILE = SHARED ? ATTN_TILE * ATTN_WARPS : ATTN_TILE;
  constexpr int V = D / 32;   // dimensions per lane
  griddep_launch_dependents();
  griddep_wait();
  const int entries = a.batch * a.tiles, group = a.hq / a.hk;
  const int e = static_cast<int>(blockIdx.x) / a.hk, h = static_cast<int>(blockIdx.x) % a.hk;
  const int r = static_cast<int>(blockIdx.y) * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const long long total = __ldcg(a.prefix + entries), start = __ldcg(a.prefix + e);
  const AttnEntry en = attn_entry_of(a, e, group, TILE);
  if (r >= en.rows) return;
  const AttnDeal deal = attn_deal(total, workers);
  const long long u0 = start + static_cast<long long>(h) * en.pages;
  const int w0 = attn_worker(deal, u0), w1 = attn_worker(deal, u0 + en.pages - 1);
  if (w0 == w1) return;   // one worker had the whole unit and has written it
  // all but the first worker's segments are that worker's first
  const size_t stride = 2ull * attn_slot_floats(D, TILE);
  const float* const first = a.part + static_cast<size_t>(attn_slot_of(deal, w0, u0)) * attn_slot_floats(D, TILE);
  const float* const rest = a.part + static_cast<size_t>(w0) * stride;   // worker w0 + i's first slot, i > 0: rest + i stride
  const int parts = w1 - w0 + 1;
  float mx = -INFINITY;
  for (int i = lane; i < parts; i += 32) mx = fmaxf(mx, __ldcg((i ? rest + i * stride : first) + r));
#pragma unroll
  for (int s = 16; s; s >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
  const float b = mx == -INFINITY ? 0.f : mx;
  float l = 0.f, o[V] = {};
#pragma unroll 8
  for (int i = 0; i < parts; ++i) {
    const float* s = i ? rest + i * stride : first;
    const float f = exp2_fast(__ldcg(s + r) - b);
    l = fmaf(__ldcg(s + TILE + r), f, l);
    const float* src = s + 2 * TILE + static_cast<size_t>(r) * D + lane * V;
    if constexpr (V == 4) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>(src));
      o[0] = fmaf(x.x, f, o[0]); o[1] = fmaf(x.y, f, o[1]); o[2] = fmaf(x.z, f, o[2]); o[3] = fmaf(x.w, f, o[3]);
    } else {
      const float2 x = __ldcg(reinterpret_cast<const float2*>(src));
      o[0] = fmaf(x.x, f, o[0]); o[1] = fmaf(x.y, f, o[1]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int rr = en.row0 + r;
  const size_t tok = en.first + rr / group;
  const int col = (h * group + rr % group) * D + lane * V;
#pragma unroll
  for (int c = 0; c < V; c += 2) {
    float x = o[c] * inv, y = o[c + 1] * inv;
    if (a.gate) {
      const uint32_t w = __ldcg(reinterpret_cast<const uint32_t*>(a.gate + tok * a.ld_gate + col + c));
      x *= sigmoid_f32(bf16lo_f32(w));
      y *= sigmoid_f32(bf16hi_f32(w));
    }
    *reinterpret_cast<__nv_bfloat162*>(a.out + tok * a.ld_out + col + c) = __floats2bfloat162_rn(x, y);
  }
}

// ---------------------------------------------------------------- host side
static int attn_sms() {
  int dev = 0, v = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return v;
}
static bool attn_shared(int max_q, int hq, int hk) { return static_cast<long long>(max_q) * (hq / hk) > ATTN_TILE; }
static int attn_tiles(int max_q, int hq, int hk) {
  const int tile = attn_shared(max_q, hq, hk) ? ATTN_TILE * ATTN_WARPS : ATTN_TILE;
  return (max_q * (hq / hk) + tile - 1) / tile;
}

long long cache_attn_ws_bytes(int batch, int max_q, int hq, int hk, int dim) {
  const int sms = attn_sms();
  if (batch < 1 || max_q < 1 || hk < 1 || hq < hk || hq % hk || (dim != 64 && dim != 128) || sms < 1) return -1;
  const bool sh = attn_shared(max_q, hq, hk);
  const long long workers = sh ? sms : static_cast<long long>(sms) * ATTN_WARPS;
  const long long part = 2 * workers * attn_slot_floats(dim, sh ? ATTN_TILE * ATTN_WARPS : ATTN_TILE) * 4;
  return part + (static_cast<long long>(batch) * attn_tiles(max_q, hq, hk) + 1) * 8;
}

template <int D, bool SHARED>
static cudaError_t attn_launch(const AttnArgs& a, int sms, cudaStream_t stream) {
  const size_t smem = attn_ring_bytes(D);
  cudaError_t e = cudaFuncSetAttribute(cache_attn_kernel<D, SHARED>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  e = launch_dependent(cache_attn_kernel<D, SHARED>, dim3(sms), dim3(ATTN_THREADS), smem, stream, a);
  if (e != cudaSuccess) return e;
  const int tile = SHARED ? ATTN_TILE * ATTN_WARPS : ATTN_TILE;
  const int rows = a.max_q * (a.hq / a.hk) < tile ? a.max_q * (a.hq / a.hk) : tile;
  const long long workers = SHARED ? sms : static_cast<long long>(sms) * ATTN_WARPS;
  const long long units = static_cast<long long>(a.batch) * a.tiles * a.hk;
  return launch_dependent(cache_attn_join_kernel<D, SHARED>, dim3(static_cast<unsigned>(units), (rows + 3) / 4), dim3(128), 0, stream, a, static_cast<int>(workers));
}

int cache_attn_dispatch(AttnArgs a, int dim, void* ws, cudaStream_t stream) {
  if (!a.q || !a.k || !a.v || !a.k_exp || !a.v_exp || !a.page_table || !a.seq_lens || !a.out || !a.status || !ws) return -1;
  if (a.m < 1 || a.batch < 1 || a.width < 1 || a.pages < 1 || a.max_q < 1 || a.hk < 1 || a.hq < a.hk || a.hq % a.hk || (dim != 64 && dim != 128)) return -2;
  if (a.width > 0x7fffffff / ATTN_PAGE || a.window < 0 || static_cast<long long>(a.max_q) * (a.hq / a.hk) > 0x3fffffff) return -3;
  if (a.ld_q % 8 || a.ld_q < static_cast<long long>(a.hq) * dim || a.ld_out % 2 || a.ld_out < static_cast<long long>(a.hq) * dim) return -4;
  if (a.gate && (a.ld_gate % 2 || a.ld_gate < static_cast<long long>(a.hq) * dim || (reinterpret_cast<uintptr_t>(a.gate) & 3))) return -4;
  if ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(ws)) & 15) return -5;
  if (reinterpret_cast<uintptr_t>(a.out) & 3) return -5;
  if (!a.cu_q && a.max_q != 1) return -6;
  const int sms = attn_sms();
  if (sms < 1) return -7;
  a.tiles = attn_tiles(a.max_q, a.hq, a.hk);
  if (static_cast<long long>(a.batch) * a.tiles * a.hk > 0x7fffffffll || static_cast<long long>(a.pages) * a.hk > 0x7fffffffll) return -3;
  const bool sh = attn_shared(a.max_q, a.hq, a.hk);
  const long long workers = sh ? sms : static_cast<long long>(sms) * ATTN_WARPS;
  a.part = static_cast<float*>(ws);
  a.prefix = reinterpret_cast<long long*>(a.part + 2 * workers * attn_slot_floats(dim, sh ? ATTN_TILE * ATTN_WARPS : ATTN_TILE));
  cudaError_t e;
  if (dim == 128) e = sh ? attn_launch<128, true>(a, sms, stream) : attn_launch<128, false>(a, sms, stream);
  else e = sh ? attn_launch<64, true>(a, sms, stream) : attn_launch<64, false>(a, sms, stream);
  return static_cast<int>(e);
}

// ---- the same plan on the host
namespace {
struct HostPlan {
  int group, tile, tiles, entries;
  long long workers, total;
  bool ok;
};
}  // namespace
static HostPlan host_plan(const int* seq_lens, int m, int batch, int width, int max_q, int hq, int hk, int window, int sms) {
  HostPlan p = {};
  p.ok = seq_lens && m >= 1 && batch >= 1 && width >= 1 && width <= 0x7fffffff / ATTN_PAGE && max_q >= 1 && hk >= 1 && hq >= hk && hq % hk == 0 &&
         window >= 0 && sms >= 1;
  if (!p.ok) return p;
  const bool sh = attn_shared(max_q, hq, hk);
  p.group = hq / hk;
  p.tile = sh ? ATTN_TILE * ATTN_WARPS : ATTN_TILE;
  p.tiles = attn_tiles(max_q, hq, hk);
  p.entries = batch * p.tiles;
  p.workers = sh ? sms : static_cast<long long>(sms) * ATTN_WARPS;
  return p;
}
static AttnEntry host_entry(const HostPlan& p, const int* seq_lens, const int* cu_q, int m, int width, int max_q, int window, int e) {
  const int b = e / p.tiles;
  return attn_entry(cu_q ? cu_q[b] : b, cu_q ? cu_q[b + 1] : b + 1, seq_lens[b], m, max_q, width * ATTN_PAGE, p.group, p.tile, e % p.tiles, window);
}

long long cache_attn_plan(const int* seq_lens, const int* cu_q, int m, int batch, int width, int max_q, int hq, int hk, int window, int sms,
                          int* segments, long long capacity) {
  HostPlan p = host_plan(seq_lens, m, batch, width, max_q, hq, hk, window, sms);
  if (!p.ok || !segments) return -1;
  for (int e = 0; e < p.entries; ++e) p.total += static_cast<long long>(host_entry(p, seq_lens, cu_q, m, width, max_q, window, e).pages) * hk;
  if (p.total == 0) return 0;
  const AttnDeal deal = attn_deal(p.total, static_cast<int>(p.workers));
  long long count = 0, start = 0;
  int e = 0;
  AttnEntry en = host_entry(p, seq_lens, cu_q, m, width, max_q, window, 0);
  for (int w = 0; w < deal.workers; ++w) {
    bool first = true;
    for (long long f = attn_range(deal, w), f1 = attn_range(deal, w + 1); f < f1;) {
      while (f >= start + static_cast<long long>(en.pages) * hk) {
        start += static_cast<long long>(en.pages) * hk;
        en = host_entry(p, seq_lens, cu_q, m, width, max_q, window, ++e);
      }
      const int off = static_cast<int>(f - start), h = off / en.pages, i = off % en.pages;
      const int n = static_cast<int>(f1 - f < en.pages - i ? f1 - f : en.pages - i);
      if (count < capacity) {
        int* s = segments + 6 * count;
        s[0] = w; s[1] = e; s[2] = h; s[3] = en.page0 + i; s[4] = n;
        s[5] = n == en.pages ? -1 : 2 * w + (first ? 0 : 1);
      }
      ++count;
      first = false;
      f += n;
    }
  }
  return count;
}

long long cache_attn_join(const int* seq_lens, const int* cu_q, int m, int batch, int width, int max_q, int hq, int hk, int window, int sms,
                          int entry, int head, int* slots, long long capacity) {
  HostPlan p = host_plan(seq_lens, m, batch, width, max_q, hq, hk, window, sms);
  if (!p.ok || !slots || entry < 0 || entry >= p.entries || head < 0 || head >= hk) return -1;
  long long before = 0;
  for (int e = 0; e < p.entries; ++e) {
    if (e == entry) before = p.total;
    p.total += static_cast<long long>(host_entry(p, seq_lens, cu_q, m, width, max_q, window, e).pages) * hk;
  }
  const AttnEntry en = host_entry(p, seq_lens, cu_q, m, width, max_q, window, entry);
  if (en.rows == 0) return 0;
  const AttnDeal deal = attn_deal(p.total, static_cast<int>(p.workers));
  const long long u0 = before + static_cast<long long>(head) * en.pages;
  const int w0 = attn_worker(deal, u0), w1 = attn_worker(deal, u0 + en.pages - 1);
  if (w0 == w1) return 0;
  for (int w = w0; w <= w1; ++w)
    if (w - w0 < capacity) slots[w - w0] = attn_slot_of(deal, w, u0);
  return w1 - w0 + 1;
}

}  // namespace muse
