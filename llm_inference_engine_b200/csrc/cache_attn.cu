// Attention of the newest tokens of each sequence over its paged 8-bit cache (rope_append.cu):
//     o[r] = sum over seen tokens p of softmax(q[r] . k[p] / sqrt(D))_p v[p],    then o *= sigmoid(gate)
// in one pass with a running maximum and sum per row (FP32, powers of two). A row sees the tokens up to its own
// position, the last `window` of them where a window is given; a row that sees none is zero.
//
// What bounds it is reading the cache: 2 D bytes per token and KV head, for all query heads that share the head (and a
// sequence's few new tokens) at once: they are the rows. The pages of all sequences and heads form one list that is
// cut into equal ranges (attn_sched.cuh), one per warp, whatever the sequences' lengths, so that a batch of any shape
// keeps every SM's loads in flight; a warp brings its pages in with bulk copies (K and V of a page and head are 64 D
// contiguous bytes each) into a ring of its own and waits for nobody else. More than 16 rows (a chunk of a prompt) take
// the kernel of cache_attn_tc.cu, with a range per CTA.
//
// The cache is the MMAs' M operand and the rows their N = 8 (or two such tiles): the work per page then follows the
// rows there are, and a page's codes are converted once for all of them. Codes become FP16 in registers (exact, as e4m3
// is a subset), q becomes FP16 under a power of two per row (rounded by at most 2^-34 of the row's largest value; BF16 values down
// to 2^-27 of it are exact), the scores take both powers in FP32. Scores S^T[token][row]: a lane's 16 bytes of k are 4 k-slots of 4 MMAs; the order of slots is free as
// long as q follows it. O^T[dim][row] += V^T[dim][token] P^T[token][row]: V is kept [dim, token], so a lane's 16 bytes are
// tokens 16 t .. 16 t + 15 of a dimension, and the token order of the score tiles is chosen so that, after one 8 x 8
// transpose in registers (movmatrix), the lane holds the same tokens' weights. Neither operand passes through
// shared memory a second time. The weights are rounded to FP16, lifted by 2^14 (2^-11 of a weight; those below 2^-28 of the
// running maximum to 2^-39 of it), a page's sum is scaled by its V exponent, and back, in FP32.
//
// Measured with the kernel that adds up split units (us, and the cache's bytes against 6.46 TB/s of copying): 64 sequences of up to
// 4000 tokens, 32 query and 16 KV heads 117 (5.02 TB/s, 0.78); 2 of 100,000, 32 and 4 heads, 46.5 (4.4 TB/s, 0.68); 21 with drafts of
// up to 4 and a window of 1000, 16 and 4 heads of 64, 17.4; 32 of 4000 with 4 drafts, 32 and 8 heads, 73; one of 300 tokens 11.1,
// where nothing is moved and the chain of the two launches is what is waited for (index tensors, page table, one page's copy,
// its products, a partial sum, adding up). The form with 16 rows and D = 128 spills 60 bytes at 255 registers. What made the difference on the way
// (64 sequences): a CTA per sequence and head with barriers 250; a ring per warp 213; equal ranges over one list 148;
// page records and q for the next unit under way early 127; parts of one unit in one CTA met in shared memory, head items 116.
#include "cache_attn.cuh"

namespace muse {

constexpr int ATTN_WARPS = 8;
constexpr int ATTN_THREADS = ATTN_WARPS * 32;

__host__ __device__ constexpr int attn_slots(int D) { return D == 128 ? 3 : 6; }              // ring slots per warp
__host__ __device__ constexpr int attn_ring_bytes(int D) { return ATTN_WARPS * attn_slots(D) * ATTN_PAGE * D; }
__device__ __forceinline__ void mma_f16_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Lists of up to so many items are spread over the SMs (a warp each) instead of filling CTA after CTA.
__host__ __device__ constexpr int attn_spread_below(int sms) { return 2 * sms; }

// 8 x 8 16-bit matrix, a row per quad of lanes: transposed.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// The state of a warp's 8 NT rows. Lane (g, t) holds rows 8 n + 2 t and + 1 of dimensions 16 d + g and + 8.
template <int D, int NT>
struct TileState {
  float o[D / 16][NT][4];
  float mx[NT][2], l[NT][2];   // running maximum (log2 units) and the lane's share of the running sum
};

template <int D, int NT>
__device__ __forceinline__ void tile_reset(TileState<D, NT>& s) {
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int d = 0; d < D / 16; ++d) s.o[d][n][0] = s.o[d][n][1] = s.o[d][n][2] = s.o[d][n][3] = 0.f;
    s.mx[n][0] = s.mx[n][1] = -INFINITY;
    s.l[n][0] = s.l[n][1] = 0.f;
  }
}

// What a warp knows of its rows: positions of the lane's rows, of the first and of the last row.
template <int NT>
struct RowInfo {
  int pos[NT][2];
  bool there[NT][2];
  int first, last;
};

// q fragments of 8 NT rows (from row0 of the unit's rows) as FP16 under a power of two per row; qs = the factor of the
// lane's rows 2 t, 2 t + 1 for the scores in log2 units.
template <int D, int NT>
__device__ __forceinline__ void load_q(const AttnArgs& a, const AttnEntry& en, int h, int row0, int rows, uint32_t (&qf)[NT][D / 16][2],
                                       float (&qs)[NT][2]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint4 w[NT][D / 32];   // 16 dimensions (two vectors) per 64
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = g + 8 * n, tok = div_group(a, row0 + r), hd = (row0 + r) - tok * a.group;
    const __nv_bfloat16* src = a.q + static_cast<size_t>(en.first + tok) * a.ld_q + static_cast<size_t>(h * a.group + hd) * D;
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
      w[n][c] = r < rows ? __ldcg(reinterpret_cast<const uint4*>(src + 64 * (c >> 1) + 16 * t + 8 * (c & 1))) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float amax = 0.f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const uint32_t u[4] = {w[n][c].x, w[n][c].y, w[n][c].z, w[n][c].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fmaxf(finite_abs(bf16lo_f32(u[i])), finite_abs(bf16hi_f32(u[i]))));
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // FP16's smallest step, 2^-24, is then 2^-34 of the largest value
    const int e = q_exponent(amax);
    const float down = exp2_byte(127 - e), up = a.scale_log2 * exp2_byte(127 + e);
    qs[n][0] = __shfl_sync(0xffffffffu, up, 8 * t);
    qs[n][1] = __shfl_sync(0xffffffffu, up, 8 * t + 4);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const uint32_t u[4] = {w[n][c].x, w[n][c].y, w[n][c].z, w[n][c].w};
#pragma unroll
      for (int i = 0; i < 4; ++i)   // word i holds dimensions 8 (c & 1) + 2 i, + 1 of the lane's 16: k-step 4 (c >> 1) + 2 (c & 1) + (i >> 1)
        qf[n][4 * (c >> 1) + 2 * (c & 1) + (i >> 1)][i & 1] = pack_half2(bf16lo_f32(u[i]) * down, bf16hi_f32(u[i]) * down);
    }
  }
}

// Raw scores of a page: s[i][n] holds tokens 16 (g >> 1) + 4 i + (g & 1) (values 0, 1: rows 2 t, 2 t + 1) and the token two
// further (values 2, 3). ks: the page's k [64][D] in shared memory.
template <int D, int NT>
__device__ __forceinline__ void page_scores(float (&s)[4][NT][4], const uint32_t (&qf)[NT][D / 16][2], uint32_t ks) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t base = ks + static_cast<uint32_t>(16 * (g >> 1) + (g & 1)) * D + 16 * t;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int n = 0; n < NT; ++n) s[i][n][0] = s[i][n][1] = s[i][n][2] = s[i][n][3] = 0.f;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const uint4 x = lds16(base + static_cast<uint32_t>(4 * i) * D + 64 * c), y = lds16(base + static_cast<uint32_t>(4 * i + 2) * D + 64 * c);
      const uint32_t u[4] = {x.x, x.y, x.z, x.w}, v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t a0 = fp8_to_half2(static_cast<uint16_t>(u[k] & 0xffffu)), a2 = fp8_to_half2(static_cast<uint16_t>(u[k] >> 16));
        const uint32_t a1 = fp8_to_half2(static_cast<uint16_t>(v[k] & 0xffffu)), a3 = fp8_to_half2(static_cast<uint16_t>(v[k] >> 16));
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16_16816(s[i][n], a0, a1, a2, a3, qf[n][4 * c + k][0], qf[n][4 * c + k][1]);
      }
    }
  }
}

// Scores to weights: p[i][n] = the weights of the lane's two tokens of tile i, packed over rows (2 t, 2 t + 1), before the
// transpose, lifted: times `unlift` (the same for all of the warp's rows) they are the weights. `a`: what the rows' sums so
// far are to be scaled by (`moved`: not all of the warp's are 1).
constexpr float ATTN_LIFT = 14.f, ATTN_UNLIFT = 1.f / 16384.f;   // FP16 then holds weights down to 2^-38 of the row's largest
template <int D, int NT>
__device__ __forceinline__ void page_softmax(TileState<D, NT>& st, float (&s)[4][NT][4], uint32_t (&p)[4][NT][2], float (&a)[NT][2], bool& moved, float& unlift,
                                             const float (&qs)[NT][2], float kscale, const RowInfo<NT>& ri, int p0, int window, bool edge) {
  const int lane = threadIdx.x & 31, g = lane >> 2;
  bool same = true, loud = false;
  float f[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (edge) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int lim = ri.there[n][c] ? ri.pos[n][c] - p0 : -1, low = window > 0 ? ri.pos[n][c] - window + 1 - p0 : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int tok = 16 * (g >> 1) + (g & 1) + 4 * i + 2 * x;
            if (tok < low || tok > lim) s[i][n][2 * x + c] = -INFINITY;
          }
      }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      f[n][c] = score_factor(qs[n][c], kscale);
      float m = s[0][n][c];
#pragma unroll
      for (int i = 0; i < 4; ++i) m = fmaxf(m, fmaxf(s[i][n][c], s[i][n][2 + c]));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
      m = fmaxf(m * f[n][c], st.mx[n][c]);               // the factor is positive
      const float b = m == -INFINITY ? 0.f : m;          // nothing seen yet: every weight is 2^-inf = 0
      a[n][c] = exp2_fast(st.mx[n][c] - b);
      same &= st.mx[n][c] == m;
      loud |= too_loud_to_lift(m);
      st.mx[n][c] = m;
    }
  }
  loud = __any_sync(0xffffffffu, loud);
  const float lift = loud ? 0.f : ATTN_LIFT;
  unlift = loud ? 1.f : ATTN_UNLIFT;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float b = st.mx[n][c] == -INFINITY ? lift : lift - st.mx[n][c];
      float l = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float e = exp2_fast(fmaf(s[i][n][2 * x + c], f[n][c], b));
          s[i][n][2 * x + c] = e;
          l += e;
        }
      st.l[n][c] = fmaf(st.l[n][c], a[n][c], l * unlift);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i][n][0] = pack_half2(s[i][n][0], s[i][n][1]);
      p[i][n][1] = pack_half2(s[i][n][2], s[i][n][3]);
    }
  }
  moved = !__all_sync(0xffffffffu, same);
}

// o = o * a + vscale * V^T P^T; vs: the page's v [D][64] in shared memory. edge: some row does not see some token. Tokens
// outside [lo, hi], what any row sees, may hold anything: their codes count as zero. Inside, a token that only some rows
// see may hold NaN, which must not reach the others through 0 * NaN: its code counts as zero too, and true is returned.
// One body for both kinds of page: a second one would have to come through the instruction cache at every unit's end.
template <int D, int NT>
__device__ __forceinline__ bool page_pv(TileState<D, NT>& st, const uint32_t (&p)[4][NT][2], uint32_t vs, const float (&a)[NT][2], bool moved, float vscale,
                                        bool edge, int lo, int hi) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint32_t b[4][NT][2], nan = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      b[i][n][0] = transpose_8x8(p[i][n][0]);
      b[i][n][1] = transpose_8x8(p[i][n][1]);
    }
  uint32_t keep[4];   // bytes of the lane's tokens that some row sees
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    keep[i] = 0xffffffffu;
    if (edge) {
      const int from = max(lo - (16 * t + 4 * i), 0), to = min(hi - (16 * t + 4 * i), 3);
      keep[i] = from > 3 || to < from ? 0u : (0xffffffffu << (8 * from)) & (0xffffffffu >> (8 * (3 - to)));
    }
  }
  if (moved) {
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        st.o[d][n][0] *= a[n][0];
        st.o[d][n][1] *= a[n][1];
        st.o[d][n][2] *= a[n][0];
        st.o[d][n][3] *= a[n][1];
      }
  }
#pragma unroll
  for (int d = 0; d < D / 16; ++d) {
    const uint4 x = lds16(vs + static_cast<uint32_t>(16 * d + g) * ATTN_PAGE + 16 * t), y = lds16(vs + static_cast<uint32_t>(16 * d + 8 + g) * ATTN_PAGE + 16 * t);
    uint32_t u[4] = {x.x, x.y, x.z, x.w}, v[4] = {y.x, y.y, y.z, y.w};
    float c[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.f;
    if (edge) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        auto tame = [&](uint32_t w) {   // code 0x7f or 0xff: NaN
          w &= keep[i];
          const uint32_t bad = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
          nan |= bad;
          return w & ~((bad >> 7) * 0xffu);
        };
        u[i] = tame(u[i]);
        v[i] = tame(v[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a0 = fp8_to_half2(static_cast<uint16_t>(u[i] & 0xffffu)), a2 = fp8_to_half2(static_cast<uint16_t>(u[i] >> 16));
      const uint32_t a1 = fp8_to_half2(static_cast<uint16_t>(v[i] & 0xffffu)), a3 = fp8_to_half2(static_cast<uint16_t>(v[i] >> 16));
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_f16_16816(c[n], a0, a1, a2, a3, b[i][n][0], b[i][n][1]);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) st.o[d][n][k] = fmaf(c[n][k], vscale, st.o[d][n][k]);
  }
  return edge && __any_sync(0xffffffffu, nan != 0);
}

// The rows that see a NaN token of an edge page become NaN in its dimension.
template <int D, int NT>
__device__ __forceinline__ void page_nan(TileState<D, NT>& st, uint32_t vs, const RowInfo<NT>& ri, int p0, int window) {
  const int g = (threadIdx.x & 31) >> 2;
#pragma unroll 1
  for (int tok = 0; tok < ATTN_PAGE; ++tok) {
    bool sees[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c)
        sees[n][c] = ri.there[n][c] && p0 + tok <= ri.pos[n][c] && (window <= 0 || p0 + tok > ri.pos[n][c] - window);
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint32_t code;
        asm volatile("ld.shared.u8 %0, [%1];" : "=r"(code) : "r"(vs + static_cast<uint32_t>(16 * d + 8 * x + g) * ATTN_PAGE + tok));
        if ((code & 0x7fu) == 0x7fu) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c)
              if (sees[n][c]) st.o[d][n][2 * x + c] = __uint_as_float(0x7fffffffu);
        }
      }
  }
}

// Output values of accumulator quads o[d] (rows row, row + 1 of the entry's tile, dimensions 16 d + g and + 8 of a head).
template <int N>
__device__ __forceinline__ void store_quads(const AttnArgs& a, const AttnEntry& en, int h, int row, int d0, const float (&o)[N][4], const float (&inv)[2],
                                            int D) {
  size_t tok[2];
  int col[2];
  unsigned short gt[2][N][2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {   // the gates of both rows are in flight before the first is used
    const int rr = en.row0 + min(row + c, en.rows - 1), tk = div_group(a, rr);
    tok[c] = en.first + tk;
    col[c] = (h * a.group + rr - tk * a.group) * D + d0;
    if (a.gate) {
      const unsigned short* g = reinterpret_cast<const unsigned short*>(a.gate + tok[c] * a.ld_gate + col[c]);
#pragma unroll
      for (int d = 0; d < N; ++d) {
        gt[c][d][0] = __ldcg(g + 16 * d);
        gt[c][d][1] = __ldcg(g + 16 * d + 8);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    if (row + c >= en.rows) continue;
    __nv_bfloat16* dst = a.out + tok[c] * a.ld_out + col[c];
#pragma unroll
    for (int d = 0; d < N; ++d) {
      float x = o[d][c] * inv[c], y = o[d][2 + c] * inv[c];
      if (a.gate) {
        x *= sigmoid_f32(bf16lo_f32(gt[c][d][0]));
        y *= sigmoid_f32(bf16lo_f32(gt[c][d][1]));
      }
      dst[16 * d] = __float2bfloat16_rn(x);
      dst[16 * d + 8] = __float2bfloat16_rn(y);
    }
  }
}

constexpr int STAGE_LD = 68;   // floats of a staged row of 64 dimensions: rows four banks apart
// A finished segment of a unit: the output rows themselves when it is the whole unit, else a partial slot.
template <int D, int NT>
__device__ __forceinline__ void tile_store(TileState<D, NT>& st, const AttnArgs& a, const AttnEntry& en, int h, bool whole, float* slot,
                                           float* stage) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float l[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      l[c] = st.l[n][c];
      l[c] += __shfl_xor_sync(0xffffffffu, l[c], 4);
      l[c] += __shfl_xor_sync(0xffffffffu, l[c], 8);
      l[c] += __shfl_xor_sync(0xffffffffu, l[c], 16);
    }
    const int row = 8 * n + 2 * t;
    if (8 * n >= en.rows) continue;   // warp-uniform
    if (whole) {
      const float inv[2] = {l[0] == 0.f ? 0.f : 1.f / l[0], l[1] == 0.f ? 0.f : 1.f / l[1]};   // no token seen: the row is zero
      // Through shared memory, 64 dimensions at a time, and out in a loop: written out for every accumulator these lines
      // were 10 KB of code that each unit's end had to bring in (6 us of a busy batch; this is 1).
#pragma unroll
      for (int half = 0; half < D / 64; ++half) {
        __syncwarp();
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            stage[(2 * t + (k & 1)) * STAGE_LD + 16 * d + 8 * (k >> 1) + g] = st.o[4 * half + d][n][k] * inv[k & 1];
        __syncwarp();
        const int here = min(8, en.rows - 8 * n);
#pragma unroll 1
        for (int it = lane; it < here * 8; it += 32) {
          const int r = it >> 3, c = (it & 7) * 8, rr = en.row0 + 8 * n + r, tk = div_group(a, rr);
          const size_t tok = en.first + tk;
          const int col = (h * a.group + rr - tk * a.group) * D + 64 * half + c;
          const float4 lo = *reinterpret_cast<const float4*>(stage + r * STAGE_LD + c), hi = *reinterpret_cast<const float4*>(stage + r * STAGE_LD + c + 4);
          float x[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
          store8(a, tok, col, x);
        }
      }
    } else {
      if (g == 0) {
        *reinterpret_cast<float2*>(slot + row) = make_float2(st.mx[n][0], st.mx[n][1]);
        *reinterpret_cast<float2*>(slot + 8 * NT + row) = make_float2(l[0], l[1]);
      }
      float4* o = reinterpret_cast<float4*>(slot + 2 * 8 * NT) + static_cast<size_t>(n) * (D / 16) * 32 + lane;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) o[d * 32] = make_float4(st.o[d][n][0], st.o[d][n][1], st.o[d][n][2], st.o[d][n][3]);
    }
  }
}

// Adds up the slots of a CTA's warps (`stride` floats apart in shared memory) into one: a warp per 16 dimensions (D = 64:
// half the warps) and 8 rows at a time, lanes as the accumulators lie.
template <int D, int NT>
__device__ __forceinline__ void merge_slots(const float* slots, int stride, float* out) {
  constexpr int TILE = 8 * NT;
  const int d = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (d >= D / 16) return;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int row = 8 * n + 2 * t;
    float2 mx = make_float2(-INFINITY, -INFINITY), m[ATTN_WARPS];
#pragma unroll
    for (int w = 0; w < ATTN_WARPS; ++w) {
      m[w] = *reinterpret_cast<const float2*>(slots + static_cast<size_t>(w) * stride + row);
      mx.x = fmaxf(mx.x, m[w].x);
      mx.y = fmaxf(mx.y, m[w].y);
    }
    const float b0 = mx.x == -INFINITY ? 0.f : mx.x, b1 = mx.y == -INFINITY ? 0.f : mx.y;
    float2 l = make_float2(0.f, 0.f);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < ATTN_WARPS; ++w) {
      const float* s = slots + static_cast<size_t>(w) * stride;
      const float2 k = *reinterpret_cast<const float2*>(s + TILE + row);
      const float4 x = reinterpret_cast<const float4*>(s + 2 * TILE)[(n * (D / 16) + d) * 32 + lane];
      const float f0 = exp2_fast(m[w].x - b0), f1 = exp2_fast(m[w].y - b1);
      l.x = fmaf(k.x, f0, l.x);
      l.y = fmaf(k.y, f1, l.y);
      o.x = fmaf(x.x, f0, o.x);
      o.y = fmaf(x.y, f1, o.y);
      o.z = fmaf(x.z, f0, o.z);
      o.w = fmaf(x.w, f1, o.w);
    }
    if (d == 0 && g == 0) {
      *reinterpret_cast<float2*>(out + row) = mx;
      *reinterpret_cast<float2*>(out + TILE + row) = l;
    }
    reinterpret_cast<float4*>(out + 2 * TILE)[(n * (D / 16) + d) * 32 + lane] = o;
  }
}

// Every warp is a worker of 8 NT rows.
template <int D, int NT>
__global__ void __launch_bounds__(ATTN_THREADS, 1) cache_attn_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int TILE = 8 * NT;
  constexpr int SLOTS = attn_slots(D);   // ring slots of a warp
  constexpr uint32_t SLOT_BYTES = ATTN_PAGE * D;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bar_full[attn_slots(D) * ATTN_WARPS];
  __shared__ int s_sum[ATTN_WARPS];
  __shared__ int s_entry[ATTN_WARPS];
  __shared__ int s_start[ATTN_WARPS];
  __shared__ __align__(16) float s_stage[ATTN_WARPS][8 * STAGE_LD];   // rows on their way out
  __shared__ int2 s_rec[ATTN_WARPS][64];   // looked-up pages: tile index in the pool, exponents (k | v << 8)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = a.hq / a.hk, entries = a.batch * a.tiles;
  uint64_t* const full = bar_full + warp * attn_slots(D);
  const uint32_t ring_base = smem_u32(smem) + static_cast<uint32_t>(warp) * attn_slots(D) * SLOT_BYTES;
  if (tid < attn_slots(D) * ATTN_WARPS) {
    mbar_init(smem_u32(&bar_full[tid]), 1);
    fence_mbar_init();
  }
  griddep_wait();
  // Only now: the kernel that adds up, when it comes in, may then take what was ready before this one as ready.
  griddep_launch_dependents();

  // The list: every thread adds up the items of its share of the entries, a scan over the CTA gives the total and where
  // each share begins; the thread whose share holds a worker's first item finds the entry.
  const int per = (entries + ATTN_THREADS - 1) / ATTN_THREADS;
  const int e0 = min(tid * per, entries), e1 = min(e0 + per, entries);
  int mine = 0;
  auto items_of = [&](int e) { return attn_items(attn_entry_of(a, e, group, TILE)) * a.hk; };
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
  __syncthreads();
  int base = 0, total = 0;
  for (int w = 0; w < ATTN_WARPS; ++w) {
    if (w < warp) base += s_sum[w];
    total += s_sum[w];
  }
  const int begin = base + incl - mine, end = base + incl;   // this thread's share of the list
  const AttnDeal deal = attn_deal(total, static_cast<int>(gridDim.x * ATTN_WARPS));
  // Neighbouring workers are a CTA's warps, so that sums of a long unit meet on chip; a list with few items is spread over
  // the SMs instead.
  const bool spread = total <= attn_spread_below(static_cast<int>(gridDim.x));
  auto worker_of = [&](int w) { return static_cast<int>(spread ? w * gridDim.x + blockIdx.x : blockIdx.x * ATTN_WARPS + w); };
  if (total > 0) {
    for (int w = 0; w < ATTN_WARPS; ++w) {
      if (worker_of(w) >= deal.workers) break;
      const int f = attn_range(deal, worker_of(w));
      if (f >= begin && f < end) {
        int at = begin;
        int e = e0;
        for (; e + 1 < e1; ++e) {
          const int next = at + items_of(e);
          if (f < next) break;
          at = next;
        }
        s_entry[w] = e;
        s_start[w] = at;
      }
    }
    if (blockIdx.x == 0) {   // for the kernel that adds up the partial sums
      int at = begin;
      for (int e = e0; e < e1; ++e) {
        a.prefix[e] = at;
        if (e + 1 < e1) at += items_of(e);
      }
    }
  }
  if (blockIdx.x == 0 && tid == 0) a.prefix[entries] = total;
  __syncthreads();
  const int worker = worker_of(warp);
  if (worker >= deal.workers) return;   // no item, and no warp waits for this one (a merging CTA's all have some)
  const int f0 = attn_range(deal, worker), items = attn_range(deal, worker + 1) - f0;

  EntryCache rd_cache, fill_cache;
  rd_cache.base = fill_cache.base = -64;
  Cursor rd, fill;   // where the warp computes, and up to where it has looked up pages
  int unit0;         // first item of the unit that rd stands in
  {
    fill.e = s_entry[warp];
    fill.en = attn_entry_cached(a, fill_cache, fill.e, entries, group, TILE);
    const int off = f0 - s_start[warp], per_unit = attn_items(fill.en);
    fill.h = off / per_unit;
    fill.i = off % per_unit - ATTN_HEAD;
    unit0 = s_start[warp] + fill.h * per_unit;
    rd_cache = fill_cache;
    rd = fill;
  }
  auto next_unit = [&](Cursor& c, EntryCache& ec) {   // false behind the last entry
    c.i = -ATTN_HEAD;
    if (++c.h < a.hk) return true;
    c.h = 0;
    do {
      if (++c.e >= entries) return false;
      c.en = attn_entry_cached(a, ec, c.e, entries, group, TILE);
    } while (c.en.pages == 0);
    return true;
  };
  // Looks up the next pages of the worker's range, up to 32, a page per lane: the tile's index in the pool (page * hk +
  // head; -1: not a page of the pool, or nothing is seen) and its two exponents, into the warp's ring of records.
  int filled = 0, fill_left = items;   // pages looked up; items of the range not yet walked
  int pend_at = 0, pend_tile = -2;     // the lane's page of the last look-up
  auto look_up = [&]() {
    int b = -1, h = 0, i = 0, off = 0;
    while (off < 32 && fill_left > 0) {
      if (fill.i < 0) {   // the unit's head items
        ++fill.i;
        --fill_left;
        continue;
      }
      const int take = min(min(fill.en.pages - fill.i, 32 - off), fill_left);
      if (lane >= off && lane < off + take) {
        b = fill.en.last < 0 ? -1 : fill.e / a.tiles;
        h = fill.h;
        i = fill.en.page0 + fill.i + lane - off;
      }
      off += take;
      fill.i += take;
      fill_left -= take;
      if (fill.i == fill.en.pages && !next_unit(fill, fill_cache)) break;
    }
    int tile = -1;
    if (b >= 0) {
      const int p = __ldcg(a.page_table + static_cast<size_t>(b) * a.width + i);
      if (p >= 0 && p < a.pages) tile = p * a.hk + h;
      else atomicOr(a.status, ST_BAD_PAGE);
    }
    if (lane < off) s_rec[warp][(filled + lane) & 63].x = tile;
    __syncwarp();
    pend_at = filled + lane;
    pend_tile = lane < off ? tile : -2;
    filled += off;
  };
  // The second half of a look-up: the exponents, needed only once the page's copy has landed.
  auto look_up_exponents = [&]() {
    int e = 127 | 127 << 8;
    if (pend_tile >= 0) e = __ldcg(a.k_exp + pend_tile) | __ldcg(a.v_exp + pend_tile) << 8;
    if (pend_tile > -2) s_rec[warp][pend_at & 63].y = e;
    __syncwarp();
  };

  int issued = 0, used = 0;               // halves (K, then V of a page) requested and consumed by this worker
  // Requests the next half.
  auto request = [&]() {
    const int slot = issued % SLOTS;
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
  // Fills the slots that are free.
  auto pump = [&]() {
    while (issued < used + SLOTS && (issued >> 1) < filled) request();
  };

  TileState<D, NT> st;
  uint32_t qf[NT][D / 16][2];
  float qs[NT][2];
  RowInfo<NT> ri;
  float* const stage = s_stage[warp];
  // All eight warps inside one unit: their sums meet in shared memory, and one slot leaves the CTA.
  const int w_first = worker - warp;
  const bool merge = !spread && attn_merged(deal, w_first, ATTN_WARPS, unit0 + ATTN_HEAD, unit0 + attn_items(rd.en));   // CTA-uniform
  bool fresh = true, gave_up = false;
  int seg_first = 0, left = items, n = 0;           // first page of the segment; items to go; pages done
  while (left > 0) {
    if (rd.i < 0) {   // the unit's head items
      ++rd.i;
      --left;
      continue;
    }
    const int my_rows = rd.en.rows;
    // Pages are looked up 32 at a time, while the records of those under way stay (the ring of records holds 64); their
    // copies are asked for before their exponents.
    const bool look = fill_left > 0 && filled - n <= SLOTS / 2 + 2;
    if (look) look_up();
    pump();
    if (look) look_up_exponents();
    if (fresh) {
      tile_reset(st);
      const int r0 = rd.en.row0, t = lane & 3;
      load_q<D, NT>(a, rd.en, rd.h, r0, my_rows, qf, qs);
      if (a.gate && (lane & 3) == 0 && (lane >> 2) < my_rows) {   // on its way to L2 while the pages are worked on
#pragma unroll
        for (int k = 0; k < NT; ++k) {
          const int rr = r0 + 8 * k + (lane >> 2), tk = div_group(a, rr);
          if (8 * k + (lane >> 2) < my_rows)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(a.gate + (rd.en.first + tk) * a.ld_gate + static_cast<size_t>(rd.h * a.group + rr - tk * a.group) * D));
        }
      }
#pragma unroll
      for (int k = 0; k < NT; ++k)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          ri.there[k][c] = 8 * k + 2 * t + c < my_rows;
          ri.pos[k][c] = rd.en.pos + div_group(a, r0 + 8 * k + 2 * t + c);
        }
      ri.first = rd.en.pos + div_group(a, r0);
      ri.last = rd.en.pos + div_group(a, r0 + max(my_rows, 1) - 1);
      fresh = false;
      seg_first = rd.i;
    }
    const int2 rec = s_rec[warp][n & 63];
    const bool live = rec.x >= 0;
    const int p0 = (rd.en.page0 + rd.i) * ATTN_PAGE;
    // some row does not see some token of the page (positions grow with the row)
    const bool edge = ri.first < p0 + ATTN_PAGE - 1 || (a.window > 0 && ri.last - a.window + 1 > p0);
    const int ks = used % SLOTS, vsl = (used + 1) % SLOTS, vt = (used + 1) / SLOTS;
    bool ok = mbar_wait_short(smem_u32(&full[ks]), (used / SLOTS) & 1), moved = false;
    float s[4][NT][4], al[NT][2], unlift = 1.f;
    uint32_t p[4][NT][2];
    if (ok && live) page_scores<D, NT>(s, qf, ring_base + static_cast<uint32_t>(ks) * SLOT_BYTES);
    __syncwarp();
    ++used;   // the K slot may be filled again
    pump();
    if (ok && live) page_softmax<D, NT>(st, s, p, al, moved, unlift, qs, exp2_byte(rec.y & 255), ri, p0, a.window, edge);
    ok = ok && mbar_wait_short(smem_u32(&full[vsl]), vt & 1);
    if (!ok) {
      gave_up = true;
      break;
    }
    if (live) {
      const uint32_t vs = ring_base + static_cast<uint32_t>(vsl) * SLOT_BYTES;
      const float vscale = exp2_byte(rec.y >> 8) * unlift;
      if (page_pv<D, NT>(st, p, vs, al, moved, vscale, edge, a.window > 0 ? ri.first - a.window + 1 - p0 : 0, ri.last - p0))
        page_nan<D, NT>(st, vs, ri, p0, a.window);
    }
    __syncwarp();
    ++used;
    ++n;
    --left;
    // end of the unit or of the range: the segment [seg_first, rd.i] is done
    const bool unit_end = rd.i == rd.en.pages - 1;
    if (unit_end || left == 0) {
      const bool whole = unit_end && seg_first == 0;
      // (a warp's ring is idle by now when it merges: its range ends with this segment)
      float* slot = merge ? reinterpret_cast<float*>(smem) + static_cast<size_t>(warp) * attn_slots(D) * SLOT_BYTES / 4
                          : a.part + static_cast<size_t>(attn_slot_of(deal, worker, unit0 + ATTN_HEAD)) * attn_slot_floats(D, TILE);
      tile_store<D, NT>(st, a, rd.en, rd.h, whole && !merge, slot, stage);
      fresh = true;
    }
    if (left > 0) {
      if (unit_end) {
        unit0 += attn_items(rd.en);
        next_unit(rd, rd_cache);
      } else {
        ++rd.i;
      }
    }
  }
  if (gave_up) {
    if (lane == 0) atomicOr(a.status, ST_ATTN_TIMEOUT);
    // leave no copy in flight behind: each slot's last request is waited for (bounded)
    for (int i = issued > SLOTS ? issued - SLOTS : 0; i < issued; ++i) mbar_wait(smem_u32(&full[i % SLOTS]), (i / SLOTS) & 1);
  }
  if (merge) {
    __syncthreads();   // every warp of the CTA comes here, also one that gave up
    merge_slots<D, NT>(reinterpret_cast<const float*>(smem), attn_slots(D) * SLOT_BYTES / 4, a.part + static_cast<size_t>(2 * w_first) * attn_slot_floats(D, TILE));
  }
}

// Adds up the partial sums of the units that were split between workers, in a fixed order (the same bits in every run).
// Lanes as the accumulators lie: a warp has 8 rows and 16 dimensions of a unit. DEEP (few units, many parts each): a CTA's
// eight warps take every eighth part of the same 16 dimensions and meet in shared memory; else a warp takes all parts.
template <int D, int TILE, bool DEEP>
__global__ void __launch_bounds__(DEEP ? 256 : D * 2) cache_attn_join_kernel(const __grid_constant__ AttnArgs a, int workers, int spread_below) {
  constexpr int STEP = DEEP ? 8 : 1, FLOATS = attn_slot_floats(D, TILE);
  __shared__ float4 s_ml[STEP][32], s_o[STEP][32];
  const int entries = a.batch * a.tiles, group = a.group;
  const int e = static_cast<int>(blockIdx.x) / a.hk, h = static_cast<int>(blockIdx.x) % a.hk;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int r0 = static_cast<int>(blockIdx.y) * 8, d = DEEP ? static_cast<int>(blockIdx.z) : warp;
  // Ready before the kernel ahead began to launch this one: the index tensors (and the gate).
  const AttnEntry en = attn_entry_of(a, e, group, TILE);
  griddep_launch_dependents();
  griddep_wait();
  const int total = __ldcg(a.prefix + entries), start = __ldcg(a.prefix + e);
  if (r0 >= en.rows) return;
  const AttnDeal deal = attn_deal(total, workers);
  const int u0 = start + h * attn_items(en) + ATTN_HEAD;
  if (attn_worker(deal, u0) == attn_worker(deal, u0 + en.pages - 1)) return;   // one worker had all of the unit's pages and has written it
  const AttnParts ps = attn_parts(deal, total <= spread_below ? 1 : ATTN_WARPS, u0, en.pages);
  // The lane's two rows and where its quad of sums lies in a part.
  const int row = r0 + 2 * t;
  const size_t quad_at = 2 * TILE + (static_cast<size_t>(r0 / 8) * (D / 16) + d) * 128 + lane * 4;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[4] = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](const float2& pm, const float2& pl, const float4& po) {   // one more part, or a warp's sums
    const float m0 = fmaxf(m[0], pm.x), m1 = fmaxf(m[1], pm.y);
    const float b0 = m0 == -INFINITY ? 0.f : m0, b1 = m1 == -INFINITY ? 0.f : m1;
    const float f0 = exp2_fast(m[0] - b0), f1 = exp2_fast(m[1] - b1), k0 = exp2_fast(pm.x - b0), k1 = exp2_fast(pm.y - b1);
    l[0] = fmaf(l[0], f0, pl.x * k0);
    l[1] = fmaf(l[1], f1, pl.y * k1);
    o[0] = fmaf(o[0], f0, po.x * k0);
    o[1] = fmaf(o[1], f1, po.y * k1);
    o[2] = fmaf(o[2], f0, po.z * k0);
    o[3] = fmaf(o[3], f1, po.w * k1);
    m[0] = m0;
    m[1] = m1;
  };
  constexpr int AHEAD = 4;
  for (int i = DEEP ? warp : 0; i < ps.parts; i += STEP * AHEAD) {
    float2 pm[AHEAD], pl[AHEAD];
    float4 po[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int j = i + k * STEP;
      if (j < ps.parts) {
        const float* s = a.part + static_cast<size_t>(attn_part_slot(ps, j)) * FLOATS;
        pm[k] = __ldcg(reinterpret_cast<const float2*>(s + row));
        pl[k] = __ldcg(reinterpret_cast<const float2*>(s + TILE + row));
        po[k] = __ldcg(reinterpret_cast<const float4*>(s + quad_at));
      }
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (i + k * STEP < ps.parts) add(pm[k], pl[k], po[k]);
  }
  if constexpr (DEEP) {
    s_ml[warp][lane] = make_float4(m[0], m[1], l[0], l[1]);
    s_o[warp][lane] = make_float4(o[0], o[1], o[2], o[3]);
    __syncthreads();
    if (warp > 0) return;
#pragma unroll
    for (int w = 1; w < 8; ++w) {
      const float4 x = s_ml[w][lane];
      add(make_float2(x.x, x.y), make_float2(x.z, x.w), s_o[w][lane]);
    }
  }
  const float inv[2] = {l[0] == 0.f ? 0.f : 1.f / l[0], l[1] == 0.f ? 0.f : 1.f / l[1]};
  const float quad[1][4] = {{o[0], o[1], o[2], o[3]}};
  store_quads<1>(a, en, h, row, 16 * d + g, quad, inv, D);
}

// The same for tiles of 128 rows, which are kept by rows: a thread has four neighbouring dimensions of GROUPS rows, 8 apart.
// Where most units are split (a chunk of 2 x 512 tokens: 147 of 256), GROUPS = 4 is what gets the latency of a CTA's
// chain of loads paid once for 32 rows.
template <int D, int GROUPS>
__global__ void __launch_bounds__(D * 2) cache_attn_join_rows_kernel(const __grid_constant__ AttnArgs a, int workers) {
  constexpr int TILE = 128, FLOATS = attn_slot_floats(D, TILE);
  const int entries = a.batch * a.tiles, group = a.group;
  const int e = static_cast<int>(blockIdx.x) / a.hk, h = static_cast<int>(blockIdx.x) % a.hk;
  const int row = static_cast<int>(blockIdx.y) * 8 * GROUPS + static_cast<int>(threadIdx.x) / (D / 4), dim = 4 * (static_cast<int>(threadIdx.x) % (D / 4));
  const AttnEntry en = attn_entry_of(a, e, group, TILE);
  griddep_launch_dependents();
  griddep_wait();
  const int total = __ldcg(a.prefix + entries), start = __ldcg(a.prefix + e);
  if (row >= en.rows) return;
  const AttnDeal deal = attn_deal(total, workers);
  const int u0 = start + h * attn_items(en) + ATTN_HEAD;
  if (attn_worker(deal, u0) == attn_worker(deal, u0 + en.pages - 1)) return;
  const AttnParts ps = attn_parts(deal, 1, u0, en.pages);
  float m[GROUPS], l[GROUPS], o[GROUPS][4];
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    m[g] = -INFINITY;
    l[g] = o[g][0] = o[g][1] = o[g][2] = o[g][3] = 0.f;
  }
  constexpr int AHEAD = GROUPS > 1 ? 2 : 4;
  for (int i = 0; i < ps.parts; i += AHEAD) {
    float pm[AHEAD][GROUPS], pl[AHEAD][GROUPS];
    float4 po[AHEAD][GROUPS];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (i + k >= ps.parts) break;
      const float* s = a.part + static_cast<size_t>(attn_part_slot(ps, i + k)) * FLOATS;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {   // (a slot has all 128 rows: those behind the tile's last hold what was there)
        pm[k][g] = __ldcg(s + row + 8 * g);
        pl[k][g] = __ldcg(s + TILE + row + 8 * g);
        po[k][g] = __ldcg(reinterpret_cast<const float4*>(s + 2 * TILE + static_cast<size_t>(row + 8 * g) * D + dim));
      }
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (i + k >= ps.parts) break;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        const float top = fmaxf(m[g], pm[k][g]), base = top == -INFINITY ? 0.f : top, f = exp2_fast(m[g] - base), p = exp2_fast(pm[k][g] - base);
        m[g] = top;
        l[g] = fmaf(l[g], f, pl[k][g] * p);
        o[g][0] = fmaf(o[g][0], f, po[k][g].x * p);
        o[g][1] = fmaf(o[g][1], f, po[k][g].y * p);
        o[g][2] = fmaf(o[g][2], f, po[k][g].z * p);
        o[g][3] = fmaf(o[g][3], f, po[k][g].w * p);
      }
    }
  }
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    if (row + 8 * g >= en.rows) break;
    const float inv = l[g] == 0.f ? 0.f : 1.f / l[g];
    const int rr = en.row0 + row + 8 * g, tk = div_group(a, rr), col = (h * group + rr - tk * group) * D + dim;
    const size_t tok = en.first + tk;
    __nv_bfloat16* out = a.out + tok * a.ld_out + col;
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = o[g][i] * inv;
      if (a.gate) x[i] *= sigmoid_f32(bf16lo_f32(__ldcg(reinterpret_cast<const unsigned short*>(a.gate + tok * a.ld_gate + col + i))));
    }
    if (a.vec_out) {
      const __nv_bfloat162 lo = __floats2bfloat162_rn(x[0], x[1]), hi = __floats2bfloat162_rn(x[2], x[3]);
      *reinterpret_cast<uint2*>(out) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i] = __float2bfloat16_rn(x[i]);
    }
  }
}

// ---------------------------------------------------------------- host side
// The form a call takes goes by the rows a KV head has at most: 8 or 16 per warp, or (cache_attn_tc.cu) 128 per CTA.
struct AttnForm {
  bool shared;
  int tile, tiles;
  int workers(int sms) const { return shared ? sms : sms * ATTN_WARPS; }
};
static AttnForm attn_form(int max_q, int hq, int hk) {
  const long long rows = static_cast<long long>(max_q) * (hq / hk);
  AttnForm f;
  f.shared = rows > 16;
  f.tile = f.shared ? 128 : rows > 8 ? 16 : 8;
  f.tiles = static_cast<int>((rows + f.tile - 1) / f.tile);
  return f;
}

long long cache_attn_ws_bytes(int batch, int max_q, int hq, int hk, int dim) {
  const int sms = device_sms();
  if (batch < 1 || max_q < 1 || hk < 1 || hq < hk || hq % hk || (dim != 64 && dim != 128) || sms < 1) return -1;
  const AttnForm f = attn_form(max_q, hq, hk);
  return 2ll * f.workers(sms) * attn_slot_floats(dim, f.tile) * 4 + (static_cast<long long>(batch) * f.tiles + 1) * 4;
}

template <int D, int NT>
static cudaError_t attn_launch(const AttnArgs& a, int sms, cudaStream_t stream) {
  const size_t smem = attn_ring_bytes(D);
  static DeviceOnce once;
  const cudaError_t e = once.run([&] { return cudaFuncSetAttribute(cache_attn_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)); });
  if (e != cudaSuccess) return e;
  return launch_dependent(cache_attn_kernel<D, NT>, dim3(sms), dim3(ATTN_THREADS), smem, stream, a);
}

template <int D, int TILE>
static cudaError_t join_launch(const AttnArgs& a, const AttnForm& f, int sms, cudaStream_t stream) {
  const int all = a.max_q * a.group, rows = all < f.tile ? all : f.tile;
  const unsigned units = static_cast<unsigned>(a.batch) * a.tiles * a.hk, groups = (rows + 7) / 8;
  // Few units may have many parts each; many units have few (there are two partial segments per worker in all).
  const bool few = static_cast<long long>(units) * groups < 2ll * sms;
  if constexpr (TILE == 128) {
    return few ? launch_dependent(cache_attn_join_rows_kernel<D, 1>, dim3(units, groups), dim3(D * 2), 0, stream, a, f.workers(sms))
               : launch_dependent(cache_attn_join_rows_kernel<D, 4>, dim3(units, (groups + 3) / 4), dim3(D * 2), 0, stream, a, f.workers(sms));
  } else {
    return few ? launch_dependent(cache_attn_join_kernel<D, TILE, true>, dim3(units, groups, D / 16), dim3(256), 0, stream, a, f.workers(sms), attn_spread_below(sms))
               : launch_dependent(cache_attn_join_kernel<D, TILE, false>, dim3(units, groups), dim3(D * 2), 0, stream, a, f.workers(sms), attn_spread_below(sms));
  }
}

template <int D>
static cudaError_t both_launch(const AttnArgs& a, const AttnForm& f, int sms, cudaStream_t stream) {
  cudaError_t e = f.shared ? cache_attn_tc_launch(a, D, sms, stream) : f.tile == 16 ? attn_launch<D, 2>(a, sms, stream) : attn_launch<D, 1>(a, sms, stream);
  if (e != cudaSuccess) return e;
  return f.shared ? join_launch<D, 128>(a, f, sms, stream) : f.tile == 16 ? join_launch<D, 16>(a, f, sms, stream) : join_launch<D, 8>(a, f, sms, stream);
}

int cache_attn_dispatch(AttnArgs a, int dim, void* ws, cudaStream_t stream) {
  if (!a.q || !a.k || !a.v || !a.k_exp || !a.v_exp || !a.page_table || !a.seq_lens || !a.out || !a.status || !ws) return -1;
  if (a.m < 1 || a.batch < 1 || a.width < 1 || a.pages < 1 || a.max_q < 1 || a.hk < 1 || a.hq < a.hk || a.hq % a.hk || (dim != 64 && dim != 128)) return -2;
  if (a.width > 0x7fffffff / ATTN_PAGE || a.window < 0 || static_cast<long long>(a.max_q) * (a.hq / a.hk) > 0x3fffffff) return -3;
  if (a.ld_q % 8 || a.ld_q < static_cast<long long>(a.hq) * dim || a.ld_out < static_cast<long long>(a.hq) * dim) return -4;
  if (a.gate && a.ld_gate < static_cast<long long>(a.hq) * dim) return -4;
  if ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(ws)) & 15) return -5;
  if ((reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.gate)) & 1) return -5;
  if (!a.cu_q && (a.max_q != 1 || a.m != a.batch)) return -6;
  if (!(a.scale_log2 > 0.f && a.scale_log2 < INFINITY)) return -6;
  const int sms = device_sms();
  if (sms < 1) return -7;
  const AttnForm f = attn_form(a.max_q, a.hq, a.hk);
  if (a.window >= a.width * ATTN_PAGE) a.window = 0;   // wider than any sequence
  a.tiles = f.tiles;
  a.group = a.hq / a.hk;
  a.vec_gate = a.ld_gate % 8 == 0 && (reinterpret_cast<uintptr_t>(a.gate) & 15) == 0;
  a.vec_out = a.ld_out % 8 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
  a.group_magic = static_cast<uint32_t>((1ull << 32) / static_cast<unsigned>(a.group) + 1);
  if (static_cast<long long>(f.tiles) * f.tile * a.group >= 1ll << 32) return -3;
  // items of the list, at most; and indices of the pool's tiles
  if (static_cast<long long>(a.batch) * a.tiles * a.hk > 0x7fffffffll / (a.width + ATTN_HEAD) || static_cast<long long>(a.pages) * a.hk > 0x7fffffffll) return -3;
  a.part = static_cast<float*>(ws);
  a.prefix = reinterpret_cast<int*>(a.part + 2ll * f.workers(sms) * attn_slot_floats(dim, f.tile));
  const cudaError_t e = dim == 128 ? both_launch<128>(a, f, sms, stream) : both_launch<64>(a, f, sms, stream);
  return static_cast<int>(e);
}

// ---- the same plan on the host
namespace {
struct HostPlan {
  AttnForm form;
  int group, entries;
  int total;
  bool ok;
};
}  // namespace
static HostPlan host_plan(const int* seq_lens, int m, int batch, int width, int max_q, int hq, int hk, int window, int sms) {
  HostPlan p = {};
  p.ok = seq_lens && m >= 1 && batch >= 1 && width >= 1 && width <= 0x7fffffff / ATTN_PAGE && max_q >= 1 && hk >= 1 && hq >= hk && hq % hk == 0 &&
         window >= 0 && sms >= 1;
  if (!p.ok) return p;
  p.form = attn_form(max_q, hq, hk);
  p.group = hq / hk;
  p.entries = batch * p.form.tiles;
  p.ok = static_cast<long long>(p.entries) * hk <= 0x7fffffffll / (width + ATTN_HEAD);
  return p;
}
static AttnEntry host_entry(const HostPlan& p, const int* seq_lens, const int* cu_q, int m, int width, int max_q, int window, int e) {
  const int b = e / p.form.tiles;
  return attn_entry(cu_q ? cu_q[b] : b, cu_q ? cu_q[b + 1] : b + 1, seq_lens[b], m, max_q, width * ATTN_PAGE, p.group, p.form.tile, e % p.form.tiles, window);
}

long long cache_attn_plan(const int* seq_lens, const int* cu_q, int m, int batch, int width, int max_q, int hq, int hk, int window, int sms,
                          int* segments, long long capacity) {
  HostPlan p = host_plan(seq_lens, m, batch, width, max_q, hq, hk, window, sms);
  if (!p.ok || !segments) return -1;
  for (int e = 0; e < p.entries; ++e) p.total += attn_items(host_entry(p, seq_lens, cu_q, m, width, max_q, window, e)) * hk;
  if (p.total == 0) return 0;
  const AttnDeal deal = attn_deal(p.total, p.form.workers(sms));
  long long count = 0;
  int start = 0;
  int e = 0;
  AttnEntry en = host_entry(p, seq_lens, cu_q, m, width, max_q, window, 0);
  for (int w = 0; w < deal.workers; ++w) {
    for (int f = attn_range(deal, w), f1 = attn_range(deal, w + 1); f < f1;) {
      while (f >= start + attn_items(en) * hk) {
        start += attn_items(en) * hk;
        en = host_entry(p, seq_lens, cu_q, m, width, max_q, window, ++e);
      }
      const int off = f - start, h = off / attn_items(en), i = off % attn_items(en) - ATTN_HEAD;
      if (i < 0) {
        ++f;
        continue;
      }
      const int n = f1 - f < en.pages - i ? f1 - f : en.pages - i;
      if (count < capacity) {
        int* s = segments + 6 * count;
        s[0] = w; s[1] = e; s[2] = h; s[3] = en.page0 + i; s[4] = n;
        const int u0 = start + h * attn_items(en) + ATTN_HEAD;
        const int per = p.form.shared || p.total <= attn_spread_below(sms) ? 1 : ATTN_WARPS, first = w - w % per;
        s[5] = n == en.pages ? -1 : attn_merged(deal, first, per, u0, u0 + en.pages) ? 2 * first : attn_slot_of(deal, w, u0);
      }
      ++count;
      f += n;
    }
  }
  return count;
}

long long cache_attn_join(const int* seq_lens, const int* cu_q, int m, int batch, int width, int max_q, int hq, int hk, int window, int sms,
                          int entry, int head, int* slots, long long capacity) {
  HostPlan p = host_plan(seq_lens, m, batch, width, max_q, hq, hk, window, sms);
  if (!p.ok || !slots || entry < 0 || entry >= p.entries || head < 0 || head >= hk) return -1;
  int before = 0;
  for (int e = 0; e < p.entries; ++e) {
    if (e == entry) before = p.total;
    p.total += attn_items(host_entry(p, seq_lens, cu_q, m, width, max_q, window, e)) * hk;
  }
  const AttnEntry en = host_entry(p, seq_lens, cu_q, m, width, max_q, window, entry);
  if (en.rows == 0) return 0;
  const AttnDeal deal = attn_deal(p.total, p.form.workers(sms));
  const int u0 = before + head * attn_items(en) + ATTN_HEAD;
  if (attn_worker(deal, u0) == attn_worker(deal, u0 + en.pages - 1)) return 0;
  const AttnParts ps = attn_parts(deal, p.form.shared || p.total <= attn_spread_below(sms) ? 1 : ATTN_WARPS, u0, en.pages);
  for (int i = 0; i < ps.parts && i < capacity; ++i) slots[i] = attn_part_slot(ps, i);
  return ps.parts;
}

}  // namespace muse
