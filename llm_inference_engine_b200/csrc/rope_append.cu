// Rotary positions on the q and k columns of a projection's rows, and the append of k and v to a paged cache in 8 bits:
// what stands between the qkv_gate projection and the attention. Token j of a sequence with n new tokens and `len`
// tokens in all has position p = len - n + j; a pair (a, b) of its head turns by the position's angle,
//     (a, b) -> (a cos - b sin, b cos + a sin),       pairs (i, i + rot / 2), or (2 i, 2 i + 1) when interleaved,
// over the first `rot` dimensions, in FP32 from a table of cos and sin (one rounding per product and sum, so that the
// codes do not depend on how the compiler contracts them). q leaves in BF16. k and v enter page p / 64 of the sequence:
//     k [page, head, token, dim],  v [page, head, dim, token]  (what the attention's MMAs read without a transpose),
// e4m3 codes with one power-of-two scale per page and head (fp8.cuh). A page's exponent never falls while the page
// fills; when new tokens raise it, the codes of the page's earlier tokens are rounded to the new scale.
//
// Memory-bound: reads the rows once, writes q, the codes and, on request, the values the codes stand for. One CTA per
// (sequence, page that new tokens fall into, head) does k and v: the new tokens stay in registers between the search
// for the largest magnitude and the rounding. The other CTAs rotate q, eight threads per head of 128.
//
// Measured on the device: three prompts of up to 1500 tokens (32 query and 16 KV heads, with the values) 39 us, 3.6 TB/s of what has to move (61 us
// while a CTA took the 64 tokens of a page in four rounds of 64 threads); 32 sequences of one token 3.7 us, 45 with drafts of
// up to 5 4.6 us: those wait for a launch, three loads one after the other (lengths, page table, exponent) and the codes' way back.
#include "cache8.cuh"
#include "fp8.cuh"

namespace muse {

// A sequence's new tokens: rows [first, first + n) of the batch, the first of them at position `pos`.
struct SeqSpan {
  int first, n, pos;
};
__device__ __forceinline__ SeqSpan seq_span(const int* cu_q, const int* seq_lens, int b, int m, int max_q, int capacity, int* status) {
  SeqSpan s;
  const int len = __ldcg(seq_lens + b);
  if (cu_q) {
    const int c0 = __ldcg(cu_q + b), c1 = __ldcg(cu_q + b + 1);
    s.first = min(max(c0, 0), m);
    s.n = max(min(c1, m) - s.first, 0);
    if (c0 < 0 || c1 < c0 || c1 > m || s.n > max_q || len > capacity || len < 0) {
      if (threadIdx.x == 0) atomicOr(status, ST_BAD_LENGTH);
      s.n = min(s.n, max_q);
    }
  } else {
    s.first = b;
    s.n = b < m ? 1 : 0;
    if ((len > capacity || len < 0) && threadIdx.x == 0) atomicOr(status, ST_BAD_LENGTH);
  }
  s.pos = len - s.n;   // a token at a position below zero or beyond the table belongs to no page
  return s;
}

__device__ __forceinline__ void unpack8(uint4 u, float (&f)[8]) {
  f[0] = bf16lo_f32(u.x); f[1] = bf16hi_f32(u.x); f[2] = bf16lo_f32(u.y); f[3] = bf16hi_f32(u.y);
  f[4] = bf16lo_f32(u.z); f[5] = bf16hi_f32(u.z); f[6] = bf16lo_f32(u.w); f[7] = bf16hi_f32(u.w);
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  auto p = [](float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  };
  return make_uint4(p(f[0], f[1]), p(f[2], f[3]), p(f[4], f[5]), p(f[6], f[7]));
}

// Sixteen dimensions of a head as the rotation takes them: unit u < rot / 16 is 8 pairs (dimensions 8 u .. and their
// partners, or 16 neighbours when interleaved), the units behind are 16 neighbours that do not turn.
struct Unit {
  int lo, hi;   // first dimension of each half
  bool turns;
};
__device__ __forceinline__ Unit unit_of(int u, int rot, int interleaved) {
  Unit d;
  d.turns = u < rot / 16;
  d.lo = d.turns && !interleaved ? 8 * u : 16 * u;
  d.hi = d.turns && !interleaved ? rot / 2 + 8 * u : 16 * u + 8;
  return d;
}
// cos and sin of a unit's 8 pairs.
struct Turn {
  float4 w[4];
  __device__ __forceinline__ void load(const float* cs, int u) {
    const float4* t = reinterpret_cast<const float4*>(cs + 16 * u);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __ldg(t + i);   // the table is as static as a weight
  }
  __device__ __forceinline__ void apply(float (&a)[8], float (&b)[8], int interleaved) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float c[2] = {w[i].x, w[i].z}, n[2] = {w[i].y, w[i].w};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int p = 2 * i + j;   // pair p of the unit
        float& x = interleaved ? (p < 4 ? a[(2 * p) & 7] : b[(2 * p) & 7]) : a[p];
        float& y = interleaved ? (p < 4 ? a[(2 * p + 1) & 7] : b[(2 * p + 1) & 7]) : b[p];
        const float x1 = __fsub_rn(__fmul_rn(x, c[j]), __fmul_rn(y, n[j]));
        const float y1 = __fadd_rn(__fmul_rn(y, c[j]), __fmul_rn(x, n[j]));
        x = x1;
        y = y1;
      }
    }
  }
};

__device__ __forceinline__ float block_max(float v, float* s, int threads) {
#pragma unroll
  for (int i = 16; i; i >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, i));
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[0];
  for (int w = 1; w < threads / 32; ++w) v = fmaxf(v, s[w]);
  return v;
}

// Codes [4 bytes] under scale 2^(old - 127) rounded to 2^(now - 127), only the bytes whose bit in `mask` is set.
__device__ __forceinline__ uint32_t recode4(uint32_t w, float ratio, uint32_t mask) {
  const float2 a = fp8_to_float2(static_cast<uint16_t>(w & 0xffffu)), b = fp8_to_float2(static_cast<uint16_t>(w >> 16));
  const uint32_t r = fp8_pack4(a.x * ratio, a.y * ratio, b.x * ratio, b.y * ratio);
  uint32_t keep = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) keep |= (mask >> i & 1u) ? 0u : 0xffu << (8 * i);
  return (w & keep) | (r & ~keep);
}

// THREADS threads, U units per thread and tensor: THREADS * U units of 16 dimensions hold the page's new tokens.
template <int D, int THREADS, int U>
__global__ void __launch_bounds__(THREADS) rope_append_kernel(const __grid_constant__ RopeArgs a, int kv_ctas, int reach, int q_ctas_per_seq) {
  constexpr int UPR = D / 16;   // units per head row
  griddep_launch_dependents();
  griddep_wait();
  const int tid = threadIdx.x;
  const int capacity = a.width * PAGE_TOKENS;
  if (static_cast<int>(blockIdx.x) >= kv_ctas) {   // ---- q
    // A thread turns one unit of up to QH heads of a token, with the unit's 8 pairs of cos and sin in registers.
    constexpr int QH = THREADS > 64 ? 4 : 1;
    const int i = static_cast<int>(blockIdx.x) - kv_ctas, b = i / q_ctas_per_seq;
    const SeqSpan s = seq_span(a.cu_q, a.seq_lens, b, a.m, a.max_q, capacity, a.status);
    const uint32_t hgroups = static_cast<uint32_t>((a.hq + QH - 1) / QH), items = static_cast<uint32_t>(s.n) * hgroups * UPR;
    for (uint32_t it = static_cast<uint32_t>(i % q_ctas_per_seq) * THREADS + tid; it < items; it += static_cast<uint32_t>(q_ctas_per_seq) * THREADS) {
      const uint32_t u = it % UPR, row_g = it / UPR, j = row_g / hgroups, hg = row_g - j * hgroups;
      const int pos = s.pos + static_cast<int>(j), h0 = static_cast<int>(hg) * QH;
      const size_t row = s.first + j;
      const Unit d = unit_of(static_cast<int>(u), a.rot, a.interleaved);
      const bool in = pos >= 0 && pos < capacity;   // a token that is in no page leaves zeros
      const __nv_bfloat16* src = a.qkv + row * a.ld_qkv + static_cast<size_t>(h0) * D;
      __nv_bfloat16* o = a.q_out + (row * a.hq + h0) * D;
      uint4 r0[QH], r1[QH];
#pragma unroll
      for (int h = 0; h < QH; ++h)
        if (in && h0 + h < a.hq) {
          r0[h] = __ldcg(reinterpret_cast<const uint4*>(src + h * D + d.lo));
          r1[h] = __ldcg(reinterpret_cast<const uint4*>(src + h * D + d.hi));
        } else {
          r0[h] = r1[h] = make_uint4(0u, 0u, 0u, 0u);
        }
      Turn turn;
      if (in && d.turns) turn.load(a.cos_sin + static_cast<size_t>(pos) * a.rot, static_cast<int>(u));
#pragma unroll
      for (int h = 0; h < QH; ++h) {
        if (h0 + h >= a.hq) break;
        if (in && d.turns) {
          float x[8], y[8];
          unpack8(r0[h], x);
          unpack8(r1[h], y);
          turn.apply(x, y, a.interleaved);
          r0[h] = pack8(x);
          r1[h] = pack8(y);
        }
        *reinterpret_cast<uint4*>(o + h * D + d.lo) = r0[h];
        *reinterpret_cast<uint4*>(o + h * D + d.hi) = r1[h];
      }
      if (!in && a.k_val) {
        const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
        for (int kh = static_cast<int>(hg); kh < a.hk; kh += static_cast<int>(hgroups)) {
          const size_t at = (row * a.hk + kh) * D;
          *reinterpret_cast<uint4*>(a.k_val + at + d.lo) = zero;
          *reinterpret_cast<uint4*>(a.k_val + at + d.hi) = zero;
          *reinterpret_cast<uint4*>(a.v_val + at + d.lo) = zero;
          *reinterpret_cast<uint4*>(a.v_val + at + d.hi) = zero;
        }
      }
    }
    return;
  }
  // ---- one page of one sequence, one head: k and v
  __shared__ float s_red[2][THREADS / 32];
  __shared__ uint32_t s_t[D][PAGE_TOKENS / 4];   // a full page of v, turned
  const int h = static_cast<int>(blockIdx.x) % a.hk, i = static_cast<int>(blockIdx.x) / a.hk, b = i / reach;
  const SeqSpan s = seq_span(a.cu_q, a.seq_lens, b, a.m, a.max_q, capacity, a.status);
  const int first_pos = max(s.pos, 0), end_pos = min(s.pos + s.n, capacity);
  const int pg = first_pos / PAGE_TOKENS + i % reach;                       // page of the sequence
  const int p0 = max(first_pos, pg * PAGE_TOKENS), p1 = min(end_pos, (pg + 1) * PAGE_TOKENS);
  if (p0 >= p1) return;   // CTA-uniform
  const int slot0 = p0 - pg * PAGE_TOKENS, n = p1 - p0;
  const int page = __ldcg(a.page_table + static_cast<size_t>(b) * a.width + pg);
  if (page < 0 || page >= a.pages) {
    if (tid == 0) atomicOr(a.status, ST_BAD_PAGE);
    if (a.k_val)
      for (int it = tid; it < n * (D / 8); it += THREADS) {
        const size_t at = (static_cast<size_t>(s.first + p0 - s.pos + it / (D / 8)) * a.hk + h) * D + it % (D / 8) * 8;
        *reinterpret_cast<uint4*>(a.k_val + at) = make_uint4(0u, 0u, 0u, 0u);
        *reinterpret_cast<uint4*>(a.v_val + at) = make_uint4(0u, 0u, 0u, 0u);
      }
    return;
  }
  float kx[U][8], ky[U][8], vx[U][8], vy[U][8];
  float kmax = 0.f, vmax = 0.f;
#pragma unroll
  for (int w = 0; w < U; ++w) {
    const int it = tid + w * THREADS;
    if (it < n * UPR) {
      const int u = it % UPR, pos = p0 + it / UPR;
      const Unit d = unit_of(u, a.rot, a.interleaved);
      const __nv_bfloat16* src = a.qkv + static_cast<size_t>(s.first + pos - s.pos) * a.ld_qkv + static_cast<size_t>(a.hq + h) * D;
      const __nv_bfloat16* vsrc = src + static_cast<size_t>(a.hk) * D + 16 * u;
      const uint4 r0 = __ldcg(reinterpret_cast<const uint4*>(src + d.lo)), r1 = __ldcg(reinterpret_cast<const uint4*>(src + d.hi));
      const uint4 r2 = __ldcg(reinterpret_cast<const uint4*>(vsrc)), r3 = __ldcg(reinterpret_cast<const uint4*>(vsrc + 8));
      unpack8(r0, kx[w]); unpack8(r1, ky[w]); unpack8(r2, vx[w]); unpack8(r3, vy[w]);
      if (d.turns) {
        Turn turn;
        turn.load(a.cos_sin + static_cast<size_t>(pos) * a.rot, u);
        turn.apply(kx[w], ky[w], a.interleaved);
      }
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        kmax = fmaxf(kmax, fmaxf(finite_abs(kx[w][c]), finite_abs(ky[w][c])));
        vmax = fmaxf(vmax, fmaxf(finite_abs(vx[w][c]), finite_abs(vy[w][c])));
      }
    }
  }
  kmax = block_max(kmax, s_red[0], THREADS);
  vmax = block_max(vmax, s_red[1], THREADS);
  const size_t ph = static_cast<size_t>(page) * a.hk + h;
  uint8_t* kp = a.k + ph * PAGE_TOKENS * D;
  uint8_t* vp = a.v + ph * PAGE_TOKENS * D;
  int ke = fp8_exponent_byte(kmax), ve = fp8_exponent_byte(vmax);
  if (slot0 > 0) {
    const int ko = __ldcg(a.k_exp + ph), vo = __ldcg(a.v_exp + ph);
    __syncthreads();   // everybody has read the old exponents
    if (ke > ko) {
      const float ratio = ko + 126 < ke ? 0.f : exp2_byte(ko - ke + 127);
      for (int it = tid; it < slot0 * D / 4; it += THREADS) {
        uint32_t* w = reinterpret_cast<uint32_t*>(kp) + it;
        *w = recode4(__ldcg(w), ratio, 15u);
      }
    }
    if (ve > vo) {
      const float ratio = vo + 126 < ve ? 0.f : exp2_byte(vo - ve + 127);
      const int words = (slot0 + 3) / 4;
      for (int it = tid; it < D * words; it += THREADS) {
        const int d = it / words, w4 = it % words, left = slot0 - 4 * w4;
        uint32_t* w = reinterpret_cast<uint32_t*>(vp + d * PAGE_TOKENS) + w4;
        *w = recode4(__ldcg(w), ratio, left >= 4 ? 15u : (1u << left) - 1u);
      }
    }
    ke = max(ke, ko);
    ve = max(ve, vo);
    __syncthreads();   // the earlier tokens' words are written before a new token's bytes go into them
  }
  if (tid == 0) {
    a.k_exp[ph] = static_cast<uint8_t>(ke);
    a.v_exp[ph] = static_cast<uint8_t>(ve);
  }
  const float ki = exp2_byte_inv(ke), vi = exp2_byte_inv(ve), kf = exp2_byte(ke), vf = exp2_byte(ve);
  const bool full = n == PAGE_TOKENS;
#pragma unroll
  for (int w = 0; w < U; ++w) {
    const int it = tid + w * THREADS;
    if (it < n * UPR) {
      const int u = it % UPR, r = it / UPR;
      const Unit d = unit_of(u, a.rot, a.interleaved);
      uint32_t q[8];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        q[c] = fp8_pack4(kx[w][4 * c] * ki, kx[w][4 * c + 1] * ki, kx[w][4 * c + 2] * ki, kx[w][4 * c + 3] * ki);
        q[2 + c] = fp8_pack4(ky[w][4 * c] * ki, ky[w][4 * c + 1] * ki, ky[w][4 * c + 2] * ki, ky[w][4 * c + 3] * ki);
        q[4 + c] = fp8_pack4(vx[w][4 * c] * vi, vx[w][4 * c + 1] * vi, vx[w][4 * c + 2] * vi, vx[w][4 * c + 3] * vi);
        q[6 + c] = fp8_pack4(vy[w][4 * c] * vi, vy[w][4 * c + 1] * vi, vy[w][4 * c + 2] * vi, vy[w][4 * c + 3] * vi);
      }
      uint8_t* kr = kp + static_cast<size_t>(slot0 + r) * D;
      *reinterpret_cast<uint2*>(kr + d.lo) = make_uint2(q[0], q[1]);
      *reinterpret_cast<uint2*>(kr + d.hi) = make_uint2(q[2], q[3]);
      if (!full) {
#pragma unroll
        for (int c = 0; c < 16; ++c) vp[(16 * u + c) * PAGE_TOKENS + slot0 + r] = static_cast<uint8_t>(q[4 + c / 4] >> (8 * (c & 3)));
      } else {
        // A full page fills every thread's units (n UPR = THREADS U or a divisor): the four lanes that hold four
        // neighbouring tokens of the same 16 dimensions swap words, so that each then has four tokens of four dimensions.
        uint32_t m[4];
        const int me = (tid / UPR) & 3;
#pragma unroll
        for (int c = 0; c < 4; ++c) {   // step c: send the word of lane me ^ c, take mine from it
          const int other = me ^ c;
          const uint32_t send = other == 0 ? q[4] : other == 1 ? q[5] : other == 2 ? q[6] : q[7];
          const uint32_t got = __shfl_xor_sync(0xffffffffu, send, c * UPR);
          if (other == 0) m[0] = got;
          if (other == 1) m[1] = got;
          if (other == 2) m[2] = got;
          if (other == 3) m[3] = got;
        }
        const uint32_t a01 = __byte_perm(m[0], m[1], 0x5140), a23 = __byte_perm(m[2], m[3], 0x5140);   // dimensions 0, 1 of tokens 0, 1 / 2, 3
        const uint32_t b01 = __byte_perm(m[0], m[1], 0x7362), b23 = __byte_perm(m[2], m[3], 0x7362);   // dimensions 2, 3
        const uint32_t t4[4] = {__byte_perm(a01, a23, 0x5410), __byte_perm(a01, a23, 0x7632), __byte_perm(b01, b23, 0x5410), __byte_perm(b01, b23, 0x7632)};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int dim = 16 * u + 4 * me + c;
          s_t[dim][(r / 4) ^ ((dim >> 2) & 15)] = t4[c];   // words of a row swizzled: two lanes per bank
        }
      }
      if (a.k_val) {
        const size_t at = (static_cast<size_t>(s.first + p0 - s.pos + r) * a.hk + h) * D;
        float f[4][8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const float2 lo = fp8_to_float2(static_cast<uint16_t>(q[c] & 0xffffu)), hi = fp8_to_float2(static_cast<uint16_t>(q[c] >> 16));
          const float sc = c < 4 ? kf : vf;
          f[c >> 1][4 * (c & 1)] = lo.x * sc; f[c >> 1][4 * (c & 1) + 1] = lo.y * sc;
          f[c >> 1][4 * (c & 1) + 2] = hi.x * sc; f[c >> 1][4 * (c & 1) + 3] = hi.y * sc;
        }
        *reinterpret_cast<uint4*>(a.k_val + at + d.lo) = pack8(f[0]);
        *reinterpret_cast<uint4*>(a.k_val + at + d.hi) = pack8(f[1]);
        *reinterpret_cast<uint4*>(a.v_val + at + 16 * u) = pack8(f[2]);
        *reinterpret_cast<uint4*>(a.v_val + at + 16 * u + 8) = pack8(f[3]);
      }
    }
  }
  if (full) {
    __syncthreads();
    for (int it = tid; it < D * PAGE_TOKENS / 4; it += THREADS) {
      const int dim = it / (PAGE_TOKENS / 4), w = it % (PAGE_TOKENS / 4);
      reinterpret_cast<uint32_t*>(vp)[it] = s_t[dim][w ^ ((dim >> 2) & 15)];
    }
  }
}

template <int D, int THREADS, int U>
static cudaError_t rope_launch(const RopeArgs& a, cudaStream_t stream) {
  const int reach = (a.max_q + PAGE_TOKENS - 2) / PAGE_TOKENS + 1;   // pages that max_q neighbouring tokens can touch
  const long long kv = static_cast<long long>(a.batch) * reach * a.hk;
  const int qh = THREADS > 64 ? 4 : 1;
  const long long items = static_cast<long long>(a.max_q) * ((a.hq + qh - 1) / qh) * (D / 16), per = (items + THREADS - 1) / THREADS;
  if (kv + per * a.batch > 0x7fffffffll || items > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  return launch_dependent(rope_append_kernel<D, THREADS, U>, dim3(static_cast<unsigned>(kv + per * a.batch)), dim3(THREADS), 0, stream, a,
                          static_cast<int>(kv), reach, static_cast<int>(per));
}

int rope_append_dispatch(RopeArgs a, int dim, cudaStream_t stream) {
  if (!a.qkv || !a.cos_sin || !a.page_table || !a.seq_lens || !a.k || !a.v || !a.k_exp || !a.v_exp || !a.q_out || !a.status) return -1;
  if ((a.k_val == nullptr) != (a.v_val == nullptr)) return -1;
  if (a.m < 1 || a.batch < 1 || a.width < 1 || a.pages < 1 || a.max_q < 1 || a.hq < 1 || a.hk < 1 || (dim != 64 && dim != 128)) return -2;
  if (a.rot < 16 || a.rot > dim || a.rot % 16 || a.width > 0x7fffffff / PAGE_TOKENS || a.table_rows < a.width * PAGE_TOKENS) return -3;
  if (a.ld_qkv % 8 || a.ld_qkv < (a.hq + 2ll * a.hk) * dim) return -4;
  if ((reinterpret_cast<uintptr_t>(a.qkv) | reinterpret_cast<uintptr_t>(a.cos_sin) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
       reinterpret_cast<uintptr_t>(a.q_out) | reinterpret_cast<uintptr_t>(a.k_val) | reinterpret_cast<uintptr_t>(a.v_val)) & 15)
    return -5;
  if (!a.cu_q && (a.max_q != 1 || a.m != a.batch)) return -6;
  if (a.max_q > a.m) a.max_q = a.m;   // no sequence has more new tokens than the batch has rows
  if (a.max_q > 0x7fffffff - PAGE_TOKENS) return -3;
  cudaError_t e;
  // A page's new tokens have to fit a CTA's registers: up to 16 tokens take 64 threads, a whole page 256.
  if (dim == 128) e = a.max_q <= 16 ? rope_launch<128, 64, 2>(a, stream) : rope_launch<128, 256, 2>(a, stream);
  else e = a.max_q <= 16 ? rope_launch<64, 64, 1>(a, stream) : rope_launch<64, 256, 1>(a, stream);
  return static_cast<int>(e);
}

}  // namespace muse
