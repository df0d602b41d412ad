// What the two kernels of the attention over the 8-bit cache share (cache_attn.cu, cache_attn_tc.cu).
#pragma once

#include "attn_sched.cuh"
#include "cache8.cuh"
#include "fp8.cuh"

namespace muse {

// Floats of one partial slot of `rows` rows: max and sum per row, then the rows' sums: as the lanes hold them, [8 rows]
// [D / 16][lane] float4, for tiles of 8 and 16 rows, as [row][D] for tiles of 128.
__host__ __device__ constexpr int attn_slot_floats(int D, int rows) { return rows * (D + 2); }

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

// A row's power of two under which q is FP16: the largest value to [2^9, 2^10). Between the powers whose inverses are normal.
__device__ __forceinline__ int q_exponent(float amax) { return max(min(static_cast<int>(__float_as_uint(amax) >> 23) - 127 - 9, 118), -100); }
// The factor of a page's scores (the row's power, the softmax scale, the page's power) stays positive and finite: the product of
// a zero row's smallest power and a zero page's would be 0 and a masked score, -inf, times 0 NaN. Where the border counts,
// scores lie below 2^-90, or above what FP32 holds.
__device__ __forceinline__ float score_factor(float row, float page) { return fminf(fmaxf(row * page, 1.17549435e-38f), 3.402823466e38f); }

// The weights enter the products with V lifted by 2^lift, and their sums are scaled back in FP32. FP16's smallest step is 2^-24: not
// lifted, weights below 2^-25 of the largest would be missing from the products (but not from the row's sum), and a long
// cache holds many of them (400,000 of 2^-25.5 are 0.8 % of the result). A maximum of 2^20 and more is itself rounded by
// enough to take a lifted weight past FP16's largest value: no lift then.
__device__ __forceinline__ bool too_loud_to_lift(float mx) { return fabsf(mx) >= 1048576.f && mx > -INFINITY; }

// Row to token: n / group, for n * group < 2^32 (the host sees to it).
__device__ __forceinline__ int div_group(const AttnArgs& a, int n) { return a.group == 1 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), a.group_magic)); }

__device__ __forceinline__ AttnEntry attn_entry_of(const AttnArgs& a, int e, int group, int tile) {
  const int b = a.tiles == 1 ? e : e / a.tiles, rt = e - b * a.tiles;
  const int c0 = a.cu_q ? __ldcg(a.cu_q + b) : b, c1 = a.cu_q ? __ldcg(a.cu_q + b + 1) : b + 1;
  return attn_entry(c0, c1, __ldcg(a.seq_lens + b), a.m, a.max_q, a.width * ATTN_PAGE, group, tile, rt, a.window);
}

// Entries as a warp walks them: 32 at a time, one per lane, so that a walk over short sequences pays one round trip
// per 32 of them.
struct EntryCache {
  int base, c0, c1, len;
};
__device__ __forceinline__ AttnEntry attn_entry_cached(const AttnArgs& a, EntryCache& c, int e, int entries, int group, int tile) {
  if (e < c.base || e >= c.base + 32) {   // warp-uniform
    c.base = e;
    const int b = min(e + static_cast<int>(threadIdx.x & 31), entries - 1) / a.tiles;
    c.c0 = a.cu_q ? __ldcg(a.cu_q + b) : b;
    c.c1 = a.cu_q ? __ldcg(a.cu_q + b + 1) : b + 1;
    c.len = __ldcg(a.seq_lens + b);
  }
  const int l = e - c.base;
  return attn_entry(__shfl_sync(0xffffffffu, c.c0, l), __shfl_sync(0xffffffffu, c.c1, l), __shfl_sync(0xffffffffu, c.len, l), a.m, a.max_q,
                    a.width * ATTN_PAGE, group, tile, e % a.tiles, a.window);
}

// A place in the list: entry, head, i-th page of the unit (below zero: the unit's head items).
struct Cursor {
  AttnEntry en;
  int e, h, i;
};

// Lengths and bounds that do not fit are clamped, and said.
__device__ __forceinline__ void attn_report_bad(const AttnArgs& a, int e) {
  const int b = e / a.tiles, len = __ldcg(a.seq_lens + b);
  bool bad = len < 0 || len > a.width * ATTN_PAGE;
  if (a.cu_q) {
    const int c0 = __ldcg(a.cu_q + b), c1 = __ldcg(a.cu_q + b + 1);
    bad |= c0 < 0 || c1 < c0 || c1 > a.m || c1 - c0 > a.max_q;
  }
  if (bad) atomicOr(a.status, ST_BAD_LENGTH);
}

__device__ __forceinline__ float sigmoid_f32(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }   // 1 + e^-x beyond 2^126: 0, as it should be

// Eight neighbouring output values, gated.
__device__ __forceinline__ void store8(const AttnArgs& a, size_t tok, int col, float (&x)[8]) {
  if (a.gate) {
    const __nv_bfloat16* g = a.gate + tok * a.ld_gate + col;
    uint32_t w[4];
    if (a.vec_gate) {
      const uint4 u = __ldcg(reinterpret_cast<const uint4*>(g));
      w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else {
      const unsigned short* p = reinterpret_cast<const unsigned short*>(g);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __ldcg(p + 2 * i) | static_cast<uint32_t>(__ldcg(p + 2 * i + 1)) << 16;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] *= sigmoid_f32(bf16lo_f32(w[i]));
      x[2 * i + 1] *= sigmoid_f32(bf16hi_f32(w[i]));
    }
  }
  __nv_bfloat16* o = a.out + tok * a.ld_out + col;
  if (a.vec_out) {
    uint32_t p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      p[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    *reinterpret_cast<uint4*>(o) = make_uint4(p[0], p[1], p[2], p[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = __float2bfloat16_rn(x[i]);
  }
}

// A wait that usually finds its phase complete: only the first look is inline (the instruction cache is what these kernels
// are short of).
static __noinline__ __device__ bool mbar_wait_on(uint32_t bar, uint32_t parity) { return mbar_wait(bar, parity); }
__device__ __forceinline__ bool mbar_wait_short(uint32_t bar, uint32_t parity) { return mbar_try_wait(bar, parity) || mbar_wait_on(bar, parity); }

cudaError_t cache_attn_tc_launch(const AttnArgs& a, int dim, int sms, cudaStream_t stream);   // cache_attn_tc.cu

}  // namespace muse
