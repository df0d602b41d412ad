// out[m, N] = x[m, K] . W[N, K]^T with both operands in 8 bits and a power-of-two scale per block of 128 (fp8.cuh):
//     out[t, n] = sum over K blocks b of 2^(ex[t, b] + ew[n / 128, b]) * sum over k in b of xq[t, k] wq[n, k]
// BF16 out; x comes in BF16 and is quantised here (one exponent per token and 128 columns), W as codes and exponent
// bytes. The products of codes are exact in FP32 and so is the scaling; the sums are FP32.
//
//   fp8_walk_kernel       up to 8 tokens: the persistent walk of fewtok_mma.cu over half the bytes. Tokens are half of the
//                     MMA's M = 16, 8 weight rows its N; a lane loads 16-byte pieces of W straight into the B fragments of
//                     two m16n8k32 MMAs (the k slots are a permutation that x follows). A warp owns whole 128-column
//                     blocks, so its x fragments, quantised in registers from BF16 (the four lanes of a token share
//                     the block: two shuffles give its largest magnitude), and their scales never change.
//   fp8_quantize_kernel   x to codes and exponents, for the many-token kernel (fp8_gemm.cu) and for callers.
//
// Measured in a replayed graph of calls, each on weights that are not in cache: 4096 x 4096 at 1 / 8 tokens 7.4 / 7.6 us (2.2 TB/s
// of W), 4096 x 8192 12.1 / 12.4 (2.7 TB/s), 256 x 4096 3.5 / 3.7. It is not memory that bounds it (35 to 43 % of its rate) but the
// chain of a call: x's way to all SMs and its rounding, a barrier and a sum over 32 warps for every 8 rows, 3.5 us of which
// are there for any W. K above 4096 takes the form with two blocks of K per warp, which spills 28 bytes at 64 registers.
// With 9 to 16 tokens in the MMA's other half it took 2.8 us more for any W (x read and quantised by every SM), where
// fp8_gemm.cu is as fast or faster, so it has no such form. fp8_quantize_kernel: 4096 x 4096 22.0 us of 7.8 for its bytes
// (bound by issue: 62 %), 256 x 4096 2.4.
#include "../../include/muse_proj.h"
#include "fp8.cuh"

namespace muse {

__device__ __forceinline__ void mma_e4m3_16832(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                               uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ---------------------------------------------------------------- x to 8 bits
// One warp per token and block of 128 columns: 4 values per lane.
__global__ void __launch_bounds__(256) fp8_quantize_kernel(const __nv_bfloat16* __restrict__ x, uint8_t* __restrict__ xq,
                                                           uint8_t* __restrict__ xe, int m, int K, int ld_x, int kblocks) {
  griddep_launch_dependents();
  griddep_wait();
  const long long item = blockIdx.x * 8ll + (threadIdx.x >> 5);
  if (item >= static_cast<long long>(m) * kblocks) return;
  const int t = static_cast<int>(item / kblocks), b = static_cast<int>(item % kblocks), lane = threadIdx.x & 31;
  const int k = b * FP8_BLOCK + lane * 4;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (k < K) {   // K % 16 == 0: a lane's four columns are in or out together
    const uint2 w = __ldcg(reinterpret_cast<const uint2*>(x + static_cast<size_t>(t) * ld_x + k));
    v[0] = bf16lo_f32(w.x); v[1] = bf16hi_f32(w.x); v[2] = bf16lo_f32(w.y); v[3] = bf16hi_f32(w.y);
  }
  float a = fmaxf(fmaxf(finite_abs(v[0]), finite_abs(v[1])), fmaxf(finite_abs(v[2]), finite_abs(v[3])));
#pragma unroll
  for (int s = 16; s; s >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, s));
  const int e = fp8_exponent_byte(a);
  const float inv = exp2_byte_inv(e);
  if (k < K) *reinterpret_cast<uint32_t*>(xq + static_cast<size_t>(t) * K + k) = fp8_pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
  if (lane == 0) xe[static_cast<size_t>(t) * kblocks + b] = static_cast<uint8_t>(e);
}

// ---------------------------------------------------------------- up to 8 tokens
// NW warps; BPW blocks of K per warp (K <= 128 * NW * BPW); D row groups in flight per warp.
// The warps are wk (a power of two) slices of K times NW / wk neighbouring row groups.
template <int NW, int BPW, int D>
__global__ void __launch_bounds__(NW * 32) fp8_walk_kernel(const uint8_t* __restrict__ W, const uint8_t* __restrict__ we,
                                                           const __nv_bfloat16* __restrict__ x, __nv_bfloat16* __restrict__ out, int m,
                                                           int N, int K, int ld_x, int ld_out, int wk) {
  constexpr int OUTS = 64;   // 8 tokens x 8 rows
  __shared__ __align__(16) float red[2][NW][OUTS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int kblocks = (K + FP8_BLOCK - 1) / FP8_BLOCK;
  const int ks = warp & (wk - 1), rs = warp / wk, rslots = NW / wk;   // this warp's K slice and row slot
  const int groups = (N + 7) >> 3;
  const int sets = (groups + rslots - 1) / rslots;                    // a CTA step walks rslots groups
  const int my_sets = static_cast<int>(blockIdx.x) < sets ? (sets - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;
  auto group_of = [&](int i) { return (static_cast<int>(blockIdx.x) + i * static_cast<int>(gridDim.x)) * rslots + rs; };

  uint4 w[D][BPW][2];
  uint32_t se[D][BPW];
  auto load = [&](uint4 (&d)[BPW][2], uint32_t (&s)[BPW], int i) {
    const int grp = group_of(i);
    const int row = min(grp * 8 + g, N - 1);
#pragma unroll
    for (int j = 0; j < BPW; ++j) {
      const int kb = ks + j * wk;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int k = kb * FP8_BLOCK + 64 * p + 16 * t;
        d[j][p] = k < K && grp < groups ? ldg_stream16(W + static_cast<size_t>(row) * K + k) : make_uint4(0u, 0u, 0u, 0u);
      }
      s[j] = kb < kblocks ? __ldg(we + static_cast<size_t>(min(grp * 8, N - 1) >> 7) * kblocks + kb) : 0u;
    }
  };
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (d < my_sets) load(w[d], se[d], d);
  griddep_launch_dependents();
  griddep_wait();   // x and out belong to the stream: only the weights were touched so far

  // x fragments: the lane's 32 columns of each of its blocks, for token g, in BF16 -> codes in registers.
  uint32_t xa[BPW][8];
  int sa[BPW];
  auto quantise = [&](int tok, int kb, uint32_t (&q)[8], int& byte) {
    uint4 v[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const int k = kb * FP8_BLOCK + 64 * (p >> 1) + 16 * t + 8 * (p & 1);
      v[p] = tok < m && k < K ? __ldcg(reinterpret_cast<const uint4*>(x + static_cast<size_t>(tok) * ld_x + k)) : make_uint4(0u, 0u, 0u, 0u);
    }
    float a = 0.f;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const uint32_t u[4] = {v[p].x, v[p].y, v[p].z, v[p].w};
#pragma unroll
      for (int c = 0; c < 4; ++c) a = fmaxf(a, fmaxf(finite_abs(bf16lo_f32(u[c])), finite_abs(bf16hi_f32(u[c]))));
    }
    a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
    a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
    byte = fp8_exponent_byte(a);
    const float inv = exp2_byte_inv(byte);
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const uint32_t u[4] = {v[p].x, v[p].y, v[p].z, v[p].w};
#pragma unroll
      for (int c = 0; c < 2; ++c)
        q[2 * p + c] = fp8_pack4(bf16lo_f32(u[2 * c]) * inv, bf16hi_f32(u[2 * c]) * inv, bf16lo_f32(u[2 * c + 1]) * inv, bf16hi_f32(u[2 * c + 1]) * inv);
    }
  };
#pragma unroll
  for (int j = 0; j < BPW; ++j) quantise(g, ks + j * wk, xa[j], sa[j]);

  for (int i0 = 0; i0 < my_sets; i0 += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int i = i0 + d;
      if (i < my_sets) {   // CTA-uniform
        float acc[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < BPW; ++j) {
          float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const uint4 u = w[d][j][p];
            mma_e4m3_16832(c, xa[j][4 * p], 0u, xa[j][4 * p + 1], 0u, u.x, u.y);
            mma_e4m3_16832(c, xa[j][4 * p + 2], 0u, xa[j][4 * p + 3], 0u, u.z, u.w);
          }
          // Both powers in one, or, where their sum lies beyond FP32 (the scaled product need not), half of it at a time.
          const int byte = static_cast<int>(se[d][j]) + sa[j] - 127;
          float s2 = exp2_byte(byte);
          if (static_cast<unsigned>(byte - 1) > 253u) {
            const float s1 = exp2_byte((byte + 127) >> 1);
            s2 = exp2_byte(byte + 127 - ((byte + 127) >> 1));
            c[0] *= s1;
            c[1] *= s1;
          }
          acc[0] = fmaf(c[0], s2, acc[0]);
          acc[1] = fmaf(c[1], s2, acc[1]);
        }
        if (i + D < my_sets) load(w[d], se[d], i + D);   // into the registers just read: in flight across the reduction
        float* mine = red[i & 1][warp];
        *reinterpret_cast<float2*>(mine + g * 8 + 2 * t) = make_float2(acc[0], acc[1]);
        __syncthreads();   // the buffer written two steps ago is free again once every warp passed this
        for (int o = threadIdx.x; o < rslots * OUTS; o += NW * 32) {
          const int slot = o / OUTS, v = o % OUTS;
          float sum = 0.f;
#pragma unroll 8
          for (int s = 0; s < wk; ++s) sum += red[i & 1][slot * wk + s][v];
          const int tok = v >> 3, row = ((static_cast<int>(blockIdx.x) + i * static_cast<int>(gridDim.x)) * rslots + slot) * 8 + (v & 7);
          if (tok < m && row < N) out[static_cast<size_t>(tok) * ld_out + row] = __float2bfloat16_rn(sum);
        }
      }
    }
  }
}

// ---------------------------------------------------------------- host side
int fp8_quantize_dispatch(const void* x, void* xq, void* xe, int m, int K, int ld_x, cudaStream_t stream) {
  if (!x || !xq || !xe || m < 1 || K < 16 || K % 16) return -1;
  if (ld_x < K || ld_x % 8 || ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(xq)) & 15)) return -2;
  const int kblocks = (K + FP8_BLOCK - 1) / FP8_BLOCK;
  const long long blocks = (static_cast<long long>(m) * kblocks + 7) / 8;
  if (blocks > 0x7fffffffll) return -3;
  return static_cast<int>(launch_dependent(fp8_quantize_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream,
                                           static_cast<const __nv_bfloat16*>(x), static_cast<uint8_t*>(xq), static_cast<uint8_t*>(xe), m, K, ld_x, kblocks));
}

template <int NW, int BPW, int D>
static cudaError_t fp8_walk_launch(const void* W, const void* we, const void* x, void* out, int m, int N, int K, int ld_x, int ld_out,
                                   int sms, cudaStream_t stream) {
  const int kblocks = (K + FP8_BLOCK - 1) / FP8_BLOCK;
  int wk = 1;
  while (wk < NW && wk < kblocks) wk *= 2;
  const int sets = ((N + 7) / 8 + NW / wk - 1) / (NW / wk);
  return launch_dependent(fp8_walk_kernel<NW, BPW, D>, dim3(sets < sms ? sets : sms), dim3(NW * 32), 0, stream,
                          static_cast<const uint8_t*>(W), static_cast<const uint8_t*>(we), static_cast<const __nv_bfloat16*>(x),
                          static_cast<__nv_bfloat16*>(out), m, N, K, ld_x, ld_out, wk);
}

int fp8_walk_dispatch(const void* W, const void* we, const void* x, void* out, int m, int N, int K, int ld_x, int ld_out, cudaStream_t stream) {
  if (!W || !we || !x || !out || m < 1 || m > MUSE_FP8_WALK_TOKENS || N < 1 || K < 16 || K % 16 || K > MUSE_FP8_WALK_K) return -1;
  if (ld_x < K || ld_x % 8 || ld_out < N || ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(W)) & 15)) return -2;
  const int sms = device_sms();
  if (sms < 1) return -4;
  // 32 warps of 64 registers hold two row groups of one block of K in flight, or one of two blocks.
  return static_cast<int>(K <= 4096 ? fp8_walk_launch<32, 1, 2>(W, we, x, out, m, N, K, ld_x, ld_out, sms, stream)
                                    : fp8_walk_launch<32, 2, 1>(W, we, x, out, m, N, K, ld_x, ld_out, sms, stream));
}

}  // namespace muse
