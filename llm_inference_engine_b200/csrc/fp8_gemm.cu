// out[m, N] = x[m, K] . W[N, K]^T, both in 8 bits with a power-of-two scale per block of 128 (fp8.cuh), for more tokens than
// the walk of fp8_linear.cu takes: TMA -> shared-memory ring -> block-scaled tcgen05.mma -> tensor memory.
//
// The scales are powers of two, so the tensor core applies them itself (kind::mxf8f6f4, one exponent byte per row and 32
// columns; four neighbouring 32-column pieces share ours): the accumulator holds the scaled sum in FP32 and nothing is
// read back between blocks. A = up to MT x 128 tokens (lanes of tensor memory), B = nt rows of W (columns). The exponents
// live in tensor memory too, as the instruction wants them: row r of 128 in lane r % 32 of every quarter, 32-bit column
// r / 32, the bytes of a word being four successive blocks of 128 columns, which the instruction descriptor
// selects; so one store serves 512 columns of K.
//
// What bounds it at many tokens is traffic from L2 into shared memory, (256 + nt) x 128 bytes per 256 x nt x 128
// products with MT = 2, hence the widest tile that tensor memory holds beside the scales (2 x 224 + 4 x 16 columns);
// at fewer it is the weight's own bytes from memory, and below 20 MB of them the start (4 us to the first MMA behind the
// quantizing kernel: set-up, x's exponents, one block's way through) and the end. K is cut where that lets all SMs load.
// Measured with the quantizing kernel in a replayed graph of calls, each on a weight that is not in cache (us; TB/s of W or
// TFLOP/s; in brackets the same weight every time): 27 x 4093 x 2064 8.9 (8.8); 16 x 4096 x 4096 10.4 (9.6); 27 x 12288 x
// 4096 14.3, 3.5 TB/s (13.7); 256 x 12288 x 4096 18.3, 1410 TFLOP/s (17.3); 4096 x 12288 x 4096 184, 2240 TFLOP/s. Kept up for
// long the last two take 20.5 and 205 to 217 (power). What gave the most: a warp that waits, issues
// and commits for several blocks of K at once (a block alone costs 730 clocks of latency, four cost 1330), uniform issue,
// exponents that are joined from whole words when used instead of byte by byte when loaded, results through shared memory.
// At 4096 tokens a block of K takes 960 clocks, 896 of them MMAs at the tensor core's rate; a fifth of a tile's time is the epilogue,
// under which nothing runs (the accumulators take all of tensor memory; twice the warps for it gained 1%). Tiles of other
// widths are slower: 192 199 us, 128 224, one token tile of 256 217.
//
// Roles: warps 0 and 6 TMA (W and x), warp 1 tensor memory and MMA issue, warps 2..5 scales (registers one group ahead)
// and epilogue, a warp per quarter of the lanes. The grid is persistent: a CTA walks tiles of (K slice, row tile, token tile), and the
// loads of its next tile start while the epilogue drains the accumulators. K slices leave FP32 sums in a workspace that a
// second kernel adds up in slice order (same bits in every run).
#include "fp8.cuh"

namespace muse {

constexpr int G8_TOK = 128;             // rows of one MMA
constexpr int G8_MAX_STAGES = 12;
constexpr int G8_SF_COL = 448;          // first tensor-memory column of the scales
constexpr int G8_SF_STRIDE = 16;        // columns of one group of scales: 4 per token tile, 8 for W's rows
constexpr int G8_SF_BUFS = 4;           // groups of scales in tensor memory: 64 columns
constexpr int G8_THREADS = 224;
constexpr int G8_SMEM = 207 * 1024;     // beside the epilogue's staging rows
constexpr int G8_MIN_SMEM = 116 * 1024;  // one CTA per SM: it takes all of tensor memory

struct G8Args {
  const uint8_t* xe;   // [m, kblocks]
  const uint8_t* we;   // [ceil(N / 128), kblocks]
  __nv_bfloat16* out;
  float* ws;           // [split, m, N] when split > 1
  int* status;
  int m, n, kblocks, ld_out;
  int nt, a_rows;      // rows of W per tile; token rows a TMA box brings
  int row_tiles, tok_tiles, split, stages;
  int at_once;         // blocks of K that the MMA warp takes at a time: 1, 2 or 4, at most half of the stages
};

__device__ __forceinline__ void umma_mxf8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// Instruction descriptor: e4m3 x e4m3 -> FP32, K-major, power-of-two scales; which byte of a scale word counts.
__host__ __device__ constexpr uint32_t g8_idesc(int N, int sf_byte) {
  return (static_cast<uint32_t>(sf_byte) << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>(G8_TOK >> 7) << 27) |
         (static_cast<uint32_t>(sf_byte) << 29);
}
// A look that never waits.
__device__ __forceinline__ bool mbar_test_wait(uint32_t bar, uint32_t parity) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"(bar), "r"(parity)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void tmem_st4(uint32_t addr, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A warp's 32 rows of 32 values, one row per lane (WORDS words), to global memory through shared memory, so that a store
// covers pieces of few rows: a row per lane would touch 32 lines with each store (the epilogue of 128 x 32 values
// took 900 clocks that way, now 550). `first` is the first row's address; `rows` rows and `cols` values of each exist; `vec`:
// rows start on 16 bytes.
template <int WORDS, int BYTES>
__device__ __forceinline__ void put_rows(uint8_t* stage, const uint32_t (&v)[WORDS], uint8_t* first, size_t ld_bytes, int rows, int cols, bool vec, int lane) {
  constexpr int PIECES = WORDS / 4, STRIDE = 32 * BYTES + 16, STEP = 32 / PIECES;
#pragma unroll
  for (int i = 0; i < PIECES; ++i)
    *reinterpret_cast<uint4*>(stage + lane * STRIDE + 16 * i) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  __syncwarp();
  if (vec && (cols * BYTES) % 16 == 0) {
    const int piece = lane % PIECES;
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += STEP) {
      const int r = r0 + lane / PIECES;
      if (r < rows && piece * 16 < cols * BYTES)
        *reinterpret_cast<uint4*>(first + static_cast<size_t>(r) * ld_bytes + 16 * piece) = *reinterpret_cast<const uint4*>(stage + r * STRIDE + 16 * piece);
    }
  } else if (lane < cols) {
#pragma unroll 4
    for (int r = 0; r < rows; ++r) {
      if constexpr (BYTES == 4) *reinterpret_cast<uint32_t*>(first + static_cast<size_t>(r) * ld_bytes + 4 * lane) = *reinterpret_cast<const uint32_t*>(stage + r * STRIDE + 4 * lane);
      else *reinterpret_cast<unsigned short*>(first + static_cast<size_t>(r) * ld_bytes + 2 * lane) = *reinterpret_cast<const unsigned short*>(stage + r * STRIDE + 2 * lane);
    }
  }
  __syncwarp();
}

template <int MT>
__global__ void __launch_bounds__(G8_THREADS, 1) fp8_gemm_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                                                                 const __grid_constant__ G8Args a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[G8_MAX_STAGES], bar_empty[G8_MAX_STAGES];
  __shared__ __align__(8) uint64_t bar_sf_full[G8_SF_BUFS], bar_sf_empty[G8_SF_BUFS], bar_acc_full, bar_acc_empty;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int s_abort;
  __shared__ __align__(16) uint8_t s_rows[4][32 * (32 * 4 + 16)];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;   // the 128-byte swizzle repeats every 1024 bytes
  const uint32_t a_tile = G8_TOK * FP8_BLOCK;                          // a token tile's place in a stage (its box may be shorter)
  const uint32_t b_bytes = static_cast<uint32_t>(a.nt) * FP8_BLOCK;
  const uint32_t stage_bytes = MT * a_tile + b_bytes;
  const int tiles = a.row_tiles * a.tok_tiles * a.split;
  // Tile t: token tiles innermost (neighbouring CTAs share W's rows through L2), then row tiles, then K slices.
  auto slice = [&](int t, int& tok, int& row, int& kb0, int& kb1) {
    tok = t % a.tok_tiles;
    row = t / a.tok_tiles % a.row_tiles;
    const int s = t / (a.tok_tiles * a.row_tiles);
    kb0 = a.kblocks * s / a.split;   // kblocks < 2^24, split <= 16
    kb1 = a.kblocks * (s + 1) / a.split;
    return s;
  };

  if (tid == 0) {
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_x);
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 2);
      mbar_init(smem_u32(&bar_empty[s]), 1);
    }
    for (int i = 0; i < G8_SF_BUFS; ++i) {
      mbar_init(smem_u32(&bar_sf_full[i]), 4);
      mbar_init(smem_u32(&bar_sf_empty[i]), 1);
    }
    mbar_init(smem_u32(&bar_acc_full), 1);
    mbar_init(smem_u32(&bar_acc_empty), 4);
    fence_mbar_init();
    s_abort = 0;
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  griddep_launch_dependents();

  if (warp == 0 || warp == 6) {
    // ---- loads, W by one warp and x by another (W's do not wait for the kernel ahead). The whole warps walk along and one
    // elected lane issues, as for the MMAs.
    const uint64_t pol = l2_policy_evict_last();
    const bool is_x = warp == 6;
    const uint32_t bytes = is_x ? MT * static_cast<uint32_t>(a.a_rows) * FP8_BLOCK : b_bytes;
    int s = 0;
    uint32_t phase = 0, issued = 0;
    bool ok = true;
    if (is_x) griddep_wait();
    for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
      int tok, row, kb0, kb1;
      slice(t, tok, row, kb0, kb1);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (issued >= static_cast<uint32_t>(a.stages) && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_empty[s]), phase ^ 1u))) {
          ok = false;
          break;
        }
        const uint32_t bar = smem_u32(&bar_full[s]), at = smem_base + static_cast<uint32_t>(s) * stage_bytes;
        if (elect_one()) {
          mbar_expect_tx(bar, bytes);
          if (is_x) {
#pragma unroll
            for (int h = 0; h < MT; ++h) tma_load_2d(at + static_cast<uint32_t>(h) * a_tile, &tm_x, kb * FP8_BLOCK, (tok * MT + h) * G8_TOK, bar, pol);
          } else {
            tma_load_2d(at + MT * a_tile, &tm_w, kb * FP8_BLOCK, row * a.nt, bar, pol);
          }
        }
        __syncwarp();
        ++issued;
        if (++s == a.stages) {
          s = 0;
          phase ^= 1u;
        }
      }
    }
    if (!ok) {
      if (lane == 0) atomicOr(a.status, ST_PRODUCER_TIMEOUT);
      s_abort = 1;
      // leave no copy in flight: the stages issued last (bounded; a stage that the other loader has not reached is waited for in vain)
      for (int i = 0; i < a.stages && i < static_cast<int>(issued); ++i) {
        const uint32_t j = issued - 1 - static_cast<uint32_t>(i);
        if (!mbar_wait(smem_u32(&bar_full[j % static_cast<uint32_t>(a.stages)]), (j / static_cast<uint32_t>(a.stages)) & 1u) && lane == 0)
          atomicOr(a.status, ST_DRAIN_TIMEOUT);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // The whole warp walks along and one elected lane issues: an MMA's operands are uniform registers, and what is the
    // same in all lanes is then known to be.
    int s = 0, sf = 0;
    uint32_t phase = 0, sf_phase = 0, acc_phase = 0;
    bool ok = true, looked = false;   // looked: the next block was seen to be there while this one's MMAs were issued
    auto wait = [&](uint64_t& bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar), parity)) != 0; };
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
      int tok, row, kb0, kb1;
      slice(t, tok, row, kb0, kb1);
      // the accumulators are free once the epilogue has read the tile before
      if (t != static_cast<int>(blockIdx.x) && !wait(bar_acc_empty, acc_phase ^ 1u)) ok = false;
      tc_fence_after_sync();
      for (int kb = kb0; kb < kb1 && ok;) {
        // `take` blocks of one group of scales at once: a look at a barrier, the election and what follows a commit take
        // 600 clocks, as long as the MMAs of a small block, and so are paid once for up to four.
        const int j0 = (kb - kb0) & 3, take = min(a.at_once, kb1 - kb);
        const int ends = s + take;
        if (!looked) {
          bool there[5];   // the looks are in flight together
          there[4] = j0 > 0 || mbar_try_wait(smem_u32(&bar_sf_full[sf]), sf_phase);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int st = s + i;
            there[i] = i >= take || mbar_try_wait(smem_u32(&bar_full[st < a.stages ? st : st - a.stages]), st < a.stages ? phase : phase ^ 1u);
          }
          looked = __all_sync(0xffffffffu, there[0] && there[1] && there[2] && there[3] && there[4]);
        }
        if (!looked) {
          if (j0 == 0 && !wait(bar_sf_full[sf], sf_phase)) ok = false;
          for (int i = s; i < ends && ok; ++i) ok = wait(bar_full[i < a.stages ? i : i - a.stages], i < a.stages ? phase : phase ^ 1u);
          if (!ok) break;
        }
        tc_fence_after_sync();
        const uint32_t sfa = tm + G8_SF_COL + static_cast<uint32_t>(sf) * G8_SF_STRIDE, sfb = sfa + 4 * MT;
        const bool sf_last = j0 + take == 4 || kb + take == kb1;
        // One block at a time is a large one: the queue of MMAs is full while its last are issued, which hides a look.
        const bool look = a.at_once == 1 && kb + 1 < kb1;
        bool seen = false;
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (i >= take) break;
            const int st = s + i < a.stages ? s + i : s + i - a.stages;
            const uint32_t at = smem_base + static_cast<uint32_t>(st) * stage_bytes;
            const uint64_t ad = umma_desc_k_sw128(at), bd = umma_desc_k_sw128(at + MT * a_tile);
            const uint32_t idesc = g8_idesc(a.nt, j0 + i), more = kb + i > kb0 ? 1u : 0u;
#pragma unroll
            for (int k = 0; k < FP8_BLOCK / 32; ++k) {   // 32 bytes further along K inside the swizzle span: +2 in 16-byte units
              if (i == 0 && k == FP8_BLOCK / 32 - 1 && look) {
                seen = mbar_test_wait(smem_u32(&bar_full[s + 1 < a.stages ? s + 1 : 0]), s + 1 < a.stages ? phase : phase ^ 1u);
                if (sf_last) seen &= mbar_test_wait(smem_u32(&bar_sf_full[sf + 1 < G8_SF_BUFS ? sf + 1 : 0]), sf + 1 < G8_SF_BUFS ? sf_phase : sf_phase ^ 1u);
              }
#pragma unroll
              for (int h = 0; h < MT; ++h)
                umma_mxf8(tm + static_cast<uint32_t>(h * a.nt), ad + h * (a_tile >> 4) + 2 * k, bd + 2 * k, idesc, sfa + 4u * static_cast<uint32_t>(h), sfb,
                          k > 0 ? 1u : more);
            }
            umma_commit(smem_u32(&bar_empty[st]));
          }
          if (sf_last) umma_commit(smem_u32(&bar_sf_empty[sf]));
          if (kb + take == kb1) umma_commit(smem_u32(&bar_acc_full));
        }
        looked = __any_sync(0xffffffffu, seen) != 0;
        if (sf_last && ++sf == G8_SF_BUFS) {
          sf = 0;
          sf_phase ^= 1u;
        }
        s = ends;
        if (s >= a.stages) {
          s -= a.stages;
          phase ^= 1u;
        }
        kb += take;
      }
      acc_phase ^= 1u;
    }
    if (!ok) {
      if (lane == 0) {
        atomicOr(a.status, ST_MMA_TIMEOUT);
        umma_commit(smem_u32(&bar_acc_full));   // on the way out, so that the epilogue is released
      }
      s_abort = 1;
    }
    __syncwarp();
  } else {
    // ---- scales and epilogue: this warp's quarter of the tensor memory lanes
    const int quarter = warp & 3;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    int sf = 0;
    uint32_t sf_phase = 0, acc_phase = 0, groups = 0;
    bool ok = true;
    // Four successive exponents of a row, wherever they start: the one or two words that they lie in, put together when
    // they are used (that must not wait for the loads here).
    auto get = [&](const uint8_t* row, int kb, int kb1, uint32_t (&w)[2]) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(row + kb);
      const uint32_t* p = reinterpret_cast<const uint32_t*>(at & ~static_cast<uintptr_t>(3));
      w[0] = __ldcg(p);
      w[1] = static_cast<int>(at & 3) + min(kb1 - kb, 4) > 4 ? __ldcg(p + 1) : 0u;
    };
    auto joined = [&](const uint32_t (&w)[2], const uint8_t* row, int kb) {
      return __funnelshift_r(w[0], w[1], 8 * static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row + kb) & 3));
    };
    for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
      int tok, row, kb0, kb1;
      const int s = slice(t, tok, row, kb0, kb1);
      auto x_row = [&](int h, int c) { return a.xe + static_cast<size_t>((tok * MT + h) * G8_TOK + 32 * c + lane) * a.kblocks; };
      auto w_row = [&](int c) { return a.we + static_cast<size_t>((row * a.nt + 32 * c + lane) >> 7) * a.kblocks; };
      auto fetch_x = [&](int kb, uint32_t (&wa)[MT][4][2]) {
#pragma unroll
        for (int h = 0; h < MT; ++h)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            wa[h][c][0] = wa[h][c][1] = 0u;
            if ((tok * MT + h) * G8_TOK + 32 * c + lane < a.m) get(x_row(h, c), kb, kb1, wa[h][c]);
          }
      };
      auto fetch_w = [&](int kb, uint32_t (&wb)[8][2]) {
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          wb[c][0] = wb[c][1] = 0u;
          if (32 * c < a.nt && row * a.nt + 32 * c + lane < a.n) get(w_row(c), kb, kb1, wb[c]);
        }
      };
      uint32_t wa[MT][4][2], wb[8][2];
      fetch_w(kb0, wb);
      if (t == static_cast<int>(blockIdx.x)) griddep_wait();   // x's exponents come from the kernel ahead, and out may still be being read
      fetch_x(kb0, wa);
      for (int kb = kb0; kb < kb1 && ok; kb += 4) {
        if (groups >= G8_SF_BUFS && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_sf_empty[sf]), sf_phase ^ 1u))) {
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t at = tmem + lanes + G8_SF_COL + static_cast<uint32_t>(sf) * G8_SF_STRIDE;
#pragma unroll
        for (int h = 0; h < MT; ++h) {
          uint32_t v[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) v[c] = joined(wa[h][c], x_row(h, c), kb);
          tmem_st4(at + 4u * static_cast<uint32_t>(h), v);
        }
        uint32_t v[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = joined(wb[c], w_row(c), kb);
        tmem_st8(at + 4 * MT, v);
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_sf_full[sf]));
        ++groups;
        if (++sf == G8_SF_BUFS) {
          sf = 0;
          sf_phase ^= 1u;
        }
        if (kb + 4 < kb1) {
          fetch_w(kb + 4, wb);
          fetch_x(kb + 4, wa);
        }
      }
      if (ok && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_acc_full), acc_phase))) ok = false;
      if (__any_sync(0xffffffffu, !ok || s_abort)) {
        if (!ok && lane == 0) atomicOr(a.status, ST_EPILOGUE_TIMEOUT);
        s_abort = 1;
        break;
      }
      acc_phase ^= 1u;
      tc_fence_after_sync();
      const bool vec = (a.ld_out & 7) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0 && (a.nt & 7) == 0;
      uint8_t* stage = s_rows[quarter];
#pragma unroll 1
      for (int h = 0; h < MT; ++h) {
        const int token = (tok * MT + h) * G8_TOK + quarter * 32 + lane;
#pragma unroll 1
        for (int c = 0; c < a.nt; c += 32) {
          uint32_t v[32];
          __syncwarp();
          tmem_ld16(tmem + lanes + static_cast<uint32_t>(h * a.nt + c), reinterpret_cast<uint32_t(&)[16]>(v[0]));
          if (c + 16 < a.nt) tmem_ld16(tmem + lanes + static_cast<uint32_t>(h * a.nt + c + 16), reinterpret_cast<uint32_t(&)[16]>(v[16]));
          tmem_ld_wait();
          const int n0 = row * a.nt + c, cols = min(min(32, a.nt - c), a.n - n0);
          if (cols <= 0) continue;   // (the same in all lanes)
          const int rows = min(32, a.m - (token - lane));
          if (a.split > 1) {
            put_rows<32, 4>(stage, v, reinterpret_cast<uint8_t*>(a.ws + (static_cast<size_t>(s) * a.m + (token - lane)) * a.n + n0),
                            static_cast<size_t>(a.n) * 4, rows, cols, (a.n & 3) == 0, lane);
          } else {
            uint32_t p[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const __nv_bfloat162 b = __floats2bfloat162_rn(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
              p[i] = *reinterpret_cast<const uint32_t*>(&b);
            }
            put_rows<16, 2>(stage, p, reinterpret_cast<uint8_t*>(a.out + static_cast<size_t>(token - lane) * a.ld_out + n0), static_cast<size_t>(a.ld_out) * 2,
                            rows, cols, vec, lane);
          }
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_acc_empty));
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// Adds up the K slices' sums, in slice order.
__global__ void __launch_bounds__(256) fp8_join_kernel(const float* __restrict__ ws, __nv_bfloat16* __restrict__ out, int m, int n, int split, int ld_out) {
  griddep_launch_dependents();
  griddep_wait();
  const long long total = static_cast<long long>(m) * n;
  const bool vec = (n & 3) == 0 && (ld_out & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & 7) == 0;
  if (vec) {
    for (long long i = (blockIdx.x * 256ll + threadIdx.x) * 4; i < total; i += static_cast<long long>(gridDim.x) * 1024) {
      float4 v = __ldcg(reinterpret_cast<const float4*>(ws + i));
      for (int s = 1; s < split; ++s) {
        const float4 u = __ldcg(reinterpret_cast<const float4*>(ws + static_cast<size_t>(s) * total + i));
        v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
      }
      const __nv_bfloat162 p = __floats2bfloat162_rn(v.x, v.y), q = __floats2bfloat162_rn(v.z, v.w);
      *reinterpret_cast<uint2*>(out + i / n * ld_out + i % n) = make_uint2(*reinterpret_cast<const uint32_t*>(&p), *reinterpret_cast<const uint32_t*>(&q));
    }
  } else {
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += static_cast<long long>(gridDim.x) * 256) {
      float v = __ldcg(ws + i);
      for (int s = 1; s < split; ++s) v += __ldcg(ws + static_cast<size_t>(s) * total + i);
      out[i / n * ld_out + i % n] = __float2bfloat16_rn(v);
    }
  }
}

// ---------------------------------------------------------------- host side
struct G8Plan {
  int mt, nt, split, stages;
};

// Stages of the ring, and blocks of K that the MMA warp takes at once.
static int g8_stages(int mt, int nt) {
  const int fit = (G8_SMEM - 1024) / ((mt * G8_TOK + nt) * FP8_BLOCK);
  return fit < G8_MAX_STAGES ? fit : G8_MAX_STAGES;
}
static int g8_at_once(int stages) { return stages >= 8 ? 4 : stages >= 4 ? 2 : 1; }

// The tile and the K slices with the shortest time by what was measured, in ns: a block of K costs a CTA the bytes that it
// brings into shared memory (140 a ns), its MMAs, or the issuing of them (385, 250 or 185 for 1, 2 or 4 blocks at once),
// whichever is longest, and all CTAs together W's bytes from memory (6000 a ns); 290 per 32 columns of the epilogue; slices cost a second launch and the sums' way through L2.
static G8Plan g8_search(int m, int n, int k, int sms) {
  const int kblocks = (k + FP8_BLOCK - 1) / FP8_BLOCK;
  const double from_memory = static_cast<double>(n) * k / 6000.0;
  G8Plan best = {};
  double best_ns = 1e30;
  for (int mt = 1; mt <= 2; ++mt) {
    if (mt == 2 && m <= G8_TOK) continue;
    const int tok_tiles = (m + mt * G8_TOK - 1) / (mt * G8_TOK);
    const double a_rows = mt == 1 && m < G8_TOK ? (m + 7) / 8 * 8 : mt * G8_TOK;
    for (int nt = 32; nt <= (mt == 2 ? 224 : 256); nt += 16) {
      const int row_tiles = (n + nt - 1) / nt, at_once = g8_at_once(g8_stages(mt, nt));
      const double issue = at_once == 4 ? 185.0 : at_once == 2 ? 250.0 : 385.0, load = (a_rows + nt) * FP8_BLOCK / 140.0, mma = 1.05 * mt * nt;
      const double block = load > mma ? (load > issue ? load : issue) : mma > issue ? mma : issue;
      for (int split = 1; split <= 16 && split <= kblocks; ++split) {
        const long long tiles = static_cast<long long>(tok_tiles) * row_tiles * split;
        const long long waves = (tiles + sms - 1) / sms;
        const int kb = (kblocks + split - 1) / split;
        double body = static_cast<double>(waves) * kb * block;
        if (body < from_memory) body = from_memory;
        double ns = body + waves * (290.0 * mt * ((nt + 31) / 32) + 300.0);
        if (split > 1) ns += 2200.0 + static_cast<double>(m) * n * split * 8 / 4000.0;
        if (ns < best_ns) {
          best_ns = ns;
          best = {mt, nt, split, g8_stages(mt, nt)};
        }
      }
    }
  }
  return best;
}

// The search takes microseconds; a thread's last shapes are kept.
static G8Plan g8_plan(int m, int n, int k, int sms) {
  struct Kept {
    int m, n, k, sms;
    G8Plan plan;
  };
  static thread_local Kept kept[64];
  Kept& c = kept[(static_cast<unsigned>(m) * 31u + static_cast<unsigned>(n) * 7u + static_cast<unsigned>(k)) & 63u];
  if (c.m != m || c.n != n || c.k != k || c.sms != sms) c = {m, n, k, sms, g8_search(m, n, k, sms)};
  return c.plan;
}

long long fp8_gemm_ws_bytes(int m, int n, int k) {
  if (m < 1 || n < 1 || k < 16 || k % 16) return -1;
  const int sms = device_sms();
  if (sms < 1) return -2;
  const G8Plan p = g8_plan(m, n, k, sms);
  return p.split > 1 ? static_cast<long long>(p.split) * m * n * 4 : 0;
}

template <int MT>
static cudaError_t g8_launch(const CUtensorMap& tx, const CUtensorMap& tw, const G8Args& a, int grid, size_t smem, cudaStream_t stream) {
  static DeviceOnce once;   // the largest any plan asks for, once
  const cudaError_t e = once.run([&] { return cudaFuncSetAttribute(fp8_gemm_kernel<MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, G8_SMEM); });
  if (e != cudaSuccess) return e;
  return launch_dependent(fp8_gemm_kernel<MT>, dim3(grid), dim3(G8_THREADS), smem, stream, tx, tw, a);
}

int encode_2d_u8(CUtensorMap* tm, const void* base, long long rows, long long cols, int box_rows);   // capi.cu

int fp8_gemm_dispatch(const void* W, const void* we, const void* xq, const void* xe, void* out, void* ws, int* status, int m, int n, int k, int ld_out,
                      cudaStream_t stream) {
  if (!W || !we || !xq || !xe || !out || !status || m < 1 || n < 1 || k < 16 || k % 16) return -1;
  if (ld_out < n || ((reinterpret_cast<uintptr_t>(xq) | reinterpret_cast<uintptr_t>(W)) & 15)) return -2;
  const int sms = device_sms();
  if (sms < 1) return -4;
  const G8Plan p = g8_plan(m, n, k, sms);
  if (p.split > 1 && (!ws || (reinterpret_cast<uintptr_t>(ws) & 15))) return -3;
  G8Args a = {};
  a.xe = static_cast<const uint8_t*>(xe);
  a.we = static_cast<const uint8_t*>(we);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.ws = static_cast<float*>(ws);
  a.status = status;
  a.m = m; a.n = n;
  a.kblocks = (k + FP8_BLOCK - 1) / FP8_BLOCK;
  a.ld_out = ld_out;
  a.nt = p.nt;
  a.a_rows = p.mt == 1 && m < G8_TOK ? (m + 7) / 8 * 8 : G8_TOK;
  a.tok_tiles = (m + p.mt * G8_TOK - 1) / (p.mt * G8_TOK);
  a.row_tiles = (n + p.nt - 1) / p.nt;
  a.split = p.split;
  a.stages = p.stages;
  a.at_once = g8_at_once(p.stages);
  CUtensorMap tx, tw;
  int r = encode_2d_u8(&tx, xq, m, k, a.a_rows);
  if (r == 0) r = encode_2d_u8(&tw, W, n, k, p.nt);
  if (r != 0) return r;
  const long long tiles = static_cast<long long>(a.row_tiles) * a.tok_tiles * a.split;
  if (tiles > 0x7fffffffll) return -3;
  const int grid = static_cast<int>(tiles < sms ? tiles : sms);
  size_t smem = static_cast<size_t>(p.stages) * (p.mt * G8_TOK + p.nt) * FP8_BLOCK + 1024;
  if (smem < G8_MIN_SMEM) smem = G8_MIN_SMEM;
  cudaError_t e = p.mt == 2 ? g8_launch<2>(tx, tw, a, grid, smem, stream) : g8_launch<1>(tx, tw, a, grid, smem, stream);
  if (e == cudaSuccess && p.split > 1) {
    const long long quads = (static_cast<long long>(m) * n + 1023) / 1024;
    e = launch_dependent(fp8_join_kernel, dim3(static_cast<unsigned>(quads < 4ll * sms ? quads : 4ll * sms)), dim3(256), 0, stream, a.ws, a.out, m, n, p.split, ld_out);
  }
  return static_cast<int>(e);
}

}  // namespace muse
