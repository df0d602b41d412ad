// Arguments of the kernels around the paged 8-bit cache (rope_append.cu, cache_attn.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace muse {

constexpr int PAGE_TOKENS = 64;

struct RopeArgs {
  const __nv_bfloat16* qkv;   // [m, >= (hq + 2 hk) D], ld_qkv elements between rows
  const float* cos_sin;       // [table_rows, rot / 2, 2]
  const int* page_table;      // [batch, width]
  const int* seq_lens;        // [batch], the new tokens included
  const int* cu_q;            // [batch + 1], or null: one token per sequence
  uint8_t* k;
  uint8_t* v;
  uint8_t* k_exp;             // [pages, hk]
  uint8_t* v_exp;
  __nv_bfloat16* q_out;       // [m, hq, D]
  __nv_bfloat16* k_val;       // [m, hk, D] or null: the values that the cache then holds
  __nv_bfloat16* v_val;
  int* status;
  long long ld_qkv;
  int m, batch, width, pages, max_q, hq, hk, rot, interleaved, table_rows;
};

struct AttnArgs {
  const __nv_bfloat16* q;      // [m, hq, D], ld_q elements between tokens
  const uint8_t* k;            // [pages, hk, 64, D]
  const uint8_t* v;            // [pages, hk, D, 64]
  const uint8_t* k_exp;        // [pages, hk]
  const uint8_t* v_exp;
  const int* page_table;       // [batch, width]
  const int* seq_lens;         // [batch]
  const int* cu_q;             // [batch + 1] or null: one token per sequence
  const __nv_bfloat16* gate;   // [m, hq D], ld_gate elements between tokens, or null
  __nv_bfloat16* out;          // [m, hq D], ld_out elements between tokens
  float* part;                 // partial sums: 2 slots per worker
  int* prefix;                 // [entries + 1] first item of each entry in the list, and their number
  int* status;
  long long ld_q, ld_gate, ld_out;
  float scale_log2;            // softmax scale * log2(e)
  int m, batch, width, pages, max_q, hq, hk, window, tiles;   // tiles: row tiles per sequence
  int group;                   // hq / hk
  int vec_gate, vec_out;       // 16-byte vectors of gate and out are aligned
  uint32_t group_magic;        // 2^32 / group + 1: a row's token without a division
};

int rope_append_dispatch(RopeArgs a, int dim, cudaStream_t stream);
int cache_attn_dispatch(AttnArgs a, int dim, void* ws, cudaStream_t stream);
long long cache_attn_ws_bytes(int batch, int max_q, int hq, int hk, int dim);
long long cache_attn_plan(const int* seq_lens, const int* cu_q, int m, int batch, int width, int max_q, int hq, int hk, int window, int sms,
                          int* segments, long long capacity);
long long cache_attn_join(const int* seq_lens, const int* cu_q, int m, int batch, int width, int max_q, int hq, int hk, int window, int sms,
                          int entry, int head, int* slots, long long capacity);

}  // namespace muse
