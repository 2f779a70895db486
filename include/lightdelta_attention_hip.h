/*
 * C ABI of the softmax-attention operators of liblightdelta_hip.so, for the layers of a model
 * that attend to all earlier tokens beside its recurrent ones: a paged cache of keys and values
 * in 8 bits (written, read back and attended to), and the per-head norm with rotary positions of
 * several axes.  No counterpart in the reference, whose layers are all recurrent.
 *
 * The conventions are lightdelta_hip.h's: plain pointers, strides and sizes, the HIP stream as
 * void*; nothing allocates, synchronises or reads device metadata on the host; 0 on success, else
 * an LD_ERR_* code with ld_last_error()'s message; empty work is a successful no-op.
 */
#ifndef LIGHTDELTA_ATTENTION_HIP_H
#define LIGHTDELTA_ATTENTION_HIP_H

#include <stdint.h>

#include "lightdelta_hip.h"
#include "lightdelta_linear_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * A paged cache and the requests of one call.  Heads have 128 elements.  A page holds page_size
 * tokens (16, 32, 64 or 128) of every kv head, in e4m3 (OCP, no infinities) with one power of
 * two per page, head and kind as the scale (e8m0: byte b stands for 2^(b - 127), within
 * 2^-100 .. 2^119):
 *   k        [num_pages, num_kv_heads, 8, page_size, 16]     element d of token t of the page at
 *                                                            [d / 16, t, d % 16]
 *   v        [num_pages, num_kv_heads, page_size / 16, 128, 16]   at [t / 16, d, t % 16]
 *   k_scale, v_scale   uint8 [num_pages, num_kv_heads]
 * Pages are k_page_stride and v_page_stride bytes apart (multiples of 16, as the pointers are),
 * scales of pages k_scale_stride and v_scale_stride bytes.
 *
 * Request r has the rows cu[r] .. cu[r+1]-1 of the call's activations, which are the last of its
 * lengths[r] tokens: row i is at position lengths[r] - cu[r+1] + i.  The token at position t lies
 * in page pages[r * pages_row_stride + t / page_size].  Positions from table_width * page_size on
 * have no page.  A page outside 1 .. num_pages - 1 is padding: never written, and its tokens are
 * attended to by none, whatever page 0 holds.  lengths[r] <= 0 is a request without tokens.
 */
typedef struct ld_paged_cache {
  void* k;
  void* v;
  uint8_t* k_scale;
  uint8_t* v_scale;
  int64_t k_page_stride;
  int64_t v_page_stride;
  int64_t k_scale_stride;
  int64_t v_scale_stride;
  const int32_t* pages;
  int64_t pages_row_stride;
  const int32_t* cu;
  const int32_t* lengths;
  int64_t num_tokens; /* rows of the activations: cu is clamped to it */
  int32_t table_width;
  int32_t num_pages;
  int32_t page_size;
  int32_t num_kv_heads;
  int32_t num_requests;
} ld_paged_cache;

/* Keys and values in bf16, [num_tokens, num_kv_heads, 128], rows k_row_stride and v_row_stride
 * elements apart. */
typedef struct ld_cache_rows {
  void* k;
  void* v;
  int64_t k_row_stride;
  int64_t v_row_stride;
} ld_cache_rows;

/*
 * Writes every request's rows to their places.  The scale of a page and head is 2^e with the
 * least e for which no finite magnitude m of the rows exceeds 448 * 2^e, within -100 .. 119; where
 * the call begins a page at its first token that is its scale, else the larger of it and the one
 * that it has.  A value x is held as the e4m3 nearest to x * 2^-e (ties to even; magnitudes over
 * 448 as 448; what is not finite as NaN); where a scale grew, values of earlier tokens of the page
 * are rounded anew to the larger one.  Bytes of later tokens of a page are left as they were.  A
 * page is written for one request of a call only, and at one place of its table.
 *
 * Here and in ld_cache_read num_kv_heads * (num_tokens / page_size + 2 * num_requests), or num_kv_heads *
 * num_tokens where that is less, is below 2^24, and num_tokens / page_size + 2 * num_requests below
 * 2^31.
 */
int ld_cache_write(const ld_paged_cache* cache, const ld_cache_rows* rows, void* stream);

/* The values at the rows' places, in bf16 (exactly); zeros where a row has no page.  Rows outside every
 * request are left as they were. */
int ld_cache_read(const ld_paged_cache* cache, const ld_cache_rows* rows, void* stream);

/*
 * Attention of every row to the tokens of its request at its own position and before, whose keys
 * and values are those of the cache (the rows' own among them: write, then attend).  q head h
 * reads kv head h / (num_q_heads / num_kv_heads):
 *   p_j = exp(scale * q . k_j) / sum_j exp(scale * q . k_j)      o = sum_j p_j v_j
 *   out = bf16(o), or with a gate bf16(o * sigmoid(gate))
 * with scores, statistics and sums in fp32 and p, ahead of its product with v, in bf16 (prefill) or as a
 * sum of two bf16 (decode).  A row that sees no token gets zeros.
 * Rows outside every request are left as they were.  What is not finite in a key or value
 * reaches the rows that see it, nothing else; a q . k past fp32's range is not finite.
 *   q, gate  bf16 [num_tokens, num_q_heads, 128], rows q_row_stride and gate_row_stride elements
 *            apart (gate NULL: none)
 *   out      bf16 [num_tokens, num_q_heads, 128] contiguous, overlaps no other argument
 */
typedef struct ld_attention_args {
  const void* q;
  int64_t q_row_stride;
  const void* gate;
  int64_t gate_row_stride;
  void* out;
  int32_t num_q_heads;
  int32_t width; /* decode only: 1 .. LD_MAX_TOKENS */
  float scale;   /* positive, log2(e) * scale finite */
  void* workspace; /* 16-byte aligned device memory, ..._workspace_bytes of it */
  int64_t workspace_bytes;
} ld_attention_args;

/* Decode and speculative verify: requests of at most `width` rows (one with more gets zeros).
 * num_requests * num_kv_heads * (tokens of a table, in 64s) is below 2^30, and num_requests *
 * num_kv_heads * (columns of a kv head, num_q_heads / num_kv_heads * width, in 4s) below 2^23. */
int ld_attention_decode(const ld_paged_cache* cache, const ld_attention_args* args, void* stream);

/* Requests of any number of rows; num_tokens * num_q_heads / num_kv_heads is at most 2^31 - 256, and
 * num_tokens * num_q_heads / 128 + num_requests * num_kv_heads below 2^24. */
int ld_attention_prefill(const ld_paged_cache* cache, const ld_attention_args* args, void* stream);

/* Workspace bytes for these sizes, of which only the sizes count; 0 where none is needed.
 * Nothing is kept in it from one call for the next; calls that may run at once need one each. */
int64_t ld_attention_decode_workspace_bytes(const ld_paged_cache* cache,
                                            const ld_attention_args* args);
int64_t ld_attention_prefill_workspace_bytes(const ld_paged_cache* cache,
                                             const ld_attention_args* args);

/*
 * ld_norm_rope with positions of several axes (time, height and width of an image or video's
 * tokens): angle i of a token is positions[axes[i] * position_axis_stride + token] * inv_freq[i].
 * Where axes[i] is outside 0 .. num_axes - 1, pair i is not turned.
 */
typedef struct ld_rope_axes {
  const int32_t* axes; /* [rotary / 2] */
  int64_t position_axis_stride; /* elements of positions */
  int32_t num_axes;
} ld_rope_axes;

int ld_norm_rope_axes(const ld_norm_rope_args* args, const ld_rope_axes* axes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LIGHTDELTA_ATTENTION_HIP_H */
