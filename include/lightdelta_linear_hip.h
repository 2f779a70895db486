/*
 * C ABI of the linear-attention operators of liblightdelta_hip.so: linear attention with a
 * decay for each head over the slot-indexed state pool (recurrent form for decode and
 * speculative verify, chunked form for prompts), and the per-head norm with position rotation
 * that goes ahead of it.  No counterpart in the reference, whose only recurrence is the gated
 * delta rule.
 *
 * The conventions are lightdelta_hip.h's: plain pointers, element strides and sizes, the HIP
 * stream as void*; nothing allocates, synchronises or reads device metadata on the host; 0 on
 * success, else an LD_ERR_* code with ld_last_error()'s message; empty work is a successful
 * no-op.
 */
#ifndef LIGHTDELTA_LINEAR_HIP_H
#define LIGHTDELTA_LINEAR_HIP_H

#include <stdint.h>

#include "lightdelta_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Linear attention with a decay for each head.  Per v-head h (k-head h / (HV / H)) with state
 * S [128 (V), 128 (K)]:
 *   S <- exp(g) S + v k^T         o = scale * S q
 *   out = bf16(o), or with a gate bf16(o * rsqrt(mean(o^2) + eps) * w * silu(gate))
 * with S, o, the norm and every sum in fp32.
 *
 * Layouts (element strides):
 *   qkv        bf16 [tokens, (2*H + HV)*128], row stride qkv_row_stride: q of k-head kh at
 *              column kh*128, k at H*128 + kh*128, v of v-head h at 2*H*128 + h*128
 *   log_decay  fp32, g of (token, head) at token*log_decay_row_stride + head; a row stride of 0
 *              is one constant decay a head.  g <= 0; -inf empties the state
 *              (of finite values: those that are not stay, as 0 times them is NaN)
 *   state      fp32 [num_slots, HV, 128(V), 128(K)], slot stride state_slot_stride, 16-byte
 *              aligned
 *   gate       bf16 [tokens, HV, 128], row stride gate_row_stride, or NULL with norm_weight
 *              NULL: no norm
 *   norm_weight fp32 or bf16 [128] (norm_weight_dtype)
 *   out        bf16 [tokens, HV, 128] contiguous
 * out and state overlap no other argument, nor do two slots or two rows of out.
 * A slot outside 1 .. num_slots - 1 is padding: never read, never written.  Non-finite values of
 * a token's activations reach that token's and later outputs, and the state, of its request alone.
 */

/*
 * One decode or speculative-verify step, requests as in ld_gdn_decode: request r covers tokens
 * cu[r] .. cu[r+1]-1; its source state is slot indices[r, accepted[r]-1] when 1 <= accepted[r]
 * <= width; the state after token t goes to slot indices[r, t].  A request with an invalid
 * source, or with more tokens than width, gets zero outputs and leaves the pool untouched; one
 * without tokens writes nothing.  Slots that two requests of a call share are undefined.
 */
typedef struct ld_linear_decode_args {
  const void* qkv;
  int64_t qkv_row_stride;
  const float* log_decay;
  int64_t log_decay_row_stride;
  const int32_t* indices;
  const int32_t* cu;
  const int32_t* accepted;
  float* state;
  int64_t state_slot_stride;
  const void* gate;
  int64_t gate_row_stride;
  const void* norm_weight;
  void* out;
  int64_t num_tokens; /* rows of qkv and out: cu is clamped to it */
  int32_t num_slots;
  int32_t num_requests;
  int32_t width; /* 1 .. LD_MAX_TOKENS */
  int32_t num_k_heads;
  int32_t num_v_heads;
  int32_t norm_weight_dtype;
  float scale;
  float eps;
  int32_t cache_policy; /* LD_CACHE_KEEP or LD_CACHE_STREAM (no effect on results) */
} ld_linear_decode_args;

int ld_linear_decode(const ld_linear_decode_args* args, void* stream);

/*
 * Prompts of num_sequences sequences, as in ld_gdn_prefill: sequence n covers rows
 * cu_seqlens[n] .. cu_seqlens[n+1]-1; its state starts from state[slots[n]] when slots[n] is not
 * padding and has_initial[n] != 0, else from zeros, and the state after its last token goes to
 * state[slots[n]] (an empty sequence writes its initial state back).  Rows outside every
 * sequence are left as they were.  Slots are distinct.  Row strides of qkv, gate and log_decay are
 * 0 .. 2^23 elements (of a single row anything), rows of out likewise (num_v_heads <= 2^16),
 * num_tokens < 2^31.
 */
typedef struct ld_linear_prefill_args {
  const void* qkv;
  int64_t qkv_row_stride;
  const float* log_decay;
  int64_t log_decay_row_stride;
  const int32_t* slots;
  const uint8_t* has_initial;
  const int32_t* cu_seqlens;
  float* state;
  int64_t state_slot_stride;
  const void* gate;
  int64_t gate_row_stride;
  const void* norm_weight;
  void* out;
  int64_t num_tokens; /* rows of qkv and out: cu_seqlens is clamped to it */
  int32_t num_slots;
  int32_t num_sequences;
  int32_t num_k_heads;
  int32_t num_v_heads;
  int32_t norm_weight_dtype;
  float scale;
  float eps;
  void* workspace; /* ld_linear_prefill_workspace_bytes of device memory, 16-byte aligned */
  int64_t workspace_bytes;
} ld_linear_prefill_args;

int ld_linear_prefill(const ld_linear_prefill_args* args, void* stream);

/*
 * Workspace bytes of ld_linear_prefill for these sizes, 64 MiB and little more at most; 0 where
 * it needs none.  Two states and a decay for each segment of a head but the first, segments of at
 * least 128 tokens (of several sequences 256).  Nothing is kept in it from one call for the next; calls that may run at once
 * need one each.
 */
int64_t ld_linear_prefill_workspace_bytes(int64_t num_tokens, int32_t num_sequences,
                                          int32_t num_v_heads);

/*
 * RMSNorm and position rotation of every q and k head, in place.  For each head row x of the
 * first q_heads + k_heads heads of a row of qkv (bf16, row stride qkv_row_stride; later columns
 * are left alone):
 *   y = x * rsqrt(mean(x^2) + eps) * w         (w: q_weight or k_weight [128], weight_dtype)
 *   a = positions[token] * inv_freq[i]         i < rotary / 2
 *   halves:      (y[i], y[i + rotary/2])  turned by a
 *   interleaved: (y[2 i], y[2 i + 1])     turned by a
 * and rounded to bf16 once; elements from `rotary` on are only normalised.  positions int32 or
 * int64 [tokens] (any value: angles are those of the exact product, reduced within 2^-44 of a turn for
 * |inv_freq| <= 1); inv_freq fp32 [rotary / 2].  rotary <= 128: a multiple of 16
 * (halves) or of 2 (interleaved); 0 for the norm alone.
 */
typedef struct ld_norm_rope_args {
  void* qkv;
  int64_t qkv_row_stride;
  const void* q_weight;
  const void* k_weight;
  int32_t q_weight_dtype;
  int32_t k_weight_dtype;
  const void* positions;
  int32_t positions_int64; /* 0: int32, 1: int64 */
  int32_t rotary;
  const float* inv_freq;
  int64_t num_tokens;
  int32_t q_heads;
  int32_t k_heads;
  int32_t interleaved;
  float eps;
} ld_norm_rope_args;

int ld_norm_rope(const ld_norm_rope_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LIGHTDELTA_LINEAR_HIP_H */
