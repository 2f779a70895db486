// Definitions shared by the linear-attention kernels (linear_decode.hip, linear_prefill.hip).
#pragma once

#include "gdn_common.h"
#include "lightdelta_linear_hip.h"

namespace ld {

struct LinearParams {
  const uint16_t* qkv;
  int64_t qkv_row;
  const float* log_decay;
  int64_t decay_row;            // 0: one decay a head
  const int32_t* indices;       // decode: [requests, width]; prefill: the slots
  const int32_t* cu;
  const int32_t* accepted;      // decode only
  const uint8_t* has_initial;   // prefill only
  float* state;
  int64_t state_slot;
  const uint16_t* gate;         // NULL: no norm
  int64_t gate_row;
  const void* norm_weight;
  uint16_t* out;
  int64_t num_tokens;
  int32_t num_slots;
  int32_t num_k_heads;
  int32_t num_v_heads;
  int32_t group;                // num_v_heads / num_k_heads
  int32_t weight_bf16;
  float scale;
  float eps;
};

// The checks and parameters that the two entry points share; returns LD_OK, or an error code
// with the message recorded.
template <typename Args>
int linear_params(const Args& a, int32_t count, const char* what, LinearParams& p) {
  if (count < 0) return fail(LD_ERR_INVALID_ARGUMENT, what);
  if (a.num_k_heads <= 0 || a.num_v_heads <= 0 || a.num_v_heads % a.num_k_heads != 0)
    return fail(LD_ERR_INVALID_ARGUMENT, "num_v_heads must be a positive multiple of num_k_heads");
  if (!(a.eps > 0.0f)) return fail(LD_ERR_INVALID_ARGUMENT, "norm epsilon must be positive");
  if (a.norm_weight_dtype != LD_DTYPE_F32 && a.norm_weight_dtype != LD_DTYPE_BF16)
    return fail(LD_ERR_INVALID_ARGUMENT, "weights must be FP32/BF16");
  if ((a.gate == nullptr) != (a.norm_weight == nullptr))
    return fail(LD_ERR_INVALID_ARGUMENT, "gate and norm weight must be given together");
  if (a.num_tokens < 0 || a.num_slots < 0)
    return fail(LD_ERR_INVALID_ARGUMENT, "num_tokens and num_slots must be >= 0");
  if (count == 0) return LD_OK;
  if (!aligned16(a.state) || (a.state_slot_stride & 3) != 0)
    return fail(LD_ERR_INVALID_ARGUMENT, "state slots must be 16-byte aligned");
  p = LinearParams{};
  p.qkv = static_cast<const uint16_t*>(a.qkv);
  p.qkv_row = a.qkv_row_stride;
  p.log_decay = a.log_decay;
  p.decay_row = a.log_decay_row_stride;
  p.state = a.state;
  p.state_slot = a.state_slot_stride;
  p.gate = static_cast<const uint16_t*>(a.gate);
  p.gate_row = a.gate_row_stride;
  p.norm_weight = a.norm_weight;
  p.out = static_cast<uint16_t*>(a.out);
  p.num_tokens = a.num_tokens;
  p.num_slots = a.num_slots;
  p.num_k_heads = a.num_k_heads;
  p.num_v_heads = a.num_v_heads;
  p.group = a.num_v_heads / a.num_k_heads;
  p.weight_bf16 = a.norm_weight_dtype == LD_DTYPE_BF16;
  p.scale = a.scale;
  p.eps = a.eps;
  return LD_OK;
}

namespace {

// A slot that holds a state: outside 1 .. num_slots - 1 is padding.
__device__ __forceinline__ bool live_slot(int slot, int num_slots) {
  return slot > 0 && slot < num_slots;
}

// A row index from device metadata, clamped to the rows there are.
__device__ __forceinline__ int64_t row_of(int cu, int64_t num_tokens) {
  return min(static_cast<int64_t>(max(cu, 0)), num_tokens);
}

}  // namespace
}  // namespace ld
