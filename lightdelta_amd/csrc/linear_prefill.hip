// Prefill of linear attention with a decay for each head, for gfx950:
//   S <- exp(g) S + v k^T ;  o = scale * S q ;  out = o, or its gated RMSNorm
// over the tokens of each sequence.  One workgroup per (sequence, v-head), its 128 x 128 state in
// registers (the lanes of gdn_step.h), token by token.
#include "gdn_step.h"
#include "linear_common.h"

namespace ld {
namespace {

__global__ __launch_bounds__(kThreads) void linear_prefill_kernel(const LinearParams p) {
  const int seq = blockIdx.x / p.num_v_heads;
  const int head = blockIdx.x - seq * p.num_v_heads;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int64_t bos = row_of(p.cu[seq], p.num_tokens);
  const int64_t eos = row_of(p.cu[seq + 1], p.num_tokens);
  const int slot = p.indices[seq];
  const bool live = live_slot(slot, p.num_slots);
  const int kq = lane & 15;
  const int row_base = 4 * wave + (lane >> 4);
  const int key_head = head / p.group;
  float* const tile = p.state + (live ? slot : 0) * p.state_slot +
                      static_cast<int64_t>(head) * kDim * kDim + row_base * kDim + kq * 4;
  __shared__ float s_o[kDim];
  f32x4 s[kPieces];
#pragma unroll
  for (int j = 0; j < kPieces; ++j)
    s[j] = live && p.has_initial[seq] != 0
               ? *reinterpret_cast<const f32x4*>(tile + tile_piece_bytes<16>(j) / 4)
               : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t token = bos; token < eos; ++token) {
    const uint16_t* row = p.qkv + token * p.qkv_row;
    f32x4 x[4];   // q, k of the lane
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[i][e] = bf16_to_f32(row[((i >> 1) * p.num_k_heads + key_head) * kDim + (i & 1) * 64 + 4 * kq + e]);
    const float decay = __expf(p.log_decay[token * p.decay_row + head]);
#pragma unroll
    for (int i = 0; i < kPieces / 2; ++i) {
      const float v = bf16_to_f32(row[(2 * p.num_k_heads + head) * kDim + row_base + 16 * i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[2 * i][e] = fmaf(v, x[2][e], s[2 * i][e] * decay);
        s[2 * i + 1][e] = fmaf(v, x[3][e], s[2 * i + 1][e] * decay);
      }
      float o = dot8(s[2 * i], s[2 * i + 1], x[0], x[1]), unused = 0.0f;
      row_sum2(o, unused);
      if (kq == 0) s_o[row_base + 16 * i] = o;
    }
    __syncthreads();
    if (wave == 0) {
      float o[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) o[e] = p.scale * s_o[2 * lane + e];
      if (p.gate != nullptr) {
        const float rstd =
            fast_rsqrt(wave_sum(fmaf(o[0], o[0], o[1] * o[1])) * (1.0f / kDim) + p.eps);
        const uint16_t* gate = p.gate + token * p.gate_row + head * kDim + 2 * lane;
#pragma unroll
        for (int e = 0; e < 2; ++e)
          o[e] = ((o[e] * rstd) * load_param(p.norm_weight, 2 * lane + e, p.weight_bf16)) *
                 silu(bf16_to_f32(gate[e]));
      }
#pragma unroll
      for (int e = 0; e < 2; ++e)
        p.out[(token * p.num_v_heads + head) * kDim + 2 * lane + e] = f32_to_bf16(o[e]);
    }
    __syncthreads();
  }
  if (live) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j)
      *reinterpret_cast<f32x4*>(tile + tile_piece_bytes<16>(j) / 4) = s[j];
  }
}

}  // namespace
}  // namespace ld

extern "C" int64_t ld_linear_prefill_workspace_bytes(int64_t, int32_t, int32_t) { return 0; }

extern "C" int ld_linear_prefill(const ld_linear_prefill_args* args, void* stream) {
  using namespace ld;
  if (args == nullptr) return fail(LD_ERR_INVALID_ARGUMENT, "ld_linear_prefill: args is NULL");
  const ld_linear_prefill_args& a = *args;
  LinearParams p{};
  const int rc = linear_params(a, a.num_sequences, "num_sequences must be >= 0", p);
  if (rc != LD_OK || a.num_sequences == 0) return rc;
  if (!a.slots || !a.has_initial || !a.cu_seqlens || !a.state ||
      (a.num_tokens > 0 && (!a.qkv || !a.log_decay || !a.out)))
    return fail(LD_ERR_INVALID_ARGUMENT, "ld_linear_prefill: NULL tensor pointer");
  const int64_t blocks = static_cast<int64_t>(a.num_sequences) * a.num_v_heads;
  if (blocks > 0x3fffff) return fail(LD_ERR_INVALID_ARGUMENT, "too many (sequence, head) tiles");
  p.indices = a.slots;
  p.cu = a.cu_seqlens;
  p.has_initial = a.has_initial;
  hipLaunchKernelGGL(linear_prefill_kernel, dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), p);
  return check_launch("ld_linear_prefill");
}
