// Decode / speculative-verify step of linear attention with a decay for each head, for gfx950:
//   S <- exp(g) S + v k^T ;  o = scale * S q ;  out = o, or its gated RMSNorm
// per (request, v-head), S a 128 x 128 fp32 tile of the state pool.
//
// Bound by memory: a tile is read once and written once a token, 4 flops an element and token.
// One workgroup of 16 waves per tile, its lanes as in gdn_step.h (16 lanes a K row, 4 V rows a
// wave and piece pair, so that a piece pair of all waves covers half the tile in address order);
// every tile load goes out first, then the pieces are worked in load order, each
// row pair scaled, updated, stored and reduced against q (8 products a lane, 4 DPP steps).  A
// token's q, k and v come straight to registers: the recurrence normalises nothing, so there is
// nothing to stage.  Two tiles a CU for one token; for verify steps, whose four tokens' inputs need
// the registers, one.
#include "gdn_step.h"
#include "linear_common.h"

namespace ld {
namespace {

// A token as a lane needs it: q and k at 4 kq .. and 64 + 4 kq .., v of its V rows.
template <int Rows>
struct LinearToken {
  uint16_t q[8], k[8], v[Rows];
  float decay;
};

constexpr int kTileWaves = 16;

template <int LoadPol, int StorePol, int Width>
__global__ __launch_bounds__(64 * kTileWaves)
__attribute__((amdgpu_waves_per_eu(Width == 1 ? 8 : 4, Width == 1 ? 8 : 4)))
void linear_decode_kernel(const int32_t* md_indices, const int32_t* md_cu,
                          const int32_t* md_accepted, int md_num_v_heads, const LinearParams p) {
  constexpr int kBlock = 64 * kTileWaves;
  constexpr int kPc = kDim / kTileWaves / 2;   // 16-byte tile pieces per lane
  constexpr int kPair = 4 * kTileWaves;        // rows that a piece pair of every wave covers
  constexpr int kRows = kPc / 2;               // V rows per lane
  const int tile = blockIdx.x;
  const int request = tile / md_num_v_heads;
  const int head = tile - request * md_num_v_heads;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;

  const int32_t* req_slots = md_indices + static_cast<int64_t>(request) * Width;
  const int64_t bos = row_of(md_cu[request], p.num_tokens);
  const int64_t eos = row_of(md_cu[request + 1], p.num_tokens);
  const int accepted = md_accepted[request];
  int slot[Width];
#pragma unroll
  for (int t = 0; t < Width; ++t) slot[t] = req_slots[t];
  const int64_t count = eos - bos;
  if (count <= 0) return;
  int source = 0;
#pragma unroll
  for (int t = 0; t < Width; ++t)
    if (accepted == t + 1) source = slot[t];
  if (!live_slot(source, p.num_slots) || count > Width) {   // zero outputs, state untouched
    for (int64_t i = tid; i < count * kDim; i += kBlock)
      p.out[((bos + (i >> 7)) * p.num_v_heads + head) * kDim + (i & (kDim - 1))] = 0;
    return;
  }
  const int num_tokens = static_cast<int>(count);

  const int kq = lane & 15;
  const int row_base = 4 * wave + (lane >> 4);   // V row of the lane's piece 0
  const int key_head = head / p.group;
  // token t (past the request's last token a copy of that one: its state is not stored, its
  // outputs are not written, and the loops have no branches)
  LinearToken<kRows> in[Width];
#pragma unroll
  for (int t = 0; t < Width; ++t) {
    const int64_t token = bos + min(t, num_tokens - 1);
    const uint16_t* row = p.qkv + token * p.qkv_row;
    const uint16_t* q = row + key_head * kDim + 4 * kq;
    const uint16_t* k = row + (p.num_k_heads + key_head) * kDim + 4 * kq;
    const uint16_t* v = row + (2 * p.num_k_heads + head) * kDim + row_base;
    __builtin_memcpy(in[t].q, q, 8);
    __builtin_memcpy(in[t].q + 4, q + 64, 8);
    __builtin_memcpy(in[t].k, k, 8);
    __builtin_memcpy(in[t].k + 4, k + 64, 8);
#pragma unroll
    for (int i = 0; i < kRows; ++i) in[t].v[i] = v[i * kPair];
    in[t].decay = p.log_decay[token * p.decay_row + head];
  }
  __builtin_amdgcn_sched_barrier(0);

  const int64_t head_offset = static_cast<int64_t>(head) * kDim * kDim;
  const uint32_t lane_bytes = static_cast<uint32_t>(row_base * kDim + kq * 4) * 4u;
  const __amdgpu_buffer_rsrc_t src = buffer_rsrc(
      p.state + static_cast<int64_t>(source) * p.state_slot + head_offset, kTileBytes);
  f32x4 s[kPc];
#pragma unroll
  for (int j = 0; j < kPc; ++j) {
    s[j] = buffer_load16<LoadPol>(src, lane_bytes + tile_piece_bytes<kPair>(j));
    __builtin_amdgcn_sched_barrier(0);   // in order: a row pair waits for its own loads only
  }
  // token t's state goes to slot indices[r, t]; without one, to a resource over 0 bytes, whose
  // stores the hardware drops
  __amdgpu_buffer_rsrc_t dst[Width];
#pragma unroll
  for (int t = 0; t < Width; ++t) {
    const bool stored = t < num_tokens && live_slot(slot[t], p.num_slots);
    dst[t] = buffer_rsrc(
        p.state + static_cast<int64_t>(stored ? slot[t] : 0) * p.state_slot + head_offset,
        stored ? kTileBytes : 0);
  }
#pragma unroll
  for (int t = 0; t < Width; ++t) in[t].decay = __expf(in[t].decay);

  __shared__ float s_o[Width][kDim];
#pragma unroll
  for (int c = 0; c < kRows; c += 2) {   // two V rows
#pragma unroll
    for (int t = 0; t < Width; ++t) {
      f32x4 k0, k1, q0, q1;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        k0[e] = bf16_to_f32(in[t].k[e]);
        k1[e] = bf16_to_f32(in[t].k[4 + e]);
        q0[e] = bf16_to_f32(in[t].q[e]);
        q1[e] = bf16_to_f32(in[t].q[4 + e]);
      }
      float o[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float v = bf16_to_f32(in[t].v[c + i]);
        f32x4& s0 = s[2 * (c + i)];
        f32x4& s1 = s[2 * (c + i) + 1];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s0[e] = fmaf(v, k0[e], s0[e] * in[t].decay);
          s1[e] = fmaf(v, k1[e], s1[e] * in[t].decay);
        }
        buffer_store16<StorePol>(s0, dst[t], lane_bytes + tile_piece_bytes<kPair>(2 * (c + i)));
        buffer_store16<StorePol>(s1, dst[t], lane_bytes + tile_piece_bytes<kPair>(2 * (c + i) + 1));
        o[i] = dot8(s0, s1, q0, q1);
      }
      row_sum2(o[0], o[1]);
      if (kq == 0) {
        s_o[t][row_base + c * kPair] = o[0];
        s_o[t][row_base + (c + 1) * kPair] = o[1];
      }
    }
  }
  lds_barrier();

  // ---- outputs of token `wave`: two columns a lane ----
  if (wave < num_tokens) {
    const int64_t token = bos + wave;
    float o[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) o[e] = p.scale * s_o[wave][2 * lane + e];
    if (p.gate != nullptr) {
      const float rstd =
          fast_rsqrt(wave_sum(fmaf(o[0], o[0], o[1] * o[1])) * (1.0f / kDim) + p.eps);
      const uint16_t* gate = p.gate + token * p.gate_row + head * kDim + 2 * lane;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        o[e] = ((o[e] * rstd) * load_param(p.norm_weight, 2 * lane + e, p.weight_bf16)) *
               silu(bf16_to_f32(gate[e]));
    }
    uint16_t* row = p.out + (token * p.num_v_heads + head) * kDim + 2 * lane;
#pragma unroll
    for (int e = 0; e < 2; ++e) row[e] = f32_to_bf16(o[e]);
  }
}

template <int LoadPol, int StorePol, int Width>
void launch_width(const LinearParams& p, uint32_t blocks, hipStream_t stream) {
  hipLaunchKernelGGL((linear_decode_kernel<LoadPol, StorePol, Width>), dim3(blocks),
                     dim3(64 * kTileWaves), 0, stream, p.indices, p.cu, p.accepted, p.num_v_heads, p);
}

// Cache policies as measured on MI355X (us; "hot" the same slots every step, "cold" slot sets
// rotated beyond the 256 MB Infinity Cache), 32 requests x 32 heads hot / cold, 119 x 48 cold, and
// a 4-token verify of 64 x 32 hot / cold:
//   non-temporal system-scope loads and stores   25.5 / 25.4   122    81.5 / 85.8   (stream)
//   plain loads, system-scope stores             21.1 / 27.6   134    88.5 / 98.3   (keep, one token)
//   plain loads, non-temporal stores             21.8 / 29.9   138    66.1 / 96.3   (keep, verify)
//   plain loads and stores                       21.8 / 29.4   137    103 / 109
// Other shapes under the stream policy: 4 waves 25.7 / 25.9, 135, 112 / 115; 8 waves 26.9 / 27.0,
// 129, 89 / 95.  At 5.1 TB/s, a large copy's rate, these calls' bytes take 26.4, 146 and 92.8 us.
void launch_linear(const LinearParams& p, int width, bool keep, uint32_t blocks, hipStream_t s) {
  switch (width) {
    case 1: return keep ? launch_width<kPolPlain, kPolSys, 1>(p, blocks, s)
                        : launch_width<kPolNTSys, kPolNTSys, 1>(p, blocks, s);
    case 2: return keep ? launch_width<kPolPlain, kPolNT, 2>(p, blocks, s)
                        : launch_width<kPolNTSys, kPolNTSys, 2>(p, blocks, s);
    case 3: return keep ? launch_width<kPolPlain, kPolNT, 3>(p, blocks, s)
                        : launch_width<kPolNTSys, kPolNTSys, 3>(p, blocks, s);
    default: return keep ? launch_width<kPolPlain, kPolNT, 4>(p, blocks, s)
                         : launch_width<kPolNTSys, kPolNTSys, 4>(p, blocks, s);
  }
}

}  // namespace
}  // namespace ld

extern "C" int ld_linear_decode(const ld_linear_decode_args* args, void* stream) {
  using namespace ld;
  if (args == nullptr) return fail(LD_ERR_INVALID_ARGUMENT, "ld_linear_decode: args is NULL");
  const ld_linear_decode_args& a = *args;
  if (a.width < 1 || a.width > LD_MAX_TOKENS)
    return fail(LD_ERR_INVALID_ARGUMENT, "decode/MTP supports 1 through 4 tokens per request");
  if (a.cache_policy != LD_CACHE_KEEP && a.cache_policy != LD_CACHE_STREAM)
    return fail(LD_ERR_INVALID_ARGUMENT, "cache_policy must be LD_CACHE_KEEP or LD_CACHE_STREAM");
  LinearParams p{};
  const int rc = linear_params(a, a.num_requests, "num_requests must be >= 0", p);
  if (rc != LD_OK || a.num_requests == 0) return rc;
  if (!a.qkv || !a.log_decay || !a.indices || !a.cu || !a.accepted || !a.state || !a.out)
    return fail(LD_ERR_INVALID_ARGUMENT, "ld_linear_decode: NULL tensor pointer");
  const int64_t blocks = static_cast<int64_t>(a.num_requests) * a.num_v_heads;
  if (blocks > 0x3fffff) return fail(LD_ERR_INVALID_ARGUMENT, "too many (request, head) tiles");
  p.indices = a.indices;
  p.cu = a.cu;
  p.accepted = a.accepted;
  launch_linear(p, a.width, a.cache_policy == LD_CACHE_KEEP, static_cast<uint32_t>(blocks),
                static_cast<hipStream_t>(stream));
  return check_launch("ld_linear_decode");
}
