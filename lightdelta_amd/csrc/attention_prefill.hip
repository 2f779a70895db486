// Attention of prompts over the paged 8-bit cache.
#include "attention_common.h"

namespace ld {
namespace {

struct AttentionParams {
  Cache cache;
  Attention a;
};

// A wave takes one row and q head: 64 tokens at a time, a token's score by a lane, then two
// elements of the output by a lane, with the running maximum and sum of the softmax.
__global__ __launch_bounds__(64) void attention_rows_kernel(const AttentionParams p) {
  const Cache& c = p.cache;
  const Attention& a = p.a;
  const int64_t row = blockIdx.x / a.q_heads;
  const int head = static_cast<int>(blockIdx.x - row * a.q_heads);
  const int r = request_at(c, row);
  const Request req = request_of(c, r);
  if (row < req.first || row >= req.last) return;
  const int lane = threadIdx.x;
  const int kv = head / a.group;
  const int64_t position = row + req.shift;
  int64_t sees = min(position + 1, static_cast<int64_t>(req.tokens));
  __shared__ float query[kDim];
  __shared__ float weight[64];
  for (int d = lane; d < kDim; d += 64) query[d] = bf16_to_f32(a.q[row * a.q_row + head * kDim + d]);
  __syncthreads();
  float top = -3.4028235e38f, total = 0.0f, o0 = 0.0f, o1 = 0.0f;
  bool any = false;
  for (int64_t t0 = 0; t0 < sees; t0 += 64) {
    const int64_t t = t0 + lane;
    const int page = t < sees ? c.pages[r * c.pages_row + (t >> c.page_log2)] : 0;
    const bool live = live_page(c, page);
    float s = -__builtin_inff();
    if (live) {
      const int at = static_cast<int>(t) & ((1 << c.page_log2) - 1);
      const uint32_t* const k = reinterpret_cast<const uint32_t*>(k_tile(c, page, kv));
      float sum = 0.0f;
      for (int d = 0; d < kDim; d += 4) {
        const uint32_t x = k[((d >> 4 << c.page_log2) + at) * 4 + (d >> 2 & 3)];
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(x, false);
        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(x, true);
        sum = fmaf(lo[0], query[d], fmaf(lo[1], query[d + 1], sum));
        sum = fmaf(hi[0], query[d + 2], fmaf(hi[1], query[d + 3], sum));
      }
      s = sum * scale_value(c.k_scale[page * c.k_scale_page + kv]);
    }
    float most = s;
    for (int d = 32; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
    const float now = fmaxf(top, most);
    const float keep = exp2f((top - now) * a.log2_scale);
    const float w = live ? exp2f((s - now) * a.log2_scale) : 0.0f;
    any = any || __any(live);
    float sum = w;
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    total = total * keep + sum;
    o0 *= keep;
    o1 *= keep;
    top = now;
    weight[lane] = w;
    __syncthreads();
    for (int j = 0; j < 64 && t0 + j < sees; ++j) {
      const int pg = __shfl(page, j);
      if (!live_page(c, pg)) continue;
      const int at = static_cast<int>(t0 + j) & ((1 << c.page_log2) - 1);
      const uint8_t* const v = v_tile(c, pg, kv) + (at >> 4) * (kDim * 16) + (at & 15);
      const auto x = __builtin_amdgcn_cvt_pk_f32_fp8(v[lane * 32] | v[lane * 32 + 16] << 8, false);
      const float vs = scale_value(c.v_scale[pg * c.v_scale_page + kv]);
      o0 = fmaf(weight[j] * vs, x[0], o0);
      o1 = fmaf(weight[j] * vs, x[1], o1);
    }
    __syncthreads();
  }
  const float inverse = 1.0f / total;
  o0 = any ? o0 * inverse : 0.0f;
  o1 = any ? o1 * inverse : 0.0f;
  if (a.gate != nullptr && any) {
    const uint16_t* const g = a.gate + row * a.gate_row + head * kDim + 2 * lane;
    o0 *= sigmoid(bf16_to_f32(g[0]));
    o1 *= sigmoid(bf16_to_f32(g[1]));
  }
  const uint32_t bits = f32_to_bf16(o0) | static_cast<uint32_t>(f32_to_bf16(o1)) << 16;
  __builtin_memcpy(a.out + (row * a.q_heads + head) * kDim + 2 * lane, &bits, 4);
}

}  // namespace
}  // namespace ld

extern "C" int64_t ld_attention_prefill_workspace_bytes(const ld_paged_cache*,
                                                        const ld_attention_args*) {
  return 0;
}

extern "C" int ld_attention_prefill(const ld_paged_cache* cache, const ld_attention_args* args,
                                    void* stream) {
  using namespace ld;
  AttentionParams p{};
  if (const int rc = cache_params(cache, p.cache)) return rc;
  if (const int rc = attention_params(*cache, args, p.a)) return rc;
  if (p.cache.requests == 0) return LD_OK;
  const int64_t blocks = p.cache.num_tokens * p.a.q_heads;
  if (blocks > 0x7fffffff) return fail(LD_ERR_INVALID_ARGUMENT, "too many rows and heads");
  hipLaunchKernelGGL(attention_rows_kernel, dim3(static_cast<uint32_t>(blocks)), dim3(64), 0,
                     static_cast<hipStream_t>(stream), p);
  return check_launch("ld_attention_prefill");
}
