// RMSNorm and position rotation of the q and k heads of qkv rows, in one pass and in place, for
// gfx950:
//   y = x * rsqrt(mean(x^2) + eps) * w ;  pairs of y turned by positions[token] * inv_freq[i]
// in fp32, rounded to bf16 once.
//
// Bound by memory: 512 bytes a head and token against about 90 vector instructions per 4 heads.
// A wave takes one token and walks its heads four at a time, 16 lanes a head, 8 consecutive
// elements (16 bytes) a lane.  A lane's 8 angles are the same for every head of the token, so it
// forms them once: the product and its reduction to a fraction of a turn in 64 bits (positions
// of millions times frequencies near 1 leave 32 bits no fraction), sine and cosine in fp32.  No
// LDS and no barrier.
#include "gdn_common.h"
#include "lightdelta_linear_hip.h"

namespace ld {
namespace {

constexpr int kHeadsPerRound = 4;

struct NormRopeParams {
  uint16_t* qkv;
  int64_t row;
  const void* q_weight;
  const void* k_weight;
  const void* positions;
  const float* inv_freq;
  int64_t num_tokens;
  int32_t q_heads;
  int32_t heads;    // q_heads + k_heads
  int32_t half;     // rotary / 2
  int32_t rounds;   // rounds of 4 heads a wave takes
  int32_t splits;   // waves a token
  int32_t q_bf16, k_bf16, positions64;
  float eps;
};

// Interleaved: a pair's elements are neighbours in a lane; else `half` elements apart, the
// partner's lane half / 8 lanes up (first half) or down.
template <bool Interleaved>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(const NormRopeParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWaves + (threadIdx.x >> 6);
  const int64_t token = unit / p.splits;
  if (token >= p.num_tokens) return;
  const int first = static_cast<int>(unit - token * p.splits) * p.rounds * kHeadsPerRound;
  const int li = lane & 15;
  const int sub = lane >> 4;
  uint16_t* const row = p.qkv + token * p.row + 8 * li;

  const double position =
      p.positions64 ? static_cast<double>(static_cast<const int64_t*>(p.positions)[token])
                    : static_cast<double>(static_cast<const int32_t*>(p.positions)[token]);
  // c[e], s[e]: cosine and signed sine of element 8 li + e; (1, 0) past the rotated ones
  float c[8], s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int element = 8 * li + e;
    const bool turned = element < 2 * p.half;
    const int i = Interleaved ? element >> 1 : (element < p.half ? element : element - p.half);
    c[e] = 1.0f;
    s[e] = 0.0f;
    if (turned) {
      const double turns = position * static_cast<double>(p.inv_freq[i]) * 0.15915494309189535;
      const float fraction = static_cast<float>(turns - rint(turns));
      c[e] = __builtin_amdgcn_cosf(fraction);
      const float sine = __builtin_amdgcn_sinf(fraction);
      const bool is_first = Interleaved ? (e & 1) == 0 : element < p.half;
      s[e] = is_first ? -sine : sine;
    }
  }
  const int partner = Interleaved ? lane : (8 * li < p.half ? lane + (p.half >> 3)
                                            : 8 * li < 2 * p.half ? lane - (p.half >> 3)
                                                                  : lane);
  for (int round = 0; round < p.rounds; ++round) {
    const int head = first + round * kHeadsPerRound + sub;
    const bool live = head < p.heads;
    if (first + round * kHeadsPerRound >= p.heads) return;
    const int at = live ? head : p.heads - 1;
    uint16_t raw[8];
    __builtin_memcpy(raw, row + static_cast<int64_t>(at) * kDim, 16);
    const bool is_q = at < p.q_heads;
    float y[8];
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[e] = bf16_to_f32(raw[e]);
      ss = fmaf(y[e], y[e], ss);
    }
    ss += dpp<kDppQuadXor1>(ss);
    ss += dpp<kDppQuadXor2>(ss);
    ss += dpp<kDppRowHalfMirror>(ss);
    ss += dpp<kDppRowMirror>(ss);
    const float rstd = fast_rsqrt(ss * (1.0f / kDim) + p.eps);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      y[e] = (y[e] * rstd) * load_param(is_q ? p.q_weight : p.k_weight, 8 * li + e,
                                        is_q ? p.q_bf16 : p.k_bf16);
    float other[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) other[e] = Interleaved ? y[e ^ 1] : __shfl(y[e], partner);
#pragma unroll
    for (int e = 0; e < 8; ++e) raw[e] = f32_to_bf16(fmaf(y[e], c[e], other[e] * s[e]));
    if (live) __builtin_memcpy(row + static_cast<int64_t>(at) * kDim, raw, 16);
  }
}

}  // namespace
}  // namespace ld

extern "C" int ld_norm_rope(const ld_norm_rope_args* args, void* stream) {
  using namespace ld;
  if (args == nullptr) return fail(LD_ERR_INVALID_ARGUMENT, "ld_norm_rope: args is NULL");
  const ld_norm_rope_args& a = *args;
  if (a.num_tokens < 0 || a.q_heads < 0 || a.k_heads < 0)
    return fail(LD_ERR_INVALID_ARGUMENT, "num_tokens, q_heads and k_heads must be >= 0");
  if (!(a.eps > 0.0f)) return fail(LD_ERR_INVALID_ARGUMENT, "norm epsilon must be positive");
  if (a.rotary < 0 || a.rotary > kDim || a.rotary % (a.interleaved ? 2 : 16) != 0)
    return fail(LD_ERR_INVALID_ARGUMENT,
                "rotary must be at most 128 and a multiple of 16 (halves) or 2 (interleaved)");
  for (const int32_t dtype : {a.q_weight_dtype, a.k_weight_dtype})
    if (dtype != LD_DTYPE_F32 && dtype != LD_DTYPE_BF16)
      return fail(LD_ERR_INVALID_ARGUMENT, "weights must be FP32/BF16");
  const int64_t heads = static_cast<int64_t>(a.q_heads) + a.k_heads;
  if (heads > (1 << 20)) return fail(LD_ERR_INVALID_ARGUMENT, "too many heads");
  if (a.num_tokens == 0 || heads == 0) return LD_OK;
  if (!a.qkv || !a.positions || (a.q_heads > 0 && !a.q_weight) || (a.k_heads > 0 && !a.k_weight) ||
      (a.rotary > 0 && !a.inv_freq))
    return fail(LD_ERR_INVALID_ARGUMENT, "ld_norm_rope: NULL tensor pointer");
  if (a.num_tokens > 1 && a.qkv_row_stride < heads * kDim)
    return fail(LD_ERR_INVALID_ARGUMENT, "qkv rows must not overlap");
  const int64_t rounds = (heads + kHeadsPerRound - 1) / kHeadsPerRound;
  NormRopeParams p{};
  p.qkv = static_cast<uint16_t*>(a.qkv);
  p.row = a.qkv_row_stride;
  p.q_weight = a.q_weight;
  p.k_weight = a.k_weight;
  p.positions = a.positions;
  p.inv_freq = a.inv_freq;
  p.num_tokens = a.num_tokens;
  p.q_heads = a.q_heads;
  p.heads = static_cast<int32_t>(heads);
  p.half = a.rotary / 2;
  p.rounds = static_cast<int32_t>(rounds);
  p.splits = 1;
  p.q_bf16 = a.q_weight_dtype == LD_DTYPE_BF16;
  p.k_bf16 = a.k_weight_dtype == LD_DTYPE_BF16;
  p.positions64 = a.positions_int64;
  p.eps = a.eps;
  const int64_t blocks = (a.num_tokens * p.splits + kWaves - 1) / kWaves;
  if (blocks > 0xffffff) return fail(LD_ERR_INVALID_ARGUMENT, "too many tokens");
  const auto kernel = a.interleaved ? norm_rope_kernel<true> : norm_rope_kernel<false>;
  hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), p);
  return check_launch("ld_norm_rope");
}
