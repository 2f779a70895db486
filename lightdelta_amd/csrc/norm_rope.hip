// RMSNorm and position rotation of the q and k heads of qkv rows, in one pass and in place, for
// gfx950:
//   y = x * rsqrt(mean(x^2) + eps) * w ;  pairs of y turned by positions[token] * inv_freq[i]
// in fp32, rounded to bf16 once.
//
// Bound by memory: 512 bytes a head and token against 164 vector instructions per 4 heads.
// A wave takes one token and four heads at a time, 16 lanes a head, 8 consecutive elements (16
// bytes) a lane, four rounds of loads in flight.  The token's angles are formed once, one a lane,
// and spread through LDS: the product and its reduction to a fraction of a turn in pairs of doubles
// (turn_fraction), sine and cosine in fp32.  A pair's other element comes from a lane of the same 16 by DPP.
//
// 32,768 tokens of 16 + 16 heads: 101 us, 5.3 TB/s (260 with a round at a time, an angle per element and
// pairs by shuffles); one token of them 2.5 us.  Few tokens are split over waves by rounds, so that a
// small launch's latency is one batch's.  With positions of several axes an angle's lane picks its own
// position; 16,384 tokens of 32 + 8 heads, half of each rotated: 73 us, 4.6 TB/s.
#include <algorithm>
#include <type_traits>

#include "gdn_common.h"
#include "lightdelta_attention_hip.h"

namespace ld {
namespace {

constexpr int kHeadsPerRound = 4;

constexpr int kBatch = 4;   // rounds whose loads are in flight together

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
  const int32_t* axes;   // with several axes: that of each angle
  int64_t axis_stride;   // between the positions of two axes
  int32_t num_axes;
};

// Where a lane finds the other elements of its pairs: its own (neighbours, interleaved), the lane
// whose number differs in bit D, or (any other half) one that a shuffle names.
constexpr int kOwn = 0;
constexpr int kShuffle = -1;

// position * inv_freq / (2 pi) less the nearest whole number, for any position: positions of millions
// leave 32 bits no fraction, 2^50 none to 64.  1 / (2 pi), and with it a turn a position, is a sum
// of two doubles, and the position one of its upper and lower 32 bits, so that what a product with
// the first double rounds off comes back by fma: within 2^-44 of a turn for frequencies up to 1.
__device__ __forceinline__ double turn_part(double position, double first, double second) {
  return fma(position, first, -rint(position * first)) + position * second;
}
__device__ __forceinline__ float turn_fraction(int64_t position, float inv_freq) {
  constexpr double kTurn = 0x1.45f306dc9c883p-3, kTurnRest = -0x1.6b01ec5417056p-57;
  const double first = inv_freq * kTurn;
  const double second = fma(static_cast<double>(inv_freq), kTurn, -first) + inv_freq * kTurnRest;
  const double upper = static_cast<double>(static_cast<int32_t>(position >> 32)) * 0x1p32;
  const double lower = static_cast<double>(static_cast<uint32_t>(position));
  const double turns = turn_part(upper, first, second) + turn_part(lower, first, second);
  return static_cast<float>(turns - rint(turns));
}

template <int D>
__device__ __forceinline__ float partner(float y, int lane) {
  if constexpr (D == 8) return dpp<0x128>(y);                                  // row_ror:8
  if constexpr (D == 4) return dpp<0x1B>(dpp<kDppRowHalfMirror>(y));           // ^ 7, ^ 3
  if constexpr (D == 2) return dpp<kDppQuadXor2>(y);
  if constexpr (D == 1) return dpp<kDppQuadXor1>(y);
  return __shfl(y, lane);
}

__device__ __forceinline__ void load_weights(float (&w)[8], const void* from, int at, bool bf16) {
  if (bf16) {
    uint16_t raw[8];
    __builtin_memcpy(raw, static_cast<const uint16_t*>(from) + at, 16);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = bf16_to_f32(raw[e]);
  } else {
    __builtin_memcpy(w, static_cast<const float*>(from) + at, 32);
  }
}

template <int D, bool Axes>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(const NormRopeParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWaves +
                       __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t token = unit / p.splits;
  if (token >= p.num_tokens) return;
  const int first = static_cast<int>(unit - token * p.splits) * p.rounds * kHeadsPerRound;
  const int li = lane & 15;
  const int sub = lane >> 4;
  uint16_t* const row = p.qkv + token * p.row + 8 * li;

  // the heads of round r: lanes past the last head repeat it and store nothing
  u32x4 raw[kBatch];
  auto head_of = [&](int r) { return first + r * kHeadsPerRound + sub; };
  auto load = [&](int r) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      __builtin_memcpy(&raw[b], row + static_cast<int64_t>(min(head_of(r + b), p.heads - 1)) * kDim, 16);
  };
  load(0);
  float wq[8] = {}, wk[8] = {};
  if (p.q_heads > 0) load_weights(wq, p.q_weight, 8 * li, p.q_bf16);
  if (p.q_heads < p.heads) load_weights(wk, p.k_weight, 8 * li, p.k_bf16);
  // angle `lane` of the token, by one lane each, and from LDS (the wave's own, so without a barrier)
  // the lane's eight; element 8 li + e has angle first + e (halves) or first + e / 2 (interleaved)
  __shared__ __attribute__((aligned(16))) float angles[kWaves][2][64];
  float* const mine = angles[threadIdx.x >> 6][0];
  if (lane < p.half) {
    int64_t at = token;
    bool turns = true;
    if constexpr (Axes) {   // (an axis that there is not: no turn)
      const int axis = p.axes[lane];
      turns = axis >= 0 && axis < p.num_axes;
      at += (turns ? axis : 0) * p.axis_stride;
    }
    const int64_t position = !turns          ? 0
                             : p.positions64 ? static_cast<const int64_t*>(p.positions)[at]
                                             : static_cast<const int32_t*>(p.positions)[at];
    const float fraction = turn_fraction(position, p.inv_freq[lane]);
    mine[lane] = __builtin_amdgcn_cosf(fraction);
    mine[64 + lane] = __builtin_amdgcn_sinf(fraction);
  }
  asm volatile("" ::: "memory");   // (a wave's LDS operations run in order)
  const int element = 8 * li;
  const bool second = D != kOwn && element >= p.half;   // the lane holds pairs' second elements
  const int angle = D == kOwn ? element >> 1 : min(second ? element - p.half : element, 56);
  float c[8], s[8];
  bool turned[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int i = angle + (D == kOwn ? e >> 1 : e);
    c[e] = mine[i];
    s[e] = (D == kOwn ? (e & 1) != 0 : second) ? mine[64 + i] : -mine[64 + i];
    turned[e] = element + e < 2 * p.half;
  }
  int other_lane = lane;
  if (D == kShuffle && 8 * li < 2 * p.half)
    other_lane = 8 * li < p.half ? lane + (p.half >> 3) : lane - (p.half >> 3);

  for (int r = 0; r < p.rounds; r += kBatch) {
    u32x4 now[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) now[b] = raw[b];
    if (r + kBatch < p.rounds) load(r + kBatch);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (r + b >= p.rounds || first + (r + b) * kHeadsPerRound >= p.heads) break;
      const int head = head_of(r + b);
      const bool is_q = head < p.q_heads;
      float y[8];
      float ss = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t pair = now[b][e >> 1];
        y[e] = __uint_as_float(e & 1 ? pair & 0xffff0000u : pair << 16);
        ss = fmaf(y[e], y[e], ss);
      }
      ss += dpp<kDppQuadXor1>(ss);
      ss += dpp<kDppQuadXor2>(ss);
      ss += dpp<kDppRowHalfMirror>(ss);
      ss += dpp<kDppRowMirror>(ss);
      const float rstd = fast_rsqrt(ss * (1.0f / kDim) + p.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = (y[e] * rstd) * (is_q ? wq[e] : wk[e]);
      float z[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float other = D == kOwn ? y[e ^ 1] : partner<D>(y[e], other_lane);
        z[e] = turned[e] ? fmaf(y[e], c[e], other * s[e]) : y[e];
      }
      u32x4 bits;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        bits[e] = f32_to_bf16(z[2 * e]) | static_cast<uint32_t>(f32_to_bf16(z[2 * e + 1])) << 16;
      if (head < p.heads) __builtin_memcpy(row + static_cast<int64_t>(head) * kDim, &bits, 16);
    }
  }
}

}  // namespace
}  // namespace ld

namespace ld {
namespace {

int launch_norm_rope(const ld_norm_rope_args* args, const ld_rope_axes* axes, const char* what,
                     void* stream) {
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
  // A wave takes all rounds of its token where tokens fill the chip (four waves a SIMD), else as
  // many waves as rounds share one.
  const int64_t rounds = (heads + kHeadsPerRound - 1) / kHeadsPerRound;
  const int64_t splits = a.num_tokens >= 4096 ? 1 : std::min<int64_t>(rounds, 4096 / a.num_tokens);
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
  p.rounds = static_cast<int32_t>((rounds + splits - 1) / splits);
  p.splits = static_cast<int32_t>((rounds + p.rounds - 1) / p.rounds);
  p.q_bf16 = a.q_weight_dtype == LD_DTYPE_BF16;
  p.k_bf16 = a.k_weight_dtype == LD_DTYPE_BF16;
  p.positions64 = a.positions_int64;
  p.eps = a.eps;
  if (axes != nullptr) {
    p.axes = axes->axes;
    p.axis_stride = axes->position_axis_stride;
    p.num_axes = axes->num_axes;
  }
  const int64_t blocks = (a.num_tokens * p.splits + kWaves - 1) / kWaves;
  if (blocks > 0xffffff) return fail(LD_ERR_INVALID_ARGUMENT, "too many tokens");
  const auto pick = [&](auto several) {
    constexpr bool kAxes = decltype(several)::value;
    return a.interleaved    ? norm_rope_kernel<kOwn, kAxes>
           : p.half == 64   ? norm_rope_kernel<8, kAxes>
           : p.half == 32   ? norm_rope_kernel<4, kAxes>
           : p.half == 16   ? norm_rope_kernel<2, kAxes>
           : p.half == 8    ? norm_rope_kernel<1, kAxes>
                            : norm_rope_kernel<kShuffle, kAxes>;
  };
  const auto kernel = axes != nullptr ? pick(std::true_type{}) : pick(std::false_type{});
  hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), p);
  return check_launch(what);
}

}  // namespace
}  // namespace ld

extern "C" int ld_norm_rope(const ld_norm_rope_args* args, void* stream) {
  return ld::launch_norm_rope(args, nullptr, "ld_norm_rope", stream);
}

extern "C" int ld_norm_rope_axes(const ld_norm_rope_args* args, const ld_rope_axes* axes,
                                 void* stream) {
  using namespace ld;
  if (axes == nullptr) return fail(LD_ERR_INVALID_ARGUMENT, "ld_norm_rope_axes: axes is NULL");
  if (axes->num_axes < 1) return fail(LD_ERR_INVALID_ARGUMENT, "num_axes must be >= 1");
  if (args != nullptr && args->rotary > 0 && args->num_tokens > 0 && axes->axes == nullptr)
    return fail(LD_ERR_INVALID_ARGUMENT, "ld_norm_rope_axes: NULL tensor pointer");
  return launch_norm_rope(args, axes, "ld_norm_rope_axes", stream);
}
