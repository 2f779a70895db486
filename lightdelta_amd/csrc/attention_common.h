// Definitions shared by the paged 8-bit cache and the attention over it (cache_io.hip,
// attention_decode.hip, attention_prefill.hip).
#pragma once

#include "matrix_common.h"
#include "lightdelta_attention_hip.h"

namespace ld {

constexpr int kScaleLow = -100, kScaleHigh = 119;   // exponents of a scale
constexpr int kScaleBias = 127;

struct Cache {
  uint8_t* k;
  uint8_t* v;
  uint8_t* k_scale;
  uint8_t* v_scale;
  int64_t k_page, v_page;              // bytes
  int64_t k_scale_page, v_scale_page;
  const int32_t* pages;
  int64_t pages_row;
  const int32_t* cu;
  const int32_t* lengths;
  int64_t num_tokens;
  int32_t table_width;
  int32_t num_pages;
  int32_t page_log2;
  int32_t kv_heads;
  int32_t requests;
};

// The checks and parameters of every entry point; LD_OK, or an error code with its message.
inline int cache_params(const ld_paged_cache* from, Cache& c) {
  if (from == nullptr) return fail(LD_ERR_INVALID_ARGUMENT, "cache is NULL");
  const ld_paged_cache& a = *from;
  if (a.num_requests < 0 || a.num_tokens < 0 || a.num_pages < 0 || a.table_width < 0)
    return fail(LD_ERR_INVALID_ARGUMENT,
                "num_requests, num_tokens, num_pages and table_width must be >= 0");
  if (a.num_kv_heads <= 0 || a.num_kv_heads > 1 << 16)
    return fail(LD_ERR_INVALID_ARGUMENT, "num_kv_heads must be 1 through 2^16");
  if (a.page_size != 16 && a.page_size != 32 && a.page_size != 64 && a.page_size != 128)
    return fail(LD_ERR_INVALID_ARGUMENT, "page_size must be 16, 32, 64 or 128");
  if (a.num_tokens >= int64_t{1} << 31)
    return fail(LD_ERR_INVALID_ARGUMENT, "too many tokens");
  c = Cache{};
  if (a.num_requests == 0 || a.num_tokens == 0) return LD_OK;
  if ((a.num_pages > 0 && (!a.k || !a.v || !a.k_scale || !a.v_scale)) || !a.cu || !a.lengths ||
      (a.table_width > 0 && !a.pages))
    return fail(LD_ERR_INVALID_ARGUMENT, "cache: NULL tensor pointer");
  if (!aligned16(a.k) || !aligned16(a.v) || (a.k_page_stride & 15) != 0 ||
      (a.v_page_stride & 15) != 0)
    return fail(LD_ERR_INVALID_ARGUMENT, "cache pages must be 16-byte aligned");
  c.k = static_cast<uint8_t*>(a.k);
  c.v = static_cast<uint8_t*>(a.v);
  c.k_scale = a.k_scale;
  c.v_scale = a.v_scale;
  c.k_page = a.k_page_stride;
  c.v_page = a.v_page_stride;
  c.k_scale_page = a.k_scale_stride;
  c.v_scale_page = a.v_scale_stride;
  c.pages = a.pages;
  c.pages_row = a.pages_row_stride;
  c.cu = a.cu;
  c.lengths = a.lengths;
  c.num_tokens = a.num_tokens;
  c.table_width = a.num_pages > 1 ? a.table_width : 0;   // (without a page none has a place)
  c.num_pages = a.num_pages;
  c.page_log2 = __builtin_ctz(a.page_size);
  c.kv_heads = a.num_kv_heads;
  c.requests = a.num_requests;
  return LD_OK;
}

struct Attention {
  const uint16_t* q;
  int64_t q_row;
  const uint16_t* gate;   // NULL: none
  int64_t gate_row;
  uint16_t* out;
  float* workspace;
  int32_t q_heads;
  int32_t group;          // q_heads / kv_heads
  int32_t width;          // decode: rows of a request at most
  float log2_scale;       // scale * log2(e)
};

// The same of the attention entry points.
inline int attention_params(const ld_paged_cache& c, const ld_attention_args* from, Attention& p) {
  if (from == nullptr) return fail(LD_ERR_INVALID_ARGUMENT, "args is NULL");
  const ld_attention_args& a = *from;
  if (a.num_q_heads <= 0 || a.num_q_heads > 1 << 16 || a.num_q_heads % c.num_kv_heads != 0)
    return fail(LD_ERR_INVALID_ARGUMENT,
                "num_q_heads must be a positive multiple of num_kv_heads, at most 2^16");
  const float log2_scale = a.scale * 1.44269504088896340736f;
  if (!(a.scale > 0.0f && log2_scale <= 3.4028235e38f))
    return fail(LD_ERR_INVALID_ARGUMENT, "scale must be positive, log2(e) times it finite");
  p = Attention{};
  if (c.num_requests == 0 || c.num_tokens == 0) return LD_OK;
  if (!a.q || !a.out) return fail(LD_ERR_INVALID_ARGUMENT, "attention: NULL tensor pointer");
  p.q = static_cast<const uint16_t*>(a.q);
  p.q_row = a.q_row_stride;
  p.gate = static_cast<const uint16_t*>(a.gate);
  p.gate_row = a.gate_row_stride;
  p.out = static_cast<uint16_t*>(a.out);
  p.workspace = static_cast<float*>(a.workspace);
  p.q_heads = a.num_q_heads;
  p.group = a.num_q_heads / c.num_kv_heads;
  p.width = a.width;
  p.log2_scale = log2_scale;
  return LD_OK;
}

// A launch has fewer than 2^32 threads in a dimension.
inline bool launches(int64_t blocks, int threads) { return blocks <= 0xffffffffLL / threads; }

namespace {

// What a request has in this call: rows first .. last - 1 of the activations, of which row i is at
// position i + shift (64 bits: lengths and cu are any int32), and the tokens that its table holds.
struct Request {
  int64_t first, last, shift;
  int32_t tokens;
};

__device__ __forceinline__ Request request_of(const Cache& c, int r) {
  Request q;
  const int64_t end = c.cu[r + 1];
  q.first = min(max(static_cast<int64_t>(c.cu[r]), int64_t{0}), c.num_tokens);
  q.last = max(min(end, c.num_tokens), int64_t{0});
  const int64_t length = c.lengths[r];
  q.shift = length - end;
  q.tokens = static_cast<int32_t>(
      max(min(length, static_cast<int64_t>(c.table_width) << c.page_log2), int64_t{0}));
  return q;
}

// Lane k's, to every lane.  (Rows are below 2^31.)
__device__ __forceinline__ Request request_from(const Request& x, int k) {
  Request q;
  q.first = __builtin_amdgcn_readlane(static_cast<int>(x.first), k);
  q.last = __builtin_amdgcn_readlane(static_cast<int>(x.last), k);
  q.shift = static_cast<int64_t>(
      static_cast<uint64_t>(static_cast<uint32_t>(
          __builtin_amdgcn_readlane(static_cast<int>(x.shift >> 32), k))) << 32 |
      static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x.shift), k)));
  q.tokens = __builtin_amdgcn_readlane(x.tokens, k);
  return q;
}

// Where each request has a run of numbers, which begins at begins(its first row, its own number) and
// never before an earlier request's: the request whose run has `number`, what it has in the call and
// how far into its run that is; false where no run has begun.  The last run that begins at or before
// it, by a 64-way search with one wave-wide load a level (one level up to 64 requests, two up to
// 4,096).  Called by every lane of a wave; the results are uniform.
template <typename F>
__device__ __forceinline__ bool find_run(const Cache& c, int number, int& r, Request& q, int& within,
                                         F begins) {
  const int lane = threadIdx.x & 63;
  int low = 0, count = c.requests;
  for (;;) {
    const int step = (count + 63) >> 6;
    const bool in = lane < (count + step - 1) / step;
    const int index = in ? low + lane * step : low;
    Request mine;
    if (step == 1) mine = request_of(c, index);   // the last level: all of each candidate at once
    else mine.first = min(max(static_cast<int64_t>(c.cu[index]), int64_t{0}), c.num_tokens);
    const int at = begins(static_cast<int>(mine.first), index);
    const uint64_t before = __ballot(in && at <= number);
    if (before == 0) return false;
    const int k = 63 - __clzll(static_cast<long long>(before));
    low += k * step;
    if (step == 1) {
      r = low;
      within = number - __builtin_amdgcn_readlane(at, k);
      q = request_from(mine, k);
      return true;
    }
    count = min(step, count - k * step);
  }
}

__device__ __forceinline__ bool live_page(const Cache& c, int page) {
  return page > 0 && page < c.num_pages;
}

// Bytes of a page and head: 128 a token.
__device__ __forceinline__ const uint8_t* k_tile(const Cache& c, int page, int head) {
  return c.k + page * c.k_page + (static_cast<int64_t>(head) << (7 + c.page_log2));
}
__device__ __forceinline__ const uint8_t* v_tile(const Cache& c, int page, int head) {
  return c.v + page * c.v_page + (static_cast<int64_t>(head) << (7 + c.page_log2));
}

// The value of the lane that Ctrl names, in the rows of RowMask; 0 where there is none.
template <int Ctrl, int RowMask>
__device__ __forceinline__ uint32_t shifted(uint32_t x) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(x), Ctrl, RowMask, 0xF, false));
}

// The sum of x over the lanes up to and with this one: within rows of 16 lanes, then from each row's
// last lane to the next row, then to the upper half.
__device__ __forceinline__ uint32_t sum_up_to(uint32_t x) {
  x += shifted<0x111, 0xf>(x);
  x += shifted<0x112, 0xf>(x);
  x += shifted<0x114, 0xf>(x);
  x += shifted<0x118, 0xf>(x);
  x += shifted<0x142, 0xa>(x);
  x += shifted<0x143, 0xc>(x);
  return x;
}

// Codes 4 w .. 4 w + 3 of each word as operands: e4m3 times a power of two is exact in bf16.
__device__ __forceinline__ bf16x8 operand8(uint32_t lo, uint32_t hi, float scale) {
  u32x4 r;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
  r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
  r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
  return __builtin_bit_cast(bf16x8, r);
}

// Of four codes, 0x80 in the byte of each that is NaN.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t codes) {
  return ((codes & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// A word whose first `count` bytes are kept.
__device__ __forceinline__ uint32_t first_bytes(int count) {
  return count >= 4 ? 0xffffffffu : count <= 0 ? 0u : (1u << (8 * count)) - 1;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// A value of this lane and of lane i ^ 16, then i ^ 32: their largest.
__device__ __forceinline__ float max_over_quarters(float x) {
  uint32_t u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  u = __float_as_uint(x);
  const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

constexpr float kLowest = -3.4028234663852886e38f;

// Weights are exp2(score * log2_scale - top * log2_scale) by one fused operation a score, whose second
// product is rounded: off by up to 2^-24 of it in the exponent, 2^-14 where it is up to this.  Past it
// (2^31, say, where that is a factor of 2^128) a wave subtracts the maximum itself ahead, exactly
// where the weight counts.
constexpr float kFar = 1024.0f;
__device__ __forceinline__ bool far_scores(float top, float log2_scale) {   // (no score: top = 0)
  return __any(fabsf(top) * log2_scale > kFar);
}

// Every weight is 2^-24 of that, the sums with them: so that a sum of products passes fp32's range
// with 2^24 of the cache's largest values (2^16 where a maximum may be behind by 2^8), not with two,
// and products with its smallest keep 16 bits.
constexpr float kHeadroom = -24.0f;

// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float power_of_two(int e) {
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}
__device__ __forceinline__ float scale_value(uint8_t b) {
  return power_of_two(min(max(static_cast<int>(b) - kScaleBias, kScaleLow), kScaleHigh));
}

}  // namespace
}  // namespace ld
