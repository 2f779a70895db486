// The paged 8-bit cache: keys and values quantised as they are written, and read back.
//
// Bound by memory: two bytes an element one way and one the other.  A workgroup of two waves takes the
// keys or the values of one head in one page.  The keys of a page lie sixteen elements of a token
// together, so that a thread moves such a piece and eight threads a token's row; the values lie
// sixteen tokens of an element together, so that a thread moves a block of four elements and
// sixteen tokens, transposed in registers, and 32 threads a row of each token.  A page's new rows
// stay in registers between the search for their largest magnitude and their rounding.
//
// 32 x 1024 tokens of 8 heads: 46 us, 4.4 TB/s (66 with two-byte loads of
// values and two passes over the rows); 16,755 tokens read back 30 us, 3.4 TB/s (83 with a token a wave):
// no byte more than those of codes and rows, but every workgroup's one page waits for lengths, table, scale
// and codes in turn.
#include <algorithm>

#include "attention_common.h"

namespace ld {
namespace {

constexpr int kIoThreads = 128;

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Four fp32 as e4m3, the first in the lowest byte: to the nearest, ties to even.  The instruction gives
// NaN past 448, so that callers limit what is finite.
__device__ __forceinline__ uint32_t four_fp8(float a, float b, float c, float d) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true));
}

// bf16 bits as a value to be rounded to e4m3: scaled and, where a page has any that need it
// (Limited), limited to 448 and NaN where not finite.
template <bool Limited>
__device__ __forceinline__ float ready(uint32_t bits, float inverse) {
  const float y = __uint_as_float(bits << 16) * inverse;
  if constexpr (!Limited) return y;
  return (bits & 0x7f80u) == 0x7f80u ? __uint_as_float(0x7fc00000u)
                                     : fminf(fmaxf(y, -448.0f), 448.0f);
}

// The exponent of the scale for a largest magnitude (bits of a finite bf16): the least e with
// m <= 448 * 2^e = 1.75 * 2^(e + 8).
__device__ __forceinline__ int scale_exponent(uint32_t m) {
  const int e = static_cast<int>(m >> 7) - 127 - 8 + ((m & 0x7fu) > 0x60u ? 1 : 0);
  return min(max(e, kScaleLow), kScaleHigh);
}

// Codes of a page whose scale grew, rounded to the new scale.
__device__ __forceinline__ uint32_t rescaled(uint32_t codes, float down) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(codes, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(codes, true);
  return four_fp8(lo[0] * down, lo[1] * down, hi[0] * down, hi[1] * down);
}

// A unit's part of a page: tokens from .. to - 1 of it, of which token t has row `row0` + t.
struct Part {
  int64_t row0;
  int32_t page, from, to;
};

// Requests have a run of units each, as many as pages that their rows can touch: rows / page + 2 (rows
// begin anywhere in a page), or as many as rows where that is less.  False where the unit has no page to do
// with; q and within are set wherever there is a request (within < 0: not).
__device__ __forceinline__ bool find_part(const Cache& c, int unit, Part& part, Request& q,
                                          int& within) {
  int r;
  within = -1;
  if (!find_run(c, unit, r, q, within, [&](int row, int request) {
        return min(row, (row >> c.page_log2) + 2 * request);
      }))
    return false;
  const int64_t begin = max(q.first + q.shift, int64_t{0});
  const int64_t end = min(q.last + q.shift, static_cast<int64_t>(q.tokens));
  const int64_t slot = (begin >> c.page_log2) + within;
  const int64_t token0 = slot << c.page_log2;
  if (begin >= end || token0 >= end) return false;
  part.page = c.pages[r * c.pages_row + slot];
  part.from = static_cast<int>(max(begin - token0, int64_t{0}));
  part.to = static_cast<int>(min(end - token0, int64_t{1} << c.page_log2));
  part.row0 = token0 - q.shift;
  return true;
}

struct RowsParams {
  Cache cache;
  uint16_t* k;
  uint16_t* v;
  int64_t k_row, v_row;
};

// The largest magnitude of packed pairs of bf16, which are ordered as whole numbers.
__device__ __forceinline__ u16x2 larger(u16x2 most, uint32_t pair) {
  return __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, pair & 0x7fff7fffu));
}
__device__ __forceinline__ uint32_t finite(uint32_t pair) {   // zero in the place of what is not
  return ((pair & 0x7f80u) == 0x7f80u ? 0u : pair & 0xffffu) |
         ((pair & 0x7f800000u) == 0x7f800000u ? 0u : pair & 0xffff0000u);
}

template <int Ctrl>
__device__ __forceinline__ uint32_t swapped(uint32_t x) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(x), Ctrl, 0xF, 0xF, false));
}
template <int Ctrl>
__device__ __forceinline__ uint32_t max_with(uint32_t x) {
  return max(x, swapped<Ctrl>(x));
}

// The largest of both waves' (`shared`: not in use).
__device__ __forceinline__ uint32_t over_workgroup(u16x2 x, uint32_t (&shared)[2]) {
  uint32_t most = max(static_cast<uint32_t>(x[0]), static_cast<uint32_t>(x[1]));
  most = max_with<kDppQuadXor1>(most);
  most = max_with<kDppQuadXor2>(most);
  most = max_with<kDppRowHalfMirror>(most);
  most = max_with<kDppRowMirror>(most);
  const auto a = __builtin_amdgcn_permlane16_swap(most, most, false, false);
  most = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(most, most, false, false);
  most = max(b[0], b[1]);
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = most;
  __syncthreads();
  return max(shared[0], shared[1]);
}

// Sixteen new elements of a token.
template <bool Limited>
__device__ __forceinline__ u32x4 quantised(const uint32_t (&x)[8], float inverse) {
  u32x4 y;
#pragma unroll
  for (int w = 0; w < 4; ++w)
    y[w] = four_fp8(ready<Limited>(x[2 * w] & 0xffffu, inverse), ready<Limited>(x[2 * w] >> 16, inverse),
                    ready<Limited>(x[2 * w + 1] & 0xffffu, inverse),
                    ready<Limited>(x[2 * w + 1] >> 16, inverse));
  return y;
}

// Tokens first .. first + 3 of an element, of which from .. to - 1 are new (x: their bf16, element
// `half` of each pair) and earlier ones held (codes, `down` where the scale grew).
template <bool Limited>
__device__ __forceinline__ uint32_t four_tokens(const uint32_t* x, int half, float inverse,
                                                uint32_t codes, bool grew, float down, int first,
                                                int from, int to) {
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = ready<Limited>(x[2 * i] >> (16 * half) & 0xffffu, inverse);
  const uint32_t made = four_fp8(f[0], f[1], f[2], f[3]);
  if (first >= from && first + 4 <= to) return made;
  const uint32_t held = first_bytes(from - first), later = ~first_bytes(to - first);
  return (made & ~held & ~later) | ((grew ? rescaled(codes, down) : codes) & held) | (codes & later);
}

// Between lanes 4 q .. 4 q + 3: lane j's piece i becomes lane i's piece j, so that a store writes whole
// 64-byte pieces of memory (a lane's own four take a request each: 51.8 us for 32 x 1024 tokens, 46.3 so).
__device__ __forceinline__ void transpose_quad(u32x4 (&y)[4]) {
  const bool odd = threadIdx.x & 1, upper = threadIdx.x & 2;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
#pragma unroll
    for (int a = 0; a < 4; a += 2) {
      const uint32_t got = swapped<kDppQuadXor1>(odd ? y[a][w] : y[a + 1][w]);
      y[a][w] = odd ? got : y[a][w];
      y[a + 1][w] = odd ? y[a + 1][w] : got;
    }
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const uint32_t got = swapped<kDppQuadXor2>(upper ? y[a][w] : y[a + 2][w]);
      y[a][w] = upper ? got : y[a][w];
      y[a + 2][w] = upper ? y[a + 2][w] : got;
    }
  }
}

template <int PageLog2>
__global__ __launch_bounds__(kIoThreads) void cache_write_kernel(const RowsParams p) {
  const Cache& c = p.cache;
  constexpr int kPage = 1 << PageLog2;
  constexpr int kKeyPieces = kPage * 8 / kIoThreads;                    // a thread's
  constexpr int kValueBlocks = (kPage * 2 + kIoThreads - 1) / kIoThreads;
  const int kinds = 2 * c.kv_heads;
  const int kind = blockIdx.x % kinds;
  const int head = kind >> 1;
  const bool is_values = kind & 1;
  Part part;
  Request q;
  int within;
  if (!find_part(c, blockIdx.x / kinds, part, q, within) || !live_page(c, part.page)) return;
  const int from = part.from, to = part.to;
  __shared__ uint32_t shared[2][2];
  u16x2 most = {0, 0};

  // new rows into registers: zeros for tokens that are not new; and what values share their pieces with
  uint32_t x[kValueBlocks * 32 > kKeyPieces * 8 ? kValueBlocks * 32 : kKeyPieces * 8] = {};
  u32x4 codes[kValueBlocks][4] = {};
  u32x4* const tile = reinterpret_cast<u32x4*>(const_cast<uint8_t*>(
      is_values ? v_tile(c, part.page, head) : k_tile(c, part.page, head)));
  const int64_t row_stride = is_values ? p.v_row : p.k_row;
  const uint16_t* const rows = (is_values ? p.v : p.k) + part.row0 * row_stride + head * kDim;
  const uint8_t* const scale_at = is_values ? c.v_scale + part.page * c.v_scale_page + head
                                            : c.k_scale + part.page * c.k_scale_page + head;
  const int old = min(max(static_cast<int>(*scale_at) - kScaleBias, kScaleLow), kScaleHigh);
  if (!is_values) {
#pragma unroll
    for (int i = 0; i < kKeyPieces; ++i) {
      const int token = (threadIdx.x >> 3) + i * (kIoThreads / 8);
      uint32_t (&mine)[8] = reinterpret_cast<uint32_t(&)[8]>(x[8 * i]);
      if (i * 16 >= to || i * 16 + 16 <= from) continue;   // (all threads)
      if (token >= from && token < to)
        __builtin_memcpy(mine, rows + token * row_stride + (threadIdx.x & 7) * 16, 32);
#pragma unroll
      for (int w = 0; w < 8; ++w) most = larger(most, mine[w]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kValueBlocks; ++i) {
      const int block = threadIdx.x + i * kIoThreads;
      const int first = (block >> 5) * 16;
#pragma unroll
      for (int t = 0; t < 16; ++t) {
        u32x2 pair = {0, 0};
        if (first + t >= from && first + t < to)
          __builtin_memcpy(&pair, rows + (first + t) * row_stride + (block & 31) * 4, 8);
        x[32 * i + 2 * t] = pair[0];
        x[32 * i + 2 * t + 1] = pair[1];
        most = larger(larger(most, pair[0]), pair[1]);
      }
      if (first < to && first + 16 > from && (first < from || first + 16 > to))
#pragma unroll
        for (int d = 0; d < 4; ++d) codes[i][d] = tile[(block >> 5) * kDim + (block & 31) * 4 + d];
    }
  }
  uint32_t largest = over_workgroup(most, shared[0]);
  const bool strange = largest >= 0x7f80u;   // what is not finite does not count
  if (strange) {
    most = u16x2{0, 0};
    constexpr int kWords = sizeof(x) / 4;
#pragma unroll
    for (int w = 0; w < kWords; ++w)
      if (is_values ? w < kValueBlocks * 32 : w < kKeyPieces * 8) most = larger(most, finite(x[w]));
    largest = over_workgroup(most, shared[1]);
  }
  int e = scale_exponent(largest);
  if (from > 0) e = max(e, old);
  const float inverse = power_of_two(-e);
  const bool grew = from > 0 && e > old;
  const float down = power_of_two(max(old - e, -126));
  const bool limited = strange || e == kScaleHigh;
  if (threadIdx.x == 0) *const_cast<uint8_t*>(scale_at) = static_cast<uint8_t>(e + kScaleBias);

  if (!is_values) {
#pragma unroll
    for (int i = 0; i < kKeyPieces; ++i) {
      const int token = (threadIdx.x >> 3) + i * (kIoThreads / 8);
      if (i * 16 >= to || (i * 16 + 16 <= from && !grew)) continue;   // (all threads)
      u32x4* const at = tile + ((threadIdx.x & 7) << PageLog2) + token;
      const uint32_t (&mine)[8] = reinterpret_cast<const uint32_t(&)[8]>(x[8 * i]);
      if (token >= from && token < to) {
        *at = limited ? quantised<true>(mine, inverse) : quantised<false>(mine, inverse);
      } else if (token < from && grew) {
        u32x4 held = *at;
#pragma unroll
        for (int w = 0; w < 4; ++w) held[w] = rescaled(held[w], down);
        *at = held;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kValueBlocks; ++i) {
      const int block = threadIdx.x + i * kIoThreads;
      const int first = (block >> 5) * 16;
      if (first >= to || first >= kPage || (first + 16 <= from && !grew)) continue;
      u32x4* const at = tile + (block >> 5) * kDim + (block & 31) * 4;
      if (first + 16 <= from)   // (held alone)
#pragma unroll
        for (int d = 0; d < 4; ++d) codes[i][d] = at[d];
      u32x4 y[4];
#pragma unroll
      for (int d = 0; d < 4; ++d) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t* const four = &x[32 * i + 8 * w + (d >> 1)];
          y[d][w] = limited ? four_tokens<true>(four, d & 1, inverse, codes[i][d][w], grew, down,
                                             first + 4 * w, from, to)
                         : four_tokens<false>(four, d & 1, inverse, codes[i][d][w], grew, down,
                                              first + 4 * w, from, to);
        }
      }
      transpose_quad(y);
      u32x4* const to_quad = tile + (block >> 5) * kDim + (block & 28) * 4 + (threadIdx.x & 3);
#pragma unroll
      for (int d = 0; d < 4; ++d) to_quad[4 * d] = y[d];
    }
  }
}

// Bytes d of four words as one: of four elements' tokens, a token's four elements.
__device__ __forceinline__ uint32_t byte_of_each(const uint32_t (&x)[4], int d) {
  const uint32_t at = static_cast<uint32_t>(d) | static_cast<uint32_t>(d + 4) << 8;
  const uint32_t lo = __builtin_amdgcn_perm(x[1], x[0], at);
  const uint32_t hi = __builtin_amdgcn_perm(x[3], x[2], at);
  return (lo & 0xffffu) | hi << 16;
}

__global__ __launch_bounds__(kIoThreads) void cache_read_kernel(const RowsParams p) {
  const Cache& c = p.cache;
  const int kinds = 2 * c.kv_heads;
  const int kind = blockIdx.x % kinds;
  const int head = kind >> 1;
  const bool is_values = kind & 1;
  const int64_t row_stride = is_values ? p.v_row : p.k_row;
  uint16_t* const rows = (is_values ? p.v : p.k) + head * kDim;
  auto zeros = [&](int64_t first, int64_t last) {
    const u32x4 none = {0, 0, 0, 0};
    for (int64_t row = first + (threadIdx.x >> 4); row < last; row += kIoThreads / 16)
      __builtin_memcpy(rows + row * row_stride + (threadIdx.x & 15) * 8, &none, 16);
  };
  Part part;
  Request q;
  int within;
  const bool some = find_part(c, blockIdx.x / kinds, part, q, within);
  if (within == 0) {   // rows before the first token and behind the table, by the first unit
    const int64_t begin = max(q.first, min(q.last, -q.shift));
    zeros(q.first, begin);
    zeros(max(begin, min(q.last, q.tokens - q.shift)), q.last);
  }
  if (!some) return;
  if (!live_page(c, part.page)) {
    zeros(part.row0 + part.from, part.row0 + part.to);
    return;
  }
  uint16_t* const to_rows = rows + part.row0 * row_stride;
  if (!is_values) {
    const u32x4* const tile = reinterpret_cast<const u32x4*>(k_tile(c, part.page, head));
    const float scale = scale_value(c.k_scale[part.page * c.k_scale_page + head]);
    for (int token = part.from + (threadIdx.x >> 3); token < part.to; token += kIoThreads / 8) {
      const u32x4 x = tile[((threadIdx.x & 7) << c.page_log2) + token];
      const u32x4 lo = __builtin_bit_cast(u32x4, operand8(x[0], x[1], scale));
      const u32x4 hi = __builtin_bit_cast(u32x4, operand8(x[2], x[3], scale));
      // four lanes have 128 bytes, and store the first 64 of them, then the others
      const bool odd = threadIdx.x & 1;
      u32x4 first, second;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        // (moves between lanes ahead of the choice: every lane takes part in them)
        const uint32_t lo01 = swapped<0x50>(lo[w]), hi01 = swapped<0x50>(hi[w]);   // lanes 0 0 1 1
        const uint32_t lo23 = swapped<0xfa>(lo[w]), hi23 = swapped<0xfa>(hi[w]);   // lanes 2 2 3 3
        first[w] = odd ? hi01 : lo01;
        second[w] = odd ? hi23 : lo23;
      }
      uint16_t* const at = to_rows + token * row_stride + (threadIdx.x & 4) * 16 + (threadIdx.x & 3) * 8;
      __builtin_memcpy(at, &first, 16);
      __builtin_memcpy(at + 32, &second, 16);
    }
  } else {
    const u32x4* const tile = reinterpret_cast<const u32x4*>(v_tile(c, part.page, head));
    const float scale = scale_value(c.v_scale[part.page * c.v_scale_page + head]);
    for (int block = threadIdx.x + (part.from >> 4) * 32; block < ((part.to + 15) >> 4) * 32;
         block += kIoThreads) {
      const int first = (block >> 5) * 16;
      u32x4 x[4];
#pragma unroll
      for (int d = 0; d < 4; ++d) x[d] = tile[(block >> 5) * kDim + (block & 31) * 4 + d];
      uint16_t* const at = to_rows + first * row_stride + (block & 31) * 4;
#pragma unroll
      for (int t = 0; t < 16; ++t) {
        const uint32_t words[4] = {x[0][t >> 2], x[1][t >> 2], x[2][t >> 2], x[3][t >> 2]};
        const uint32_t codes = byte_of_each(words, t & 3);
        u32x2 y;
        y[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false));
        y[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true));
        if (first + t >= part.from && first + t < part.to)
          __builtin_memcpy(at + t * row_stride, &y, 8);
      }
    }
  }
}

int rows_params(const ld_paged_cache* cache, const ld_cache_rows* rows, RowsParams& p,
                int64_t& blocks) {
  if (const int rc = cache_params(cache, p.cache)) return rc;
  if (rows == nullptr) return fail(LD_ERR_INVALID_ARGUMENT, "rows is NULL");
  if (p.cache.requests > 0 && (!rows->k || !rows->v))
    return fail(LD_ERR_INVALID_ARGUMENT, "cache rows: NULL tensor pointer");
  p.k = static_cast<uint16_t*>(rows->k);
  p.v = static_cast<uint16_t*>(rows->v);
  p.k_row = rows->k_row_stride;
  p.v_row = rows->v_row_stride;
  const int64_t counted = (p.cache.num_tokens >> p.cache.page_log2) +
                          2 * static_cast<int64_t>(p.cache.requests);
  if (counted > 0x7fffffff) return fail(LD_ERR_INVALID_ARGUMENT, "too many requests");
  const int64_t units = std::min(counted, p.cache.num_tokens);
  blocks = units * 2 * p.cache.kv_heads;
  if (!launches(blocks, kIoThreads)) return fail(LD_ERR_INVALID_ARGUMENT, "too many pages and heads");
  return LD_OK;
}

}  // namespace
}  // namespace ld

extern "C" int ld_cache_write(const ld_paged_cache* cache, const ld_cache_rows* rows,
                              void* stream) {
  using namespace ld;
  RowsParams p{};
  int64_t blocks;
  if (const int rc = rows_params(cache, rows, p, blocks)) return rc;
  if (p.cache.requests == 0 || p.cache.table_width == 0) return LD_OK;
  const auto kernel = p.cache.page_log2 == 4   ? cache_write_kernel<4>
                      : p.cache.page_log2 == 5 ? cache_write_kernel<5>
                      : p.cache.page_log2 == 6 ? cache_write_kernel<6>
                                               : cache_write_kernel<7>;
  hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(blocks)), dim3(kIoThreads), 0,
                     static_cast<hipStream_t>(stream), p);
  return check_launch("ld_cache_write");
}

extern "C" int ld_cache_read(const ld_paged_cache* cache, const ld_cache_rows* rows,
                             void* stream) {
  using namespace ld;
  RowsParams p{};
  int64_t blocks;
  if (const int rc = rows_params(cache, rows, p, blocks)) return rc;
  if (p.cache.requests == 0) return LD_OK;
  if (p.cache.num_tokens > 1 && (p.k_row < p.cache.kv_heads * kDim || p.v_row < p.cache.kv_heads * kDim))
    return fail(LD_ERR_INVALID_ARGUMENT, "rows of k and v must not overlap");
  hipLaunchKernelGGL(cache_read_kernel, dim3(static_cast<uint32_t>(blocks)), dim3(kIoThreads), 0,
                     static_cast<hipStream_t>(stream), p);
  return check_launch("ld_cache_read");
}
