// The paged 8-bit cache: keys and values quantised as they are written, and read back.
#include "attention_common.h"

namespace ld {
namespace {

// Two fp32 as e4m3 in the low 16 bits: to the nearest, ties to even.  The instruction gives NaN
// past 448, so that callers limit what is finite.
__device__ __forceinline__ uint32_t two_fp8(float a, float b) {
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false)) & 0xffffu;
}

// bf16 bits as a value to be rounded to e4m3: scaled, limited, NaN where not finite.
__device__ __forceinline__ float ready(uint32_t bits, float inverse) {
  const float x = __uint_as_float(bits << 16);
  const float y = fminf(fmaxf(x * inverse, -448.0f), 448.0f);
  return (bits & 0x7f80u) == 0x7f80u ? __uint_as_float(0x7fc00000u) : y;
}

// The exponent of the scale for a largest magnitude (bits of a finite bf16): the least e with
// m <= 448 * 2^e = 1.75 * 2^(e + 8).
__device__ __forceinline__ int scale_exponent(uint32_t m) {
  const int e = static_cast<int>(m >> 7) - 127 - 8 + ((m & 0x7fu) > 0x60u ? 1 : 0);
  return min(max(e, kScaleLow), kScaleHigh);
}

// A code of a page whose scale grew by 2^up, rounded to the new scale (up >= 0).
__device__ __forceinline__ uint32_t rescaled(uint32_t codes, float down) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(codes, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(codes, true);
  return two_fp8(lo[0] * down, lo[1] * down) | two_fp8(hi[0] * down, hi[1] * down) << 16;
}

struct WriteParams {
  Cache cache;
  const uint16_t* k;
  const uint16_t* v;
  int64_t k_row, v_row;
};

// A workgroup takes the keys or the values of one head in one page.  Requests have a run of units
// each, as many as pages that their rows can touch: rows / page + 2 (pages begin anywhere).
__global__ __launch_bounds__(kThreads) void cache_write_kernel(const WriteParams p) {
  const Cache& c = p.cache;
  const int page_size = 1 << c.page_log2;
  const int kinds = 2 * c.kv_heads;
  const int64_t unit = blockIdx.x / kinds;
  const int kind = blockIdx.x % kinds;
  const int head = kind >> 1;
  const bool values = kind & 1;
  int low = 0, high = c.requests - 1;
  while (low < high) {
    const int mid = low + (high - low + 1) / 2;
    if ((max(static_cast<int64_t>(c.cu[mid]), int64_t{0}) >> c.page_log2) + 2ll * mid <= unit) low = mid;
    else high = mid - 1;
  }
  const Request q = request_of(c, low);
  const int64_t within = unit - ((q.first >> c.page_log2) + 2ll * low);
  const int64_t begin = max(q.first + q.shift, int64_t{0});
  const int64_t end = min(q.last + q.shift, static_cast<int64_t>(q.tokens));
  const int64_t slot = (begin >> c.page_log2) + within;
  if (begin >= end || within < 0 || slot << c.page_log2 >= end) return;
  const int page = c.pages[low * c.pages_row + slot];
  if (!live_page(c, page)) return;
  const int from = static_cast<int>(max(begin - (slot << c.page_log2), int64_t{0}));
  const int to = static_cast<int>(min(end - (slot << c.page_log2), static_cast<int64_t>(page_size)));
  const int64_t row_stride = values ? p.v_row : p.k_row;
  // the row of the page's first token (before the tensor's first where it is held already)
  const uint16_t* const rows = (values ? p.v : p.k) +
                               ((slot << c.page_log2) - q.shift) * row_stride + head * kDim;
  uint8_t* const tile = const_cast<uint8_t*>(values ? v_tile(c, page, head) : k_tile(c, page, head));
  uint8_t* const scale = values ? c.v_scale + page * c.v_scale_page + head
                                : c.k_scale + page * c.k_scale_page + head;

  // the largest finite magnitude of the rows: bf16 magnitudes are ordered as whole numbers
  uint32_t most = 0;
  for (int i = threadIdx.x; i < (to - from) * 16; i += kThreads) {
    uint16_t x[8];
    __builtin_memcpy(x, rows + (from + (i >> 4)) * row_stride + (i & 15) * 8, 16);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t m = x[e] & 0x7fffu;
      most = max(most, m < 0x7f80u ? m : 0u);
    }
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), d)));
  __shared__ uint32_t shared[kWaves];
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = most;
  const int old = min(max(static_cast<int>(*scale) - kScaleBias, kScaleLow), kScaleHigh);
  __syncthreads();
  most = max(max(shared[0], shared[1]), max(shared[2], shared[3]));
  int e = scale_exponent(most);
  if (from > 0) e = max(e, old);
  const float inverse = power_of_two(-e);
  const bool grew = from > 0 && e > old;
  const float down = power_of_two(max(old - e, -126));
  if (threadIdx.x == 0) *scale = static_cast<uint8_t>(e + kScaleBias);

  if (!values) {
    if (grew) {
      for (int i = threadIdx.x; i < from * 8; i += kThreads) {
        u32x4* const at = reinterpret_cast<u32x4*>(tile) + ((i & 7) << c.page_log2) + (i >> 3);
        u32x4 x = *at;
#pragma unroll
        for (int w = 0; w < 4; ++w) x[w] = rescaled(x[w], down);
        *at = x;
      }
    }
    for (int i = threadIdx.x; i < (to - from) * 8; i += kThreads) {
      const int token = from + (i >> 3);
      uint16_t x[16];
      __builtin_memcpy(x, rows + token * row_stride + (i & 7) * 16, 32);
      u32x4 y;
#pragma unroll
      for (int w = 0; w < 4; ++w)
        y[w] = two_fp8(ready(x[4 * w], inverse), ready(x[4 * w + 1], inverse)) |
               two_fp8(ready(x[4 * w + 2], inverse), ready(x[4 * w + 3], inverse)) << 16;
      reinterpret_cast<u32x4*>(tile)[((i & 7) << c.page_log2) + token] = y;
    }
  } else {
    // 16 tokens of an element a thread: held ones kept or rounded anew, new ones put in, later
    // ones left
    for (int i = threadIdx.x + (grew ? 0 : (from >> 4) * kDim); i < ((to + 15) >> 4) * kDim;
         i += kThreads) {
      const int first = (i >> 7) * 16;
      u32x4* const at = reinterpret_cast<u32x4*>(tile) + i;
      u32x4 x = {0, 0, 0, 0};
      if (first < from || first + 16 > to) x = *at;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t moved = grew ? rescaled(x[w], down) : x[w];
        float f[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int token = first + 4 * w + b;
          const bool fresh = token >= from && token < to;
          f[b] = ready(fresh ? rows[token * row_stride + (i & 127)] : 0, inverse);
        }
        const uint32_t made = two_fp8(f[0], f[1]) | two_fp8(f[2], f[3]) << 16;
        uint32_t y = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int token = first + 4 * w + b;
          const uint32_t mask = 0xffu << (8 * b);
          y |= (token >= to ? x[w] : token >= from ? made : moved) & mask;
        }
        x[w] = y;
      }
      *at = x;
    }
  }
}

struct ReadParams {
  Cache cache;
  uint16_t* k;
  uint16_t* v;
  int64_t k_row, v_row;
};

// A wave takes the key and value of one row and head, two elements a lane.
__global__ __launch_bounds__(kThreads) void cache_read_kernel(const ReadParams p) {
  const Cache& c = p.cache;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWaves + (threadIdx.x >> 6);
  const int64_t row = unit / c.kv_heads;
  const int head = static_cast<int>(unit - row * c.kv_heads);
  if (row >= c.num_tokens) return;
  const Request q = request_of(c, request_at(c, row));
  if (row < q.first || row >= q.last) return;
  const int r = request_at(c, row);
  const int64_t position = row + q.shift;
  const int lane = threadIdx.x & 63;
  const int d = 2 * lane;
  uint32_t kb = 0, vb = 0;
  if (position >= 0 && position < q.tokens) {
    const int page = c.pages[r * c.pages_row + (position >> c.page_log2)];
    if (live_page(c, page)) {
      const int at = static_cast<int>(position) & ((1 << c.page_log2) - 1);
      const uint8_t* const kt = k_tile(c, page, head);
      const uint8_t* const vt = v_tile(c, page, head);
      const int ki = (((d >> 4) << c.page_log2) + at) * 16 + (d & 15);
      const int vi = ((at >> 4) * kDim + d) * 16 + (at & 15);
      const auto kf = __builtin_amdgcn_cvt_pk_f32_fp8(kt[ki] | kt[ki + 1] << 8, false);
      const auto vf = __builtin_amdgcn_cvt_pk_f32_fp8(vt[vi] | vt[vi + 16] << 8, false);
      const float ks = scale_value(c.k_scale[page * c.k_scale_page + head]);
      const float vs = scale_value(c.v_scale[page * c.v_scale_page + head]);
      kb = f32_to_bf16(kf[0] * ks) | static_cast<uint32_t>(f32_to_bf16(kf[1] * ks)) << 16;
      vb = f32_to_bf16(vf[0] * vs) | static_cast<uint32_t>(f32_to_bf16(vf[1] * vs)) << 16;
    }
  }
  __builtin_memcpy(p.k + row * p.k_row + head * kDim + d, &kb, 4);
  __builtin_memcpy(p.v + row * p.v_row + head * kDim + d, &vb, 4);
}

int check_rows(const ld_cache_rows* rows, const Cache& c) {
  if (rows == nullptr) return fail(LD_ERR_INVALID_ARGUMENT, "rows is NULL");
  if (c.requests > 0 && (!rows->k || !rows->v))
    return fail(LD_ERR_INVALID_ARGUMENT, "cache rows: NULL tensor pointer");
  return LD_OK;
}

}  // namespace
}  // namespace ld

extern "C" int ld_cache_write(const ld_paged_cache* cache, const ld_cache_rows* rows,
                              void* stream) {
  using namespace ld;
  WriteParams p{};
  if (const int rc = cache_params(cache, p.cache)) return rc;
  if (const int rc = check_rows(rows, p.cache)) return rc;
  if (p.cache.requests == 0 || p.cache.table_width == 0) return LD_OK;
  p.k = static_cast<const uint16_t*>(rows->k);
  p.v = static_cast<const uint16_t*>(rows->v);
  p.k_row = rows->k_row_stride;
  p.v_row = rows->v_row_stride;
  const int64_t units = (p.cache.num_tokens >> p.cache.page_log2) + 2ll * p.cache.requests;
  const int64_t blocks = units * 2 * p.cache.kv_heads;
  if (blocks > 0x7fffffff) return fail(LD_ERR_INVALID_ARGUMENT, "too many pages and heads");
  hipLaunchKernelGGL(cache_write_kernel, dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), p);
  return check_launch("ld_cache_write");
}

extern "C" int ld_cache_read(const ld_paged_cache* cache, const ld_cache_rows* rows,
                             void* stream) {
  using namespace ld;
  ReadParams p{};
  if (const int rc = cache_params(cache, p.cache)) return rc;
  if (const int rc = check_rows(rows, p.cache)) return rc;
  if (p.cache.requests == 0) return LD_OK;
  if (p.cache.num_tokens > 1 && (rows->k_row_stride < p.cache.kv_heads * kDim ||
                                 rows->v_row_stride < p.cache.kv_heads * kDim))
    return fail(LD_ERR_INVALID_ARGUMENT, "rows of k and v must not overlap");
  p.k = static_cast<uint16_t*>(rows->k);
  p.v = static_cast<uint16_t*>(rows->v);
  p.k_row = rows->k_row_stride;
  p.v_row = rows->v_row_stride;
  const int64_t blocks = (p.cache.num_tokens * p.cache.kv_heads + kWaves - 1) / kWaves;
  if (blocks > 0x7fffffff) return fail(LD_ERR_INVALID_ARGUMENT, "too many tokens and heads");
  hipLaunchKernelGGL(cache_read_kernel, dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), p);
  return check_launch("ld_cache_read");
}
