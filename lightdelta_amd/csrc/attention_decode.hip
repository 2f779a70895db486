// Attention of up to four rows a request to its tokens in the paged 8-bit cache.
//
// Bound by memory: 256 bytes a token and kv head against 4 * 128 operations a query.  All tiles of
// 64 tokens, request after request and head after head, are cut into equal runs, one a workgroup,
// whatever the lengths are (they are known on the device alone); runs that begin or end inside a
// head's tiles leave sums in the workspace, which a second launch joins.
//
// Each of four waves takes every fourth tile of its workgroup's run, straight from memory into the
// operands of v_mfma_f32_16x16x32_bf16: the cache's order of bytes is theirs.  With m = lane % 16 and h = lane / 16,
//   scores [token, column]: operand A holds the keys of token 16 (m / 4) + 4 t + m % 4 of the tile
//     in product t (0 .. 3), so that a lane finds the scores of tokens 16 h .. 16 h + 15 of column m;
//   outputs [element, column]: operand B is these sixteen weights, A sixteen bytes of a page's v,
//     the same tokens of element 16 b + m.
// Columns are the request's rows times the q heads of a kv head.  Where they are more than 16, two or
// four waves take the same tile for 16 columns each (the second read of a tile is the L2's): a wave of
// 32 columns does not fit in the registers of two a SIMD, and what it keeps in scratch memory waits
// for the tiles in flight (31.7 us for a verify of 64 requests of up to 4,000 tokens, 23.4 without).
// e4m3 times its scale is exact in bf16; weights are two bf16 each (2^-17 of one is lost), in a product
// each with the same operand of values: the 33 requests below 51.4 us (50.5 with one bf16), the verify 24.5
// (23.3).
//
// 33 requests of up to 8,000 tokens, 8 kv heads: 47 us and 5 for the join, 221 MB at 4.7 TB/s; of it about
// 5 until a workgroup's first tile is there (lengths, table and codes wait for one another).  One request
// of 177 tokens: 6.0 and 3.4 us.  64 requests of up to four rows and 4,000 tokens: 21 and 5.  512 requests
// of one row and 250 to 2,000 tokens, 2 kv heads: 54 in all, 221 MB at 4.1 TB/s.
#include <algorithm>

#include "attention_common.h"

namespace ld {
namespace {

constexpr int kTile = 64;        // tokens

struct DecodeAttention {
  Cache cache;
  Attention a;
  int32_t workers;
  int32_t columns;   // width * group
};

// The workspace: the sums of runs, two a workgroup (a run's first piece and, where it is another
// one, its last), of all columns each: outputs, then the maximum and sum of each column.  Ahead
// of them the run's length and of each request the tiles ahead of it, for the second launch.
struct Layout {
  int64_t plan;      // floats
  int64_t columns;   // of a piece
  __device__ __host__ int64_t piece(int64_t worker, int which) const {
    return plan + (worker * 2 + which) * columns * (kDim + 2);
  }
};
__device__ __host__ inline Layout layout_of(int64_t requests, int64_t columns) {
  return Layout{(requests + 2 + 3) & ~int64_t{3}, columns};
}

// Requests and their tiles, 64 requests at a time, one a lane; every lane of a wave calls it.
struct Walk {
  int base = 0;            // the first of the 64
  uint32_t before = 0;     // tiles of the requests before it
  Request mine;            // this lane's request
  uint32_t tiles = 0;      // its tiles
  uint32_t behind = 0;     // tiles of the 64 up to and with it
  uint32_t all = 0;        // of the 64

  __device__ __forceinline__ void load(const DecodeAttention& p, int first) {
    const int lane = threadIdx.x & 63;
    base = first;
    const bool real = first + lane < p.cache.requests;
    mine = request_of(p.cache, real ? first + lane : 0);
    const int64_t rows = mine.last - mine.first;
    tiles = real && rows > 0 && rows <= p.a.width
                ? (static_cast<uint32_t>(mine.tokens) + kTile - 1) / kTile : 0;
    behind = sum_up_to(tiles);
    all = __builtin_amdgcn_readlane(behind, 63);
  }
  // Tiles of all requests; ends at the first 64 again.  `plan`: where those ahead of each request
  // are written (NULL: nowhere).
  __device__ __forceinline__ uint32_t total(const DecodeAttention& p, uint32_t* plan) {
    uint32_t sum = 0;
    for (int first = 0;; first += 64) {
      load(p, first);
      const int r = first + (threadIdx.x & 63);
      if (plan != nullptr && r < p.cache.requests) plan[1 + r] = sum + behind - tiles;
      sum += all;
      if (first + 64 >= p.cache.requests) break;
    }
    if (p.cache.requests > 64) load(p, 0);
    return sum;
  }
  // The request that has tile `at` of all (which there is, and which is not before the 64): its
  // tiles, those of the requests before it, its number and what it has in the call.
  __device__ __forceinline__ uint32_t find(const DecodeAttention& p, uint32_t at, uint32_t& first,
                                           int& number, Request& q) {
    while (at >= before + all) {
      before += all;
      load(p, base + 64);
    }
    const uint32_t local = at - before;
    const int k = __popcll(__ballot(behind <= local));
    const uint32_t n = __builtin_amdgcn_readlane(tiles, k);
    first = before + __builtin_amdgcn_readlane(behind, k) - n;
    number = base + k;
    q = request_from(mine, k);
    return n;
  }
};

// Tiles of a workgroup's run.  (With a whole number for each of its waves, of which there would be
// fewer runs, 32 requests of 13 to 96 tokens take 17.1 us in a graph and not 8.9, their heads being taken
// one after another, and 64 of 250 to 2,000 tokens and 8 kv heads 30.3 and not 27.9.)
__device__ __forceinline__ uint32_t run_length(const DecodeAttention& p, uint32_t total) {
  const uint32_t workers = static_cast<uint32_t>(p.workers);
  return max((total * p.cache.kv_heads + workers - 1) / workers, 1u);
}

__device__ __forceinline__ u32x4 eight_bf16(const float (&x)[8]) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = bf16_pair(f32x2{x[2 * i], x[2 * i + 1]});
  return r;
}

// Eight elements of an output: divided, gated and rounded.
__device__ __forceinline__ void store_out(const Attention& a, int64_t row, int head, int d,
                                          float (&o)[8], float top, float total) {
  const bool some = top > -__builtin_inff();   // the row sees a token
  const float inverse = 1.0f / total;
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = some ? o[i] * inverse : 0.0f;
  if (a.gate != nullptr && some) {
    uint16_t g[8];
    __builtin_memcpy(g, a.gate + row * a.gate_row + head * kDim + d, 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] *= sigmoid(bf16_to_f32(g[i]));
  }
  const u32x4 bits = eight_bf16(o);
  __builtin_memcpy(a.out + (row * a.q_heads + head) * kDim + d, &bits, 16);
}

// Split: waves a tile, 16 columns each.
template <int Split>
__global__ __launch_bounds__(kThreads, 2) void attention_decode_kernel(const DecodeAttention p) {
  const Cache& c = p.cache;
  const Attention& a = p.a;
  constexpr int kPad = kDim + 4;
  __shared__ __attribute__((aligned(16))) float sums[kWaves][16][kPad];
  __shared__ float stats[kWaves][2][16];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 15, h = lane >> 4;
  const int column0 = blockIdx.y * 16 * Split;
  constexpr int step = kWaves / Split;   // tiles that the workgroup's waves take at a time
  const int column = column0 + 16 * (wave & (Split - 1)) + m;

  const Layout layout = layout_of(c.requests, static_cast<int64_t>(gridDim.y) * 16 * Split);
  const bool planner = blockIdx.x == 0 && blockIdx.y == 0 && wave == 0;
  uint32_t* const plan = planner ? reinterpret_cast<uint32_t*>(a.workspace) : nullptr;
  Walk walk;
  const uint32_t total = walk.total(p, plan);
  const uint32_t run = run_length(p, total);
  if (planner && lane == 0) {
    plan[0] = run;
    plan[1 + c.requests] = total;
  }
  // (the host has seen to it that all tiles and two runs are below 2^32)
  const uint32_t start = blockIdx.x * run;
  const uint32_t end = min(start + run, total * c.kv_heads);
  for (uint32_t at = start; at < end;) {
    uint32_t first;
    int r;
    Request q;
    const uint32_t tiles = walk.find(p, at / c.kv_heads, first, r, q);
    const uint32_t local = at - first * c.kv_heads;
    const int head = static_cast<int>(local / tiles);
    const uint32_t from = local - head * tiles;
    const uint32_t to = min(tiles, from + (end - at));
    const int rows = static_cast<int>(q.last - q.first);
    const int32_t* const table = c.pages + r * c.pages_row;

    // The tiles' pages first: the keys wait for them.  A tile's pages: that of tokens 16 (m / 4) .. for
    // the keys, 16 h .. for the values (0, whose bytes are read and not used, where there is none).
    auto page_of = [&](uint32_t tile, int group) {
      const int token = static_cast<int>(tile) * kTile + 16 * group;
      const int page = tile < to && token < q.tokens ? table[token >> c.page_log2] : 0;
      return live_page(c, page) ? page : 0;
    };
    uint32_t tile = from + wave / Split;
    int k_page = page_of(tile, m >> 2), v_page = page_of(tile, h);
    int k_next = page_of(tile + step, m >> 2), v_next = page_of(tile + step, h);

    // the column's query, and how many tokens it sees (one that there is not: all)
    const int t_row = column / a.group;
    const bool real = column < p.columns && t_row < rows;
    const int limit = real ? static_cast<int>(max(min(q.first + t_row + q.shift + 1,
                                                      static_cast<int64_t>(q.tokens)), int64_t{0}))
                           : q.tokens;
    const uint16_t* const from_q = a.q + (q.first + (real ? t_row : 0)) * a.q_row +
                                   (head * a.group + (real ? column - t_row * a.group : 0)) * kDim;
    bf16x8 query[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      u32x4 x;
      __builtin_memcpy(&x, from_q + 16 * (4 * (s >> 1) + h) + 8 * (s & 1), 16);
      query[s] = __builtin_bit_cast(bf16x8, real ? x : u32x4{0, 0, 0, 0});
    }
    const int least = static_cast<int>(max(min(q.first + q.shift + 1, static_cast<int64_t>(q.tokens)),
                                           int64_t{0}));   // what the first row sees

    f32x4 o[8];
    float top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
    for (int b = 0; b < 8; ++b) o[b] = f32x4{0, 0, 0, 0};

    u32x4 keys[4][2], values[8];
    float k_scale, v_scale;
    auto load_keys = [&](uint32_t tile, int page) {
      const int in = (static_cast<int>(tile) * kTile + 16 * (m >> 2)) & ((1 << c.page_log2) - 1);
      const uint8_t* const at_k = k_tile(c, page, head) + (((h << c.page_log2) + in + (m & 3)) << 4);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int s = 0; s < 2; ++s)
          keys[t][s] = *reinterpret_cast<const u32x4*>(at_k + 64 * t + (s << (6 + c.page_log2)));
      k_scale = scale_value(c.k_scale[page * c.k_scale_page + head]);
    };
    auto load_values = [&](uint32_t tile, int page) {
      const int in = (static_cast<int>(tile) * kTile + 16 * h) & ((1 << c.page_log2) - 1);
      const uint8_t* const at_v = v_tile(c, page, head) + (in >> 4) * (kDim * 16) + m * 16;
#pragma unroll
      for (int b = 0; b < 8; ++b) values[b] = *reinterpret_cast<const u32x4*>(at_v + b * 256);
      v_scale = scale_value(c.v_scale[page * c.v_scale_page + head]);
    };

    if (tile < to) {
      load_keys(tile, k_page);
      load_values(tile, v_page);
    }
    uint32_t strange = 0;
    for (; tile < to; tile += step) {
      const int token0 = static_cast<int>(tile) * kTile;
      const bool live = v_page > 0;
      f32x4 score[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        score[t] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const u32x4 x = keys[t][s >> 1];
          score[t] = mfma16(operand8(x[2 * (s & 1)], x[2 * (s & 1) + 1], k_scale), query[s], score[t]);
        }
      }
      const bool more = tile + step < to;
      if (more) load_keys(tile + step, k_next);
      k_page = k_next;
      const int v_now = v_next;
      k_next = page_of(tile + 2 * step, m >> 2);
      v_next = page_of(tile + 2 * step, h);

      // a tile that some column does not see whole: scores of -inf, weights of zero
      const bool whole = token0 + kTile <= least && __all(live);
      float most = kLowest;   // (of a score of -inf that is seen: a weight of zero, not none)
      if (!whole) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!live || token0 + 16 * h + 4 * t + i >= limit) score[t][i] = -__builtin_inff();
        if (!live || token0 + 16 * h >= limit) most = -__builtin_inff();
      }
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) most = fmaxf(most, score[t][i]);
      most = max_over_quarters(most);
      const float now = fmaxf(top, most);
      if (__any(now > top)) {
        const float keep = now == top ? 1.0f : exp2_fast((top - now) * a.log2_scale);
        sum *= keep;
#pragma unroll
        for (int b = 0; b < 8; ++b) o[b] *= keep;
        top = now;
      }
      const float some = now == -__builtin_inff() ? 0.0f : now;
      float less = fmaf(-some, a.log2_scale, kHeadroom);
      if (far_scores(some, a.log2_scale)) {
#pragma unroll
        for (int t = 0; t < 4; ++t) score[t] -= some;
        less = kHeadroom;
      }
      u32x4 bits[2], rest[2];   // weights as two bf16 each
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] = exp2_fast(fmaf(score[t][i], a.log2_scale, less));
          sum += w[i];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t pair = bf16_pair(f32x2{w[2 * i], w[2 * i + 1]});
          bits[t >> 1][2 * (t & 1) + i] = pair;
          rest[t >> 1][2 * (t & 1) + i] =
              bf16_pair(f32x2{w[2 * i] - __uint_as_float(pair << 16),
                              w[2 * i + 1] - __uint_as_float(pair & 0xffff0000u)});
        }
      }

      if (!whole) {
        // values behind the last token, or without a page, are zeros; so are those that are not
        // finite, and marked below
        const int kept = live ? q.tokens - (token0 + 16 * h) : 0;
#pragma unroll
        for (int b = 0; b < 8; ++b)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t x = values[b][w] & first_bytes(kept - 4 * w);
            const uint32_t at_nan = nan_bytes(x);
            strange |= at_nan;
            values[b][w] = x & ~((at_nan >> 7) * 0xffu);
          }
      }
#pragma unroll
      for (int b = 0; b < 8; ++b)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const bf16x8 v = operand8(values[b][2 * u], values[b][2 * u + 1], v_scale);
          o[b] = mfma16(v, __builtin_bit_cast(bf16x8, rest[u]), o[b]);
          o[b] = mfma16(v, __builtin_bit_cast(bf16x8, bits[u]), o[b]);
        }
      v_page = v_now;
      if (more) load_values(tile + step, v_page);
    }

    if (__any(strange != 0)) {
      // values that are not finite reach the columns that see their tokens alone: counted from the
      // codes of those tiles, by products of ones
      f32x4 count[8];
#pragma unroll
      for (int b = 0; b < 8; ++b) count[b] = f32x4{0, 0, 0, 0};
      for (tile = from + wave / Split; tile < to; tile += step) {
        const int first = static_cast<int>(tile) * kTile + 16 * h;   // this lane's sixteen tokens
        const int page = page_of(tile, h);
        if (static_cast<int>(tile) * kTile + kTile <= least && __all(page > 0)) continue;
        load_values(tile, page);
        u32x4 seen[2];
#pragma unroll
        for (int w = 0; w < 8; ++w)
          seen[w >> 2][w & 3] = (first + 2 * w < limit ? 0x3f80u : 0u) |
                                (first + 2 * w + 1 < limit ? 0x3f800000u : 0u);
#pragma unroll
        for (int b = 0; b < 8; ++b) {
          u32x4 ones;   // e4m3's 1 where a value is NaN
#pragma unroll
          for (int w = 0; w < 4; ++w) ones[w] = page > 0 ? (nan_bytes(values[b][w]) >> 7) * 0x38u : 0u;
#pragma unroll
          for (int u = 0; u < 2; ++u)
            count[b] = mfma16(operand8(ones[2 * u], ones[2 * u + 1], 1.0f),
                              __builtin_bit_cast(bf16x8, seen[u]), count[b]);
        }
      }
#pragma unroll
      for (int b = 0; b < 8; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (count[b][i] > 0.0f) o[b][i] = __builtin_nanf("");
    }

    // the waves' sums joined: thread (column, eight elements) of each sixteen columns
    const bool entire = from == 0 && to == tiles;
    float* const piece = a.workspace + layout.piece(blockIdx.x, at == start ? 0 : 1);
    sum = add_partner<32>(add_partner<16>(sum));
    if (h == 0) {
      stats[wave][0][m] = top;
      stats[wave][1][m] = sum;
    }
#pragma unroll
    for (int b = 0; b < 8; ++b) *reinterpret_cast<f32x4*>(&sums[wave][m][16 * b + 4 * h]) = o[b];
    __syncthreads();
    const int mine = threadIdx.x >> 4, d = 8 * (threadIdx.x & 15);
#pragma unroll
    for (int ct = 0; ct < Split; ++ct) {
      const int joined = column0 + 16 * ct + mine;
      const int t = joined / a.group;
      if (joined >= p.columns || t >= rows) continue;
      float best = -__builtin_inff(), all = 0.0f, x[8] = {};
#pragma unroll
      for (int w = ct; w < kWaves; w += Split) best = fmaxf(best, stats[w][0][mine]);
#pragma unroll
      for (int w = ct; w < kWaves; w += Split) {
        const float theirs = stats[w][0][mine];
        const float keep = theirs == best ? 1.0f : exp2_fast((theirs - best) * a.log2_scale);
        if (theirs > -__builtin_inff()) {
          all = fmaf(stats[w][1][mine], keep, all);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = fmaf(sums[w][mine][d + i], keep, x[i]);
        }
      }
      if (entire) {
        store_out(a, q.first + t, head * a.group + joined - t * a.group, d, x, best, all);
      } else {
        float* const to_o = piece + static_cast<int64_t>(joined) * kDim + d;
        *reinterpret_cast<f32x4*>(to_o) = f32x4{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<f32x4*>(to_o + 4) = f32x4{x[4], x[5], x[6], x[7]};
        if (d == 0)
          *reinterpret_cast<f32x2*>(piece + layout.columns * kDim + 2 * joined) = f32x2{best, all};
      }
    }
    __syncthreads();
    at += to - from;
  }
}

// Some columns of a request and kv head a workgroup: joins the sums of the runs that its tiles were
// cut into; zeros for a request without tokens or with more rows than the width.  Groups of threads
// take every Groups-th piece, a thread eight elements of a column.
// Four columns and eight groups start sooner than sixteen and four (both launches in a graph, 8 q heads on
// each of 2: one request of 177 tokens 8.4 and 8.7 us, of 7,000 17.7 and 26.2, 32 of 125 to 1,000 10.9 and
// 11.9, 64 of four rows and 500 to 4,000 25.9 and 25.7).  A head that may be in more than 48 pieces has two
// columns and 32 groups (one request of 7,000 tokens 13.4 and 17.7, of 35,000 18.0 and 27.1, of 100,000, 223
// pieces, 23.8 and 34.4; four of 20,000, 63 pieces, 19.7 and 20.8; of 177 in a table for 100,000s 9.4 and
// 8.6).
constexpr int kJoinColumns = 4, kJoinGroups = 8;
constexpr int kFewColumns = 2, kFewGroups = 32;
constexpr int kManyPieces = 48;
template <int Columns, int Groups>
__global__ __launch_bounds__(Columns * 16 * Groups) void attention_join_kernel(const DecodeAttention p,
                                                                               Layout layout, int parts) {
  const Cache& c = p.cache;
  const Attention& a = p.a;
  const int part = blockIdx.x % parts;
  const int rest = blockIdx.x / parts;
  const int head = rest % c.kv_heads;
  const int r = rest / c.kv_heads;
  const uint32_t* const plan = reinterpret_cast<const uint32_t*>(a.workspace);
  const uint32_t run = plan[0], first = plan[1 + r];
  const uint32_t tiles = plan[2 + r] - first;
  const Request q = request_of(c, r);
  const int64_t rows = q.last - q.first;
  const int group = threadIdx.x / (16 * Columns);
  const int mine = (threadIdx.x >> 4) % Columns, d = 8 * (threadIdx.x & 15);
  const int column = Columns * part + mine;
  const int t = column / a.group;
  const int q_head = head * a.group + column - t * a.group;
  if (tiles == 0) {
    const u32x4 none = {0, 0, 0, 0};
    if (group == 0 && column < p.columns)
      for (int64_t row = q.first + t; row < q.last; row += a.width)
        __builtin_memcpy(a.out + (row * a.q_heads + q_head) * kDim + d, &none, 16);
    return;
  }
  const uint32_t begin = first * c.kv_heads + head * tiles;
  const uint32_t w0 = begin / run, w1 = (begin + tiles - 1) / run;
  if (w0 == w1) return;   // one run had them all
  const bool real = column < p.columns && t < rows;
  float best = -__builtin_inff(), all = 0.0f, x[8] = {};
  if (real) {
#pragma unroll 4
    for (uint32_t w = w0 + group; w <= w1; w += Groups) {
      const float* const from = a.workspace + layout.piece(w, w == w0 && begin != w * run);
      const f32x2 stat = *reinterpret_cast<const f32x2*>(from + layout.columns * kDim + 2 * column);
      const f32x4 lo = *reinterpret_cast<const f32x4*>(from + static_cast<int64_t>(column) * kDim + d);
      const f32x4 hi = *reinterpret_cast<const f32x4*>(from + static_cast<int64_t>(column) * kDim + d + 4);
      const float now = fmaxf(best, stat[0]);
      if (stat[0] > -__builtin_inff()) {   // (what saw nothing has sums of zero)
        const float keep = best == now ? 1.0f : exp2_fast((best - now) * a.log2_scale);
        const float add = stat[0] == now ? 1.0f : exp2_fast((stat[0] - now) * a.log2_scale);
        best = now;
        all = all * keep + stat[1] * add;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = x[i] * keep + lo[i] * add;
          x[4 + i] = x[4 + i] * keep + hi[i] * add;
        }
      }
    }
  }
  __shared__ __attribute__((aligned(16))) float sums[Groups][Columns][kDim + 4];
  __shared__ f32x2 stats[Groups][Columns];
  *reinterpret_cast<f32x4*>(&sums[group][mine][d]) = f32x4{x[0], x[1], x[2], x[3]};
  *reinterpret_cast<f32x4*>(&sums[group][mine][d + 4]) = f32x4{x[4], x[5], x[6], x[7]};
  if (d == 0) stats[group][mine] = f32x2{best, all};
  __syncthreads();
  if (group > 0 || !real) return;
#pragma unroll
  for (int g = 0; g < Groups; ++g) best = fmaxf(best, stats[g][mine][0]);
  all = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = 0.0f;
#pragma unroll
  for (int g = 0; g < Groups; ++g) {
    const f32x2 stat = stats[g][mine];
    if (stat[0] > -__builtin_inff()) {
      const float add = stat[0] == best ? 1.0f : exp2_fast((stat[0] - best) * a.log2_scale);
      all = fmaf(stat[1], add, all);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = fmaf(sums[g][mine][d + i], add, x[i]);
    }
  }
  store_out(a, q.first + t, q_head, d, x, best, all);
}

// Workgroups of the first launch: two a CU, fewer where tables have not a tile for each; waves a tile;
// and how often all of it for 64 columns each.
struct Shape {
  int64_t workers;
  int split, blocks;
  double most;       // tiles of 64 tokens, were every table full
  int64_t bytes;
};

Shape decode_shape(const ld_paged_cache& c, int64_t q_heads, int64_t width) {
  Shape s{};
  const int64_t columns = width * (q_heads / c.num_kv_heads);
  s.split = columns <= 16 ? 1 : columns <= 32 ? 2 : 4;
  s.blocks = static_cast<int>((columns + 16 * s.split - 1) / (16 * s.split));
  const int64_t tiles = (static_cast<int64_t>(c.table_width) * c.page_size + kTile - 1) / kTile;
  s.most = static_cast<double>(tiles) * c.num_requests * c.num_kv_heads;
  const int64_t chip = std::max<int64_t>(64, 512 / s.blocks);
  s.workers = s.most >= chip ? chip : static_cast<int64_t>(s.most) + 1;
  s.bytes = layout_of(c.num_requests, 16 * s.split * s.blocks).piece(s.workers, 0) * 4;
  return s;
}

int check_decode(const ld_paged_cache* cache, const ld_attention_args* args, DecodeAttention& p) {
  if (const int rc = cache_params(cache, p.cache)) return rc;
  if (const int rc = attention_params(*cache, args, p.a)) return rc;
  if (args->width < 1 || args->width > LD_MAX_TOKENS)
    return fail(LD_ERR_INVALID_ARGUMENT, "decode/MTP supports 1 through 4 tokens per request");
  return LD_OK;
}

}  // namespace
}  // namespace ld

extern "C" int64_t ld_attention_decode_workspace_bytes(const ld_paged_cache* cache,
                                                       const ld_attention_args* args) {
  using namespace ld;
  if (cache == nullptr || args == nullptr || cache->num_requests <= 0 || cache->num_tokens <= 0 ||
      cache->num_kv_heads <= 0 || args->num_q_heads < cache->num_kv_heads || args->width < 1 ||
      args->width > LD_MAX_TOKENS || cache->table_width < 0)
    return 0;
  return decode_shape(*cache, args->num_q_heads, args->width).bytes;
}

extern "C" int ld_attention_decode(const ld_paged_cache* cache, const ld_attention_args* args,
                                   void* stream) {
  using namespace ld;
  DecodeAttention p{};
  if (const int rc = check_decode(cache, args, p)) return rc;
  if (p.cache.requests == 0) return LD_OK;
  const Shape s = decode_shape(*cache, p.a.q_heads, p.a.width);
  if (p.a.workspace == nullptr || !aligned16(p.a.workspace) || args->workspace_bytes < s.bytes)
    return fail(LD_ERR_INVALID_ARGUMENT, "workspace missing or too small");
  p.columns = p.a.width * p.a.group;
  const bool few = s.workers > static_cast<int64_t>(kManyPieces) * p.cache.requests * p.cache.kv_heads;
  const int each = few ? kFewColumns : kJoinColumns;
  const int parts = (p.columns + each - 1) / each;
  const int64_t joins = static_cast<int64_t>(p.cache.requests) * p.cache.kv_heads * parts;
  const int join_threads = few ? kFewColumns * 16 * kFewGroups : kJoinColumns * 16 * kJoinGroups;
  if (!launches(joins, join_threads))
    return fail(LD_ERR_INVALID_ARGUMENT, "too many requests and heads");
  if (s.most > 0x3fffffff)
    return fail(LD_ERR_INVALID_ARGUMENT, "too many tokens of all tables and heads");
  p.workers = static_cast<int32_t>(s.workers);
  const auto kernel = s.split == 1   ? attention_decode_kernel<1>
                      : s.split == 2 ? attention_decode_kernel<2>
                                     : attention_decode_kernel<4>;
  const hipStream_t on = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(s.workers), s.blocks),
                     dim3(kThreads), 0, on, p);
  if (const int rc = check_launch("ld_attention_decode")) return rc;
  hipLaunchKernelGGL((few ? attention_join_kernel<kFewColumns, kFewGroups>
                          : attention_join_kernel<kJoinColumns, kJoinGroups>),
                     dim3(static_cast<uint32_t>(joins)), dim3(join_threads), 0, on, p,
                     layout_of(p.cache.requests, 16 * s.split * s.blocks), parts);
  return check_launch("ld_attention_decode");
}
