// Attention of prompts to their tokens in the paged 8-bit cache.
//
// Bound by the matrix cores: 4 * 128 operations a query and token, a tile of 64 tokens read once for
// 128 columns.  A workgroup takes 128 columns of a request and kv head (rows times the q heads that
// share it), 32 a wave, and walks the tokens that they see, 64 at a time: the tile's codes are loaded
// ahead, made bf16 (exact: e4m3 times its scale) and laid out in LDS as operands of
// v_mfma_f32_32x32x16_bf16.  With m = lane % 32 and h = lane / 32,
//   scores [token, column]: operand A holds, in row m of product t, the key of token 32 t + 16 (m / 4 % 2)
//     + 4 (m / 8) + m % 4, so that a lane finds tokens 32 t + 16 h + (0 .. 15) of column m in its registers;
//   outputs [element, column]: operand B is these weights, rounded to bf16, as they lie there (their sum
//     is of the unrounded ones).
// With a second bf16 for what the first rounds off, products are 3 for 2: 1 x 8,192 tokens 408 us and not 284,
// 13 prompts 88 and not 66, 3 behind long contexts 52 and not 43, for an error of 0.0016 of the outputs' size
// and not 0.0018, 0.0016 of it the outputs' own rounding.
// Statistics are a lane's own but for one exchange of halves.  Outputs are scaled anew only where a
// maximum grew by more than 2^8 in weights.
//
// Where there are few columns the tokens are split over workgroups too, whose sums a second launch
// joins.
//
// One prompt of 8,192 tokens, 16 q heads on 2: 284 us, 970 TFLOP/s, the matrix cores busy 46% of the cycles
// (at the 2.0 GHz that the card holds) and vector issue 43%.  13 prompts of 1 to 1,132 tokens behind up
// to 1,000, 32 q heads on 8: 66 us; three of 32 to 78 behind 5,300 to 21,200: 42, of it 11 for the join.
#include <algorithm>

#include "attention_common.h"

namespace ld {
namespace {

constexpr int kTile = 64;        // tokens
constexpr int kColumns = 128;    // of a workgroup
constexpr int kPieces = kTile * kDim * 2 / 16;   // 16 bytes each, of a tile's keys or values as operands

struct PrefillAttention {
  Cache cache;
  Attention a;
  int32_t units;    // blocks of columns of all requests, at most
  uint32_t room;    // sums that the workspace holds
};

// Where blocks of columns are fewer than CUs, a request's tokens are split over as many workgroups as
// make shares of about equal length: the plan, worked out by every workgroup from the lengths, and
// left in the workspace for the launch that joins.  Sums of a share are 66 KB, written and read
// again, so that a request whose first rows see fewer than 16 tiles is left whole (a new prompt of 1,500
// tokens 41 us, split 53), as is every one where blocks fill the CUs (one of 2,048 tokens 52 and 62);
// 512 tokens behind 2,800 take 40 us, whole 78.
constexpr int kCus = 256;
constexpr int kShares = 2 * kCus;
constexpr int kLeastShare = 8;    // tiles
constexpr int kLeastWalk = 16;

struct Share {
  uint32_t first;    // share of the request's first block, per kv head
  uint32_t splits;   // shares a block
};

struct Shares {
  Request mine;         // of this lane's request of the 64 at hand
  uint32_t splits, blocks, behind, all, before = 0;
  int base = 0;

  __device__ __forceinline__ uint32_t load(const PrefillAttention& p, int first) {
    const int r = first + (threadIdx.x & 63);
    base = first;
    mine = request_of(p.cache, min(r, p.cache.requests - 1));
    const int64_t rows = r < p.cache.requests ? max(mine.last - mine.first, int64_t{0}) : 0;
    blocks = (static_cast<uint32_t>(rows) * p.a.group + kColumns - 1) / kColumns;
    return (static_cast<uint32_t>(mine.tokens) + kTile - 1) / kTile;   // tiles of its last block
  }
  __device__ __forceinline__ void split(uint32_t tiles, uint32_t share) {
    splits = mine.first + mine.shift < kLeastWalk * kTile ? 1u : (tiles + share - 1) / share;
    behind = sum_up_to(blocks * splits);
    all = __builtin_amdgcn_readlane(behind, 63);
  }
  // The share's length: all tiles over the shares, a little more for what 32 bits round off, so that
  // shares are at most kShares and a block and kv head's one more.
  __device__ __forceinline__ uint32_t length(const PrefillAttention& p, uint32_t& tiles) {
    float total = 0.0f;
    for (int first = 0;; first += 64) {
      tiles = load(p, first);
      total += wave_sum(static_cast<float>(blocks) * tiles);
      if (first + 64 >= p.cache.requests) break;
    }
    if (p.cache.requests > 64) tiles = load(p, 0);
    const float each = total * p.cache.kv_heads * (1.0001f / kShares);
    return max(static_cast<uint32_t>(min(each, 1e9f)) + 1, static_cast<uint32_t>(kLeastShare));
  }
};

// Share -> request, block of its columns and which of its splits; false where there is none.
__device__ __forceinline__ bool find_share(const PrefillAttention& p, uint32_t share, Share* plan,
                                           int& r, Request& q, int& block, int& split, int& splits) {
  Shares s;
  uint32_t tiles;
  const uint32_t length = s.length(p, tiles);
  s.split(tiles, length);
  if (plan != nullptr) {
    for (;;) {
      const int mine = s.base + (threadIdx.x & 63);
      if (mine < p.cache.requests)
        plan[mine] = Share{s.before + s.behind - s.blocks * s.splits, s.splits};
      if (s.base + 64 >= p.cache.requests) break;
      s.before += s.all;
      tiles = s.load(p, s.base + 64);
      s.split(tiles, length);
    }
    s.before = 0;
    if (p.cache.requests > 64) s.split(s.load(p, 0), length);
  }
  while (share >= s.before + s.all) {
    if (s.base + 64 >= p.cache.requests) return false;
    s.before += s.all;
    tiles = s.load(p, s.base + 64);
    s.split(tiles, length);
  }
  const uint32_t local = share - s.before;
  const int k = __popcll(__ballot(s.behind <= local));
  splits = __builtin_amdgcn_readlane(s.splits, k);
  const uint32_t first = __builtin_amdgcn_readlane(s.behind, k) -
                         __builtin_amdgcn_readlane(s.blocks, k) * splits;
  r = s.base + k;
  q = request_from(s.mine, k);
  block = (local - first) / splits;
  split = (local - first) % splits;
  return true;
}

// Unit -> request, what it has in the call, and block of its columns; false where there is none.
// Requests have a run of units each, one more than their columns can fill at the most.  (The host has
// seen to it that columns are below 2^31.)
__device__ __forceinline__ bool find_unit(const PrefillAttention& p, int unit, int& r, Request& q,
                                          int& block) {
  return find_run(p.cache, unit, r, q, block, [&](int row, int request) {
    return static_cast<int>(static_cast<uint32_t>(row) * p.a.group / kColumns) + request;
  });
}

__device__ __host__ inline int64_t plan_floats(int64_t requests) { return (2 * requests + 3) & ~int64_t{3}; }
__device__ __forceinline__ float* split_at(const PrefillAttention& p, int64_t place) {
  return p.a.workspace + plan_floats(p.cache.requests) + place * kColumns * (kDim + 2);
}

// Four elements of an output: divided, gated and rounded.
__device__ __forceinline__ void store_four(const Attention& a, int64_t row, int head, int d, f32x4 o,
                                           bool some, float inverse) {
  if (a.gate != nullptr && some) {
    uint16_t g[4];
    __builtin_memcpy(g, a.gate + row * a.gate_row + head * kDim + d, 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] *= sigmoid(bf16_to_f32(g[i]));
  }
  uint32_t bits[2] = {0, 0};
  if (some) {
    bits[0] = bf16_pair(f32x2{o[0] * inverse, o[1] * inverse});
    bits[1] = bf16_pair(f32x2{o[2] * inverse, o[3] * inverse});
  }
  __builtin_memcpy(a.out + (row * a.q_heads + head) * kDim + d, bits, 8);
}

// Eight elements of an output that is divided already, gated and rounded.
__device__ __forceinline__ void store_out(const Attention& a, int64_t row, int head, int d,
                                          float (&o)[8], bool some) {
  if (a.gate != nullptr) {
    uint16_t g[8];
    __builtin_memcpy(g, a.gate + row * a.gate_row + head * kDim + d, 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] *= sigmoid(bf16_to_f32(g[i]));
  }
  u32x4 bits;
#pragma unroll
  for (int i = 0; i < 4; ++i) bits[i] = some ? bf16_pair(f32x2{o[2 * i], o[2 * i + 1]}) : 0u;
  __builtin_memcpy(a.out + (row * a.q_heads + head) * kDim + d, &bits, 16);
}

// Split: workgroups are shares, else units.
template <bool Split>
__global__ __launch_bounds__(kThreads, 2) void attention_prefill_kernel(const PrefillAttention p) {
  const Cache& c = p.cache;
  const Attention& a = p.a;
  // the tile's keys: [16 elements of a token][half of them][token in the operand's order], and its
  // values [16 tokens][half of them][element], in pieces of eight
  __shared__ __attribute__((aligned(16))) u32x4 lds[4][kPieces];
  u32x4 (&lds_keys)[2][kPieces] = reinterpret_cast<u32x4(&)[2][kPieces]>(lds[0]);
  u32x4 (&lds_values)[2][kPieces] = reinterpret_cast<u32x4(&)[2][kPieces]>(lds[2]);
  __shared__ int lds_strange;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 31, h = lane >> 5;

  const int head = blockIdx.x % c.kv_heads;
  const int rest = blockIdx.x / c.kv_heads;
  int r, block, split = 0, splits = 1;
  Request q;
  if constexpr (Split) {
    Share* const plan = blockIdx.x == 0 && wave == 0 ? reinterpret_cast<Share*>(a.workspace) : nullptr;
    if (!find_share(p, rest, plan, r, q, block, split, splits)) return;
  } else {
    if (!find_unit(p, p.units - 1 - rest, r, q, block)) return;   // (a request's longest walks first)
  }
  const int columns = static_cast<int>(q.last - q.first) * a.group;   // (none: not above zero)
  if (block * kColumns >= columns) return;
  const int32_t* const table = c.pages + r * c.pages_row;

  // this lane's column, and how many tokens it, the wave's first and last and the workgroup's last see
  const int column = block * kColumns + 32 * wave + m;
  auto sees = [&](uint32_t t) {
    return static_cast<int>(max(min(q.first + t + q.shift + 1, static_cast<int64_t>(q.tokens)), int64_t{0}));
  };
  const bool real = column < columns;
  const uint32_t group = a.group;
  const uint32_t t_row = (real ? column : columns - 1) / group;
  const int g_row = (real ? column : columns - 1) - t_row * group;
  const int limit = sees(t_row);
  const int least = __builtin_amdgcn_readlane(limit, 0);
  const int first_limit = sees(block * kColumns / group);
  const int all_tiles = (sees((min(block * kColumns + kColumns, columns) - 1) / group) + kTile - 1) / kTile;
  const int each = (all_tiles + splits - 1) / splits;
  const int begin = min(split * each, all_tiles), end = min(begin + each, all_tiles);
  const bool works = block * kColumns + 32 * wave < columns;

  bf16x8 query[8];
  {
    const uint16_t* const from = a.q + (q.first + t_row) * a.q_row + (head * a.group + g_row) * kDim;
#pragma unroll
    for (int s = 0; s < 8; ++s)
      __builtin_memcpy(&query[s], from + 16 * (2 * (s >> 1) + h) + 8 * (s & 1), 16);
  }

  f32x16 o[4];
  float top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[b][i] = 0.0f;

  // A thread's share of a tile: sixteen elements of token `lane` of chunks `wave` and `wave` + 4 of the keys, and
  // sixteen tokens (groups wave / 2 and wave / 2 + 2) of one element of the values.
  const int element = threadIdx.x & 127;
  const int slot = (lane & 32) + 8 * (lane >> 2 & 3) + 4 * (lane >> 4 & 1) + (lane & 3);
  auto page_of = [&](int tile) {
    const int token = tile * kTile + lane;
    const int page = tile < end && token < q.tokens ? table[token >> c.page_log2] : 0;
    return live_page(c, page) ? page : 0;
  };
  u32x4 keys[2], values[2];
  float k_scale, v_scale[2];
  auto load_keys = [&](int tile, int page) {
    const int in = (tile * kTile + lane) & ((1 << c.page_log2) - 1);
    const uint8_t* const at_k = k_tile(c, page, head) + (((wave << c.page_log2) + in) << 4);
    keys[0] = *reinterpret_cast<const u32x4*>(at_k);
    keys[1] = *reinterpret_cast<const u32x4*>(at_k + (64 << c.page_log2));
    k_scale = scale_value(c.k_scale[page * c.k_scale_page + head]);
  };
  auto load_values = [&](int tile, int page) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int group = (wave >> 1) + 2 * i;
      const int theirs = __builtin_amdgcn_readlane(page, 16 * group);
      const int at = (tile * kTile + 16 * group) & ((1 << c.page_log2) - 1);
      values[i] = *reinterpret_cast<const u32x4*>(v_tile(c, theirs, head) + (at >> 4) * (kDim * 16) +
                                                  element * 16);
      v_scale[i] = scale_value(c.v_scale[theirs * c.v_scale_page + head]);
    }
  };
  auto stage_keys = [&](int to) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int chunk = wave + 4 * i;
      lds_keys[to][2 * chunk * kTile + slot] =
          __builtin_bit_cast(u32x4, operand8(keys[i][0], keys[i][1], k_scale));
      lds_keys[to][(2 * chunk + 1) * kTile + slot] =
          __builtin_bit_cast(u32x4, operand8(keys[i][2], keys[i][3], k_scale));
    }
  };
  auto stage_values = [&](int tile, uint64_t live, int to) {
    // values behind the last token, or without a page, are zeros; so are those that are not finite,
    // and marked below, in tiles that some column does not see to its end
    const bool partial = tile * kTile + kTile > first_limit;
    if (partial || live != ~uint64_t{0}) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int group = (wave >> 1) + 2 * i;
        const int kept = live >> (16 * group) & 1 ? q.tokens - (tile * kTile + 16 * group) : 0;
        uint32_t any = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t x = values[i][w] & first_bytes(kept - 4 * w);
          const uint32_t at_nan = partial ? nan_bytes(x) : 0u;
          any |= at_nan;
          values[i][w] = x & ~((at_nan >> 7) * 0xffu);
        }
        if (any != 0) lds_strange = 1;
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int group = (wave >> 1) + 2 * i;
      lds_values[to][(2 * group) * kDim + element] =
          __builtin_bit_cast(u32x4, operand8(values[i][0], values[i][1], v_scale[i]));
      lds_values[to][(2 * group + 1) * kDim + element] =
          __builtin_bit_cast(u32x4, operand8(values[i][2], values[i][3], v_scale[i]));
    }
  };
  auto scores = [&](int at, f32x16 (&x)[2]) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) x[t][i] = 0.0f;
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const u32x4 k = lds_keys[at][(2 * (2 * (s >> 1) + h) + (s & 1)) * kTile + 32 * t + m];
        x[t] = mfma32(__builtin_bit_cast(bf16x8, k), query[s], x[t]);
      }
  };
  // Scores of -inf, for weights of zero, where the column does not see a token; what a new maximum
  // changes; and what scores are less by in the exponent.
  float less = 0.0f;
  auto settle = [&](int tile, uint64_t live, f32x16 (&x)[2]) {
    float most = kLowest;   // (of a score of -inf that is seen: a weight of zero, not none)
    if (!(tile * kTile + kTile <= least && live == ~uint64_t{0})) {
      bool any = false;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int token = tile * kTile + 32 * t + 16 * h;
        const bool lives = live >> (32 * t + 16 * h) & 1;
        any = any || (lives && token < limit);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (!lives || token + i >= limit) x[t][i] = -__builtin_inff();
      }
      if (!any) most = -__builtin_inff();
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) most = fmaxf(most, x[t][i]);
    const uint32_t u = __float_as_uint(most);
    const auto y = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    most = fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
    if (__any((most - top) * a.log2_scale > 8.0f)) {
      const float now = fmaxf(top, most);
      const float keep = now == top ? 1.0f : exp2_fast((top - now) * a.log2_scale);
      sum *= keep;
#pragma unroll
      for (int b = 0; b < 4; ++b) o[b] *= keep;
      top = now;
    }
    const float some = top == -__builtin_inff() ? 0.0f : top;
    less = fmaf(-some, a.log2_scale, kHeadroom);
    if (far_scores(some, a.log2_scale)) {
#pragma unroll
      for (int t = 0; t < 2; ++t) x[t] -= some;
      less = kHeadroom;
    }
  };

  if (threadIdx.x == 0) lds_strange = 0;
  __syncthreads();
  // A step finds its tile's scores settled and computes the next tile's beside the weights: keys are
  // in LDS a tile ahead of values.
  int page = page_of(begin), page_next = page_of(begin + 1), page_then = page_of(begin + 2);
  f32x16 score[2];
  if (begin < end) {
    load_keys(begin + 1, page_next);
    const u32x4 second[2] = {keys[0], keys[1]};
    const float second_scale = k_scale;
    load_keys(begin, page);
    load_values(begin, page);
    stage_keys(0);
    stage_values(begin, __ballot(page > 0), 0);
    keys[0] = second[0];
    keys[1] = second[1];
    k_scale = second_scale;
    stage_keys(1);
    lds_barrier();
    if (works) {
      scores(0, score);
      settle(begin, __ballot(page > 0), score);
    }
    lds_barrier();
  }
  auto step = [&](int tile, int now_at, f32x16 (&mine)[2], f32x16 (&next)[2]) {
    // (past the last tile pages are 0: bytes that nothing uses)
    load_values(tile + 1, page_next);
    load_keys(tile + 2, page_then);
    page = page_next;
    page_next = page_then;
    page_then = page_of(tile + 3);
    const uint64_t live = __ballot(page > 0);
    if (works) {
      __builtin_amdgcn_s_setprio(1);   // (ahead of a wave that stages: 8,192 tokens 287 us, without 317)
      scores(now_at ^ 1, next);
      bf16x8 weight[2][2];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          u32x4 bits;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float x = exp2_fast(fmaf(mine[t][8 * u + 2 * w], a.log2_scale, less));
            const float y = exp2_fast(fmaf(mine[t][8 * u + 2 * w + 1], a.log2_scale, less));
            sum += x;
            sum += y;
            bits[w] = bf16_pair(f32x2{x, y});
          }
          weight[t][u] = __builtin_bit_cast(bf16x8, bits);
        }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const u32x4 v = lds_values[now_at][(2 * (2 * t + h) + u) * kDim + 32 * b + m];
            o[b] = mfma32(__builtin_bit_cast(bf16x8, v), weight[t][u], o[b]);
          }
      // (a product of the next scores, an operand read and seven of the weights' instructions at a time)
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 7, 0);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
    stage_values(tile + 1, live, now_at ^ 1);
    stage_keys(now_at);
    if (works) settle(tile + 1, live, next);
    lds_barrier();
  };
  f32x16 other[2];
  for (int tile = begin; tile < end; tile += 2) {
    step(tile, 0, score, other);
    if (tile + 1 < end) step(tile + 1, 1, other, score);
  }

  if (lds_strange) {
    // values that are not finite reach the columns that see their tokens alone: counted from the
    // codes of those tiles, by products of ones
    f32x16 count[4];
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) count[b][i] = 0.0f;
    for (int tile = max(begin, first_limit / kTile); tile < end; ++tile)
      for (int t = 0; t < 2; ++t) {
        const int first = tile * kTile + 32 * t + 16 * h;   // this lane's sixteen tokens
        const int page = first < q.tokens ? table[first >> c.page_log2] : 0;
        u32x4 seen[2];
#pragma unroll
        for (int w = 0; w < 8; ++w)
          seen[w >> 2][w & 3] = (first + 2 * w < limit ? 0x3f80u : 0u) |
                                (first + 2 * w + 1 < limit ? 0x3f800000u : 0u);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          u32x4 codes = {0, 0, 0, 0};
          if (live_page(c, page)) {
            const int in = first & ((1 << c.page_log2) - 1);
            codes = *reinterpret_cast<const u32x4*>(v_tile(c, page, head) +
                                                    ((in >> 4) * kDim + 32 * b + m) * 16);
          }
#pragma unroll
          for (int w = 0; w < 4; ++w) codes[w] = (nan_bytes(codes[w]) >> 7) * 0x38u;   // e4m3's 1
#pragma unroll
          for (int u = 0; u < 2; ++u)
            count[b] = mfma32(operand8(codes[2 * u], codes[2 * u + 1], 1.0f),
                              __builtin_bit_cast(bf16x8, seen[u]), count[b]);
        }
      }
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (count[b][i] > 0.0f) o[b][i] = __builtin_nanf("");
  }
  sum = add_partner<32>(sum);
  if (splits == 1) {
    // by way of LDS, a wave's 32 columns a quarter of it, so that sixteen lanes store a row's 256 bytes
    // (a lane's own are sixteen pieces of 8, stored so 128 prompts of 128 tokens take 63 us, now 58); piece j
    // of column n at j ^ n
    __syncthreads();   // (the last values read)
    u32x4* const mine = lds[wave];
    const bool some = top > -__builtin_inff();   // the row sees a token
    const float inverse = 1.0f / sum;
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f32x4 x = quad(o[b], e);
        x *= inverse;
        mine[32 * m + ((8 * b + 2 * e + h) ^ m)] = __builtin_bit_cast(u32x4, x);
      }
    lds_order();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int n = 4 * i + (lane >> 4), j = lane & 15;
      const int t = __shfl(static_cast<int>(t_row), n), g = __shfl(g_row, n);
      const bool any = __shfl(some ? 1 : 0, n) != 0;
      if (block * kColumns + 32 * wave + n >= columns) continue;
      const f32x4 lo = __builtin_bit_cast(f32x4, mine[32 * n + ((2 * j) ^ n)]);
      const f32x4 hi = __builtin_bit_cast(f32x4, mine[32 * n + ((2 * j + 1) ^ n)]);
      float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      store_out(a, q.first + t, head * a.group + g, 8 * j, x, any);
    }
  } else if (real) {
    float* const to = split_at(p, blockIdx.x);
    const int at = 32 * wave + m;
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<f32x4*>(to + at * kDim + 32 * b + 8 * e + 4 * h) = quad(o[b], e);
    if (h == 0) *reinterpret_cast<f32x2*>(to + kColumns * kDim + 2 * at) = f32x2{top, sum};
  }
}

// Joins the sums of a unit's shares: thread (column, four elements), eight columns a workgroup and
// Groups of threads that take every Groups-th share.  Few units have many shares each: four groups (three
// prompts behind up to 21,200 tokens, 30 shares: 10 us, one group 23); with more, whose shares are
// few, the threads of one group start in less time (one prompt of 1,024 tokens 32 us in all, four 37).
constexpr int kGatherColumns = 8;
constexpr int kFewUnits = 64;
template <int Groups>
__global__ __launch_bounds__(Groups * 256) void attention_gather_kernel(const PrefillAttention p) {
  const Cache& c = p.cache;
  const Attention& a = p.a;
  const int part = blockIdx.x % (kColumns / kGatherColumns);
  const int rest = blockIdx.x / (kColumns / kGatherColumns);
  const int head = rest % c.kv_heads;
  int r, block;
  Request q;
  if (!find_unit(p, rest / c.kv_heads, r, q, block)) return;
  const int columns = static_cast<int>(q.last - q.first) * a.group;
  if (block * kColumns + part * kGatherColumns >= columns) return;
  const Share plan = reinterpret_cast<const Share*>(a.workspace)[r];
  const uint32_t first = plan.first + block * plan.splits;
  // (rows that two requests claim make a plan that the workspace has no room for)
  if (plan.splits == 1 || static_cast<uint64_t>(first + plan.splits) * c.kv_heads > p.room) return;
  const int group = threadIdx.x >> 8;
  const int mine = threadIdx.x >> 5 & 7;
  const int within = part * kGatherColumns + mine;
  const int column = block * kColumns + within;
  const int d = 4 * (threadIdx.x & 31);
  float best = -__builtin_inff(), all = 0.0f;
  f32x4 x = {0, 0, 0, 0};
  auto add = [&](float top, float total, f32x4 theirs) {
    if (top > -__builtin_inff()) {   // (what saw nothing has sums of zero)
      const float now = fmaxf(best, top);
      const float keep = best == now ? 1.0f : exp2_fast((best - now) * a.log2_scale);
      const float by = top == now ? 1.0f : exp2_fast((top - now) * a.log2_scale);
      best = now;
      all = all * keep + total * by;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = x[i] * keep + theirs[i] * by;
    }
  };
  if (column < columns) {
#pragma unroll 8
    for (uint32_t s = group; s < plan.splits; s += Groups) {
      const float* const from = split_at(p, static_cast<int64_t>(first + s) * c.kv_heads + head);
      const f32x2 stat = *reinterpret_cast<const f32x2*>(from + kColumns * kDim + 2 * within);
      add(stat[0], stat[1], *reinterpret_cast<const f32x4*>(from + within * kDim + d));
    }
  }
  if constexpr (Groups > 1) {
    __shared__ f32x4 sums[Groups - 1][kGatherColumns][32];
    __shared__ f32x2 stats[Groups - 1][kGatherColumns];
    if (group > 0) {
      sums[group - 1][mine][threadIdx.x & 31] = x;
      if (d == 0) stats[group - 1][mine] = f32x2{best, all};
    }
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int g = 0; g < Groups - 1; ++g)
      add(stats[g][mine][0], stats[g][mine][1], sums[g][mine][threadIdx.x & 31]);
  }
  if (column >= columns) return;
  const int t = column / a.group;
  store_four(a, q.first + t, head * a.group + column - t * a.group, d, x,
             best > -__builtin_inff(), 1.0f / all);
}

// Blocks of columns, at most, and workgroups: one a block and kv head, or shares where those would not
// give each CU one and a table holds tokens for more than one.
struct Shape {
  int64_t units, blocks, bytes;
};

Shape prefill_shape(const ld_paged_cache& c, int64_t q_heads) {
  Shape s{};
  const int64_t group = q_heads / c.num_kv_heads;
  s.units = c.num_tokens * group / kColumns + c.num_requests;
  s.blocks = s.units * c.num_kv_heads;
  if (s.blocks < kCus &&
      static_cast<int64_t>(c.table_width) * c.page_size > kTile * kLeastWalk) {
    s.blocks += kShares;
    s.bytes = (plan_floats(c.num_requests) + s.blocks * kColumns * (kDim + 2)) * 4;
  }
  return s;
}

}  // namespace
}  // namespace ld

extern "C" int64_t ld_attention_prefill_workspace_bytes(const ld_paged_cache* cache,
                                                        const ld_attention_args* args) {
  using namespace ld;
  if (cache == nullptr || args == nullptr || cache->num_requests <= 0 || cache->num_tokens <= 0 ||
      cache->num_kv_heads <= 0 || args->num_q_heads < cache->num_kv_heads || cache->table_width < 0)
    return 0;
  return prefill_shape(*cache, args->num_q_heads).bytes;
}

extern "C" int ld_attention_prefill(const ld_paged_cache* cache, const ld_attention_args* args,
                                    void* stream) {
  using namespace ld;
  PrefillAttention p{};
  if (const int rc = cache_params(cache, p.cache)) return rc;
  if (const int rc = attention_params(*cache, args, p.a)) return rc;
  if (p.cache.requests == 0) return LD_OK;
  const Shape s = prefill_shape(*cache, p.a.q_heads);
  if (s.bytes > 0 && (p.a.workspace == nullptr || !aligned16(p.a.workspace) ||
                      args->workspace_bytes < s.bytes))
    return fail(LD_ERR_INVALID_ARGUMENT, "workspace missing or too small");
  if (!launches(s.blocks, kThreads) || p.cache.num_tokens * p.a.group > 0x7fffff00)
    return fail(LD_ERR_INVALID_ARGUMENT, "too many rows and heads");
  p.units = static_cast<int32_t>(s.units);
  p.room = static_cast<uint32_t>(s.blocks);
  const hipStream_t on = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<uint32_t>(s.blocks));
  if (s.bytes == 0) {
    hipLaunchKernelGGL(attention_prefill_kernel<false>, grid, dim3(kThreads), 0, on, p);
    return check_launch("ld_attention_prefill");
  }
  hipLaunchKernelGGL(attention_prefill_kernel<true>, grid, dim3(kThreads), 0, on, p);
  if (const int rc = check_launch("ld_attention_prefill")) return rc;
  // (fewer than 256 units and heads)
  const int64_t joins = s.units * p.cache.kv_heads * (kColumns / kGatherColumns);
  const int groups = s.units * p.cache.kv_heads <= kFewUnits ? 4 : 1;
  hipLaunchKernelGGL(groups == 4 ? attention_gather_kernel<4> : attention_gather_kernel<1>,
                     dim3(static_cast<uint32_t>(joins)), dim3(groups * 256), 0, on, p);
  return check_launch("ld_attention_prefill");
}
