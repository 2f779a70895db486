// Prefill of linear attention with a decay for each head, for gfx950:
//   S <- exp(g) S + v k^T ;  o = scale * S q ;  out = o, or its gated RMSNorm
// in chunks of 64 tokens.  With c_t the sum of g over the chunk's tokens up to t:
//   o_t = scale (e^(c_t) S q_t + sum over s <= t of e^(c_t - c_s) (k_s . q_t) v_s)
//   S'  = e^(c_63) S + sum over s of k_s (e^(c_63 - c_s) v_s)^T
//
// A workgroup of four waves walks the chunks of one (sequence, v-head).  Wave w owns state rows
// v = 32 w .. 32 w + 31 as S^T in the accumulators of v_mfma_f32_32x32x16_bf16, with the summation
// index assigned as in prefill_heads.hip: for lane l, lj = l % 32 and hi = l / 32, an accumulator
// holds rows i(r) = 8 (r / 4) + 4 hi + r % 4, r < 16, of column lj, so its registers 8 u ..
// 8 u + 7, split into bf16 planes, are directly the operand of step u of the next product; keys
// are in an order in which a step takes 16 consecutive bytes of a q row, step u of a sum over
// tokens takes token 16 u + 8 (e / 4) + 4 hi + e % 4.
//   O^T = S Q^T        S as three planes
//   P = (K Q^T) . D    32 x 32 blocks over the waves, three planes, exchanged through LDS
//   O^T = O^T diag(e^c) + V^T P^T
//   S' = e^(c_63) S + K^T (e^(c_63 - c) V)    e V as three planes
// O crosses LDS in fp32, in the place of v, to whole rows, whose norm and 16-byte stores run
// beside the next chunk's first products.  The transposed operands come by ds_read_b64_tr_b16.
//
// Decays come from differences of 64-bit prefix sums: their error over thousands of tokens would
// be the state's.  Operands of the bf16 matrix cores, whose sums are fp32, are taken exactly: three
// planes hold fp32's 24 bits.  (Two planes of S and P, 16 bits, leave the outputs' error what bf16's
// rounding, up to 2^-8 of a value, makes it, but round one output in 500 to the other neighbour,
// against one in 9,000; 32 prompts of 1024 tokens then take 326 us, with three of S alone 355, with
// three of both 366.)
//
// Bound by issue, with memory close behind.  32 prompts of 1024 tokens, 32 v-heads and a norm: 329 to
// 367 us as clock and power allow (313 to 318 without the norm; their bytes at a large copy's rate,
// 236), in which two waves a SIMD keep the vector unit busy 43% and the matrix cores 44% of the time,
// mostly by turns: two workgroups a CU finish a chunk each in 10.7 us, one alone in 5.0.  512 prompts of
// 8 to 56 tokens: 427 to 433 us of 394, states read and written at 4.7 TB/s.  Hence the layout: operands that
// stay in registers, remainders by matrix products, no branch around a load, four waves of 32 columns
// (against eight of 16, which read every K and Q operand twice: 415 us and 332 at one time).
//
// A sequence longer than a segment is cut into segments, since the recurrence over them is
// associative: one launch reduces every segment but a sequence's last to the state after it from zeros
// and its decay, a second (where there are many) joins these along each sequence, a third walks all
// segments from the joined states, and the sequences of one segment.  One prompt of 4096 tokens and
// 32 heads, 16 segments: 23 and 63 us by the kernel trace, 78 to 84 a call in a loop (walked in one
// piece by 32 workgroups, 64 chunks' chain alone would be 320).
#include <algorithm>
#include <cstddef>

#include "linear_common.h"
#include "matrix_common.h"

namespace ld {
namespace {

constexpr int kBlockWaves = 4;
constexpr int kBlock = 64 * kBlockWaves;
constexpr int kTokens = 64;                     // tokens per chunk
constexpr int kRowsBytes = kTokens * kTileRow;  // q, k or v of a chunk
constexpr int kPlaneUpper = 32 * 32 * 2;
constexpr int kPlaneBytes = kPlaneUpper + 32 * 64 * 2;
constexpr int64_t kTileFloats = kDim * kDim;
constexpr int64_t kMaxRow = 1 << 23;            // a chunk's rows within 32-bit byte offsets

// Per-token scalars of a chunk: c in units of log 2 as a sum of two floats, scale * e^c and
// e^(c_63 - c); and e^(c_63).
struct alignas(16) ChunkScalars {
  float hi[kTokens], lo[kTokens], eq[kTokens], ek[kTokens];
  float gamma;
};

struct SegmentLds {
  alignas(16) uint8_t k[kRowsBytes];
  alignas(16) uint8_t q[kRowsBytes];
  // v; behind it, in its place and another 16 KiB, the chunk's O in fp32
  alignas(16) uint8_t v[kTokens * kDim * 4];
  // two planes of P: 32 rows of 32 columns, 32 of 64; the third is behind v
  alignas(16) uint8_t p[2][kPlaneBytes];
  ChunkScalars scalars[2];
  alignas(16) float weight[kDim];
  int nonfinite[kDim];   // per column, where a wave says so, the chunk's first v that is not finite
};
struct SearchLds {
  int wave_sums[kBlockWaves];
  int found[3];
};
static_assert(offsetof(SegmentLds, v) + sizeof(SegmentLds::v) == kTileBytes, "k, q and v are a tile");
static_assert(2 * (sizeof(SegmentLds) + sizeof(SearchLds)) <= 160 * 1024, "two workgroups a CU");

// bf16 of registers 8 u .. 8 u + 7 of an accumulator: an operand of step u.
__device__ __forceinline__ bf16x8 plane_of(const f32x16& x, int u) {
  u32x4 w;
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = bf16_pair(f32x2{x[8 * u + 2 * j], x[8 * u + 2 * j + 1]});
  return __builtin_bit_cast(bf16x8, w);
}

// x less its planes, by products with -1: the matrix cores have the room that vector issue, which
// bounds the kernel, has not (two products instead of 32 vector instructions; exact either way,
// as fp32 holds what rounding to bf16 leaves).
struct Remainder {
  bf16x8 minus[2];   // A[i][k] of step u: -1 where row i is the step's summation index k
  __device__ __forceinline__ explicit Remainder(int lane) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      u32x4 w = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int row = 16 * u + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
        if (row == (lane & 31)) w[e >> 1] |= e & 1 ? 0xbf800000u : 0xbf80u;
      }
      minus[u] = __builtin_bit_cast(bf16x8, w);
    }
  }
  __device__ __forceinline__ f32x16 operator()(const f32x16& x, bf16x8 p0, bf16x8 p1) const {
    return mfma32(minus[1], p1, mfma32(minus[0], p0, x));
  }
};

__device__ __forceinline__ double read_lane(double x, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(u), lane);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(u >> 32), lane);
  return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}

// Inclusive sums over the 64 lanes.
__device__ __forceinline__ double prefix_sum64(double x, int lane) {
  x += dpp64<0x111>(x);   // row_shr:1, 2, 4, 8: zeros from below the row
  x += dpp64<0x112>(x);
  x += dpp64<0x114>(x);
  x += dpp64<0x118>(x);
  const double row0 = read_lane(x, 15), row1 = read_lane(x, 31), row2 = read_lane(x, 47);
  if (lane >= 16) x += row0;
  if (lane >= 32) x += row1;
  if (lane >= 48) x += row2;
  return x;
}

// The scalars of a chunk whose token `lane` has log decay g (0 past the end), by one wave;
// returns the sum of g in units of log 2.  Below -150 a decay is 0 in fp32 like -inf's, which a
// sum could not hold.
__device__ __forceinline__ double chunk_scalars(ChunkScalars& s, float g, float scale, int lane) {
  const double c = prefix_sum64(static_cast<double>(g < -150.0f ? -150.0f : g) *
                                    1.4426950408889634, lane);
  const double total = read_lane(c, 63);
  const float hi = static_cast<float>(c);
  s.hi[lane] = hi;
  s.lo[lane] = static_cast<float>(c - hi);
  s.eq[lane] = scale * __builtin_amdgcn_exp2f(hi);
  s.ek[lane] = __builtin_amdgcn_exp2f(static_cast<float>(total - c));
  if (lane == 0) s.gamma = __builtin_amdgcn_exp2f(static_cast<float>(total));
  return total;
}

// Keeps LDS reads, matrix instructions and global loads in the program's order (vector and
// scalar instructions may cross): reads stay the distance ahead of their use that the source gives them.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0x406); }

__device__ __forceinline__ bf16x8 join(bf16x4 a, bf16x4 b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

constexpr int kScalarWave = 3;   // makes the chunks' scalars: the wave without a block of P

// The state in a wave's accumulators, st[T][8 u + 4 h + r] = S[32 w + lj][32 T + 16 u + 8 hi + 4 h + r],
// to and from memory by way of LDS, so that memory is read and written in whole lines: row v's
// 16-byte pieces are XORed with v % 16.
struct StateTile {
  uint8_t* tile;
  uint32_t at;
  __device__ __forceinline__ explicit StateTile(SegmentLds& lds) : tile(lds.k) {
    const int tid = threadIdx.x, lj = tid & 31, hi = (tid >> 5) & 1;
    at = (32 * (tid >> 6) + lj) * (kDim * 4) + (((2 * hi) ^ (lj & 15)) << 4);
  }
  __device__ __forceinline__ f32x4* piece(int T, int q) const {   // of st[T][4 q ..]
    return reinterpret_cast<f32x4*>(tile + (at ^ ((8 * T + 4 * (q >> 1) + (q & 1)) << 4)));
  }
  __device__ __forceinline__ f32x4* line(int i) const {           // the thread's 16 bytes of line i
    const int tid = threadIdx.x, v = 8 * i + (tid >> 5);
    return reinterpret_cast<f32x4*>(tile + v * (kDim * 4) + (((tid & 31) ^ (v & 15)) << 4));
  }
  // From the pool, and a copy in `kept` unless null.
  __device__ __forceinline__ void load(const float* from, float* kept, f32x16 (&st)[4]) const {
    const __amdgpu_buffer_rsrc_t rs = buffer_rsrc(from, kTileBytes);
    f32x4 lines[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) lines[i] = buffer_load16<kPolNTSys>(rs, threadIdx.x * 16 + 4096 * i);
    if (kept != nullptr) {
      const __amdgpu_buffer_rsrc_t copy = buffer_rsrc(kept, kTileBytes);
#pragma unroll
      for (int i = 0; i < 16; ++i) buffer_store16<kPolPlain>(lines[i], copy, threadIdx.x * 16 + 4096 * i);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) *line(i) = lines[i];
    take(st);
  }
  // From the workspace: `count` tiles, each (but the first) added to its decay times those ahead.
  __device__ __forceinline__ void load_joined(const float* tiles, const float* decays, int count,
                                              int num_v_heads, f32x16 (&st)[4]) const {
    constexpr int kFlight = 2, kLines = 8;   // tiles in flight, half of their lines at a time
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      f32x4 sum[kLines] = {}, part[kFlight][kLines];
      auto fetch = [&](int a, int k) __attribute__((always_inline)) {   // (past the last, that again)
        const __amdgpu_buffer_rsrc_t rs =
            buffer_rsrc(tiles + min(k, count - 1) * (num_v_heads * kTileFloats), kTileBytes);
#pragma unroll
        for (int i = 0; i < kLines; ++i)
          part[a][i] = buffer_load16<kPolPlain>(rs, threadIdx.x * 16 + 4096 * (kLines * half + i));
      };
#pragma unroll
      for (int a = 0; a < kFlight; ++a) fetch(a, a);
      for (int k = 0; k < count; k += kFlight) {
#pragma unroll
        for (int a = 0; a < kFlight; ++a) {
          if (k + a < count) {
            const float by = k + a == 0 ? 0.0f : decays[(k + a) * num_v_heads];
#pragma unroll
            for (int i = 0; i < kLines; ++i) sum[i] = sum[i] * by + part[a][i];
          }
          fetch(a, k + a + kFlight);
        }
      }
#pragma unroll
      for (int i = 0; i < kLines; ++i) *line(kLines * half + i) = sum[i];
    }
    take(st);
  }
  __device__ __forceinline__ void take(f32x16 (&st)[4]) const {   // from LDS
    lds_barrier();
#pragma unroll
    for (int T = 0; T < 4; ++T)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 x = *piece(T, q);
#pragma unroll
        for (int r = 0; r < 4; ++r) st[T][4 * q + r] = x[r];
      }
    lds_barrier();
  }
  template <int Pol>
  __device__ __forceinline__ void store(float* to, const f32x16 (&st)[4]) const {
    lds_barrier();   // (the last chunk's reads of LDS)
#pragma unroll
    for (int T = 0; T < 4; ++T)
#pragma unroll
      for (int q = 0; q < 4; ++q) *piece(T, q) = quad(st[T], q);
    lds_barrier();
    const __amdgpu_buffer_rsrc_t rs = buffer_rsrc(to, kTileBytes);
#pragma unroll
    for (int i = 0; i < 16; ++i) buffer_store16<Pol>(*line(i), rs, threadIdx.x * 16 + 4096 * i);
  }
};

// Transposed operands of a lane, as byte offsets: k's rows 16 u + 8 h + .. in the state's order of
// columns (^ (T << 6) ^ (h << 5)), v's in the wave's columns (^ (h << 5)).
__device__ __forceinline__ uint32_t k_offset(int lane) {
  const int m = lane & 15, c16 = (lane >> 4) & 1, hi = lane >> 5;
  return (4 * hi + (m >> 2)) * kTileRow + (((2 * c16 + (m & 1)) ^ ((m >> 2) << 2) ^ hi) << 4) +
         ((m >> 1) & 1) * 8;
}
__device__ __forceinline__ uint32_t v_offset(int lane, int w) {
  const int m = lane & 15, c16 = (lane >> 4) & 1, hi = lane >> 5;
  return (4 * hi + (m >> 2)) * kTileRow +
         (((4 * w + 2 * c16 + ((m & 3) >> 1)) ^ ((m >> 2) << 2) ^ hi) << 4) + (m & 1) * 8;
}
__device__ __forceinline__ bf16x8 v_operand(const uint8_t* v, uint32_t at, int u) {
  return join(read_tr(v + at + 16 * u * kTileRow), read_tr(v + (at ^ (1 << 5)) + (16 * u + 8) * kTileRow));
}
__device__ __forceinline__ bf16x8 k_operand(const uint8_t* k, uint32_t at, int u, int T) {
  return join(read_tr(k + (at ^ (T << 6)) + 16 * u * kTileRow),
              read_tr(k + (at ^ (T << 6) ^ (1 << 5)) + (16 * u + 8) * kTileRow));
}
// e V of 32 tokens (from token `first`) in accumulator order.
__device__ __forceinline__ f32x16 decayed(const bf16x8 (&v)[2], const float* ek, int first, int hi) {
  f32x16 x;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const f32x4 e = *reinterpret_cast<const f32x4*>(ek + first + 8 * q + 4 * hi);
#pragma unroll
    for (int r = 0; r < 4; ++r) x[4 * q + r] = static_cast<float>(v[q >> 1][4 * (q & 1) + r]) * e[r];
  }
  return x;
}

// A v that is not finite must not meet the outputs ahead of it in a product, whose scores with it
// are zeros: it becomes a zero in `v`, a lane's operands of the 32 tokens from `first`.  Returns the
// first such token of the lane's column, kTokens without one.
__device__ __forceinline__ int take_nonfinite(bf16x8 (&v)[2], int first, int hi) {
  int from = kTokens;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    u32x4 x = __builtin_bit_cast(u32x4, v[u]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t exponent = e & 1 ? 0x7f800000u : 0x7f80u;
      if ((x[e >> 1] & exponent) == exponent) {
        from = min(from, first + 16 * u + 8 * (e >> 2) + 4 * hi + (e & 3));
        x[e >> 1] &= e & 1 ? 0xffffu : 0xffff0000u;
      }
      __builtin_amdgcn_sched_barrier(0);   // (one at a time: the path is rare, registers are not)
    }
    v[u] = __builtin_bit_cast(bf16x8, x);
  }
  return min(from, __shfl_xor(from, 32));
}

// A segment of `rows` rows (whole chunks) from row `bos`, reduced to the state after it, from the
// state at `start` (kept in `kept`) or, if null, from zeros, at `end`; returns, on wave kScalarWave,
// the sum of log decays in units of log 2.
// Rows of k and v go to one half of the tile's LDS while the other is worked on: one barrier a
// chunk.
template <bool Wide>
__device__ __forceinline__ double reduce(const LinearParams& p, SegmentLds& lds, int64_t bos, int rows,
                                         int head, const float* start, float* kept, float* end) {
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hi = lane >> 5;
  const int key_head = head / p.group;
  const int chunks = rows / kTokens;
  u32x4 next_k[4], next_v[4];
  const int srow = tid >> 4;
  const int spiece = tid & 15;
  const uint32_t row_bytes = static_cast<uint32_t>(p.qkv_row) * 2;
  const uint32_t lane_row = srow * row_bytes + spiece * 16;
  const int k_col = (p.num_k_heads + key_head) * kTileRow;
  const int v_col = (2 * p.num_k_heads + head) * kTileRow;
  const uint32_t width = (2 * p.num_k_heads + p.num_v_heads) * kTileRow;
  auto fetch = [&](int c) __attribute__((always_inline)) {   // (past the end zeros)
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t*>(p.qkv + (bos + static_cast<int64_t>(c) * kTokens) * p.qkv_row), 0,
        c < chunks ? (kTokens - 1) * row_bytes + width : 0, 0x00020000);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      next_k[i] = load_piece<Wide>(rs, lane_row + 16 * i * row_bytes, k_col);
      next_v[i] = load_piece<Wide>(rs, lane_row + 16 * i * row_bytes, v_col);
    }
  };
  const uint32_t dst = srow * kTileRow + ((spiece ^ swizzle(srow)) << 4);
  auto put = [&](int c) __attribute__((always_inline)) {
    uint8_t* const at = lds.k + (c & 1) * 2 * kRowsBytes + dst;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      *reinterpret_cast<u32x4*>(at + 16 * i * kTileRow) = next_k[i];
      *reinterpret_cast<u32x4*>(at + kRowsBytes + 16 * i * kTileRow) = next_v[i];
    }
  };
  auto load_decay = [&](int c) __attribute__((always_inline)) {
    const uint32_t step = static_cast<uint32_t>(p.decay_row) * 4;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<float*>(p.log_decay + (bos + static_cast<int64_t>(c) * kTokens) * p.decay_row + head),
        0, c < chunks ? (kTokens - 1) * step + 4 : 0, 0x00020000);
    return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, lane * step, 0, 0));
  };
  const uint32_t kt_at = k_offset(lane);
  const uint32_t vt_at = v_offset(lane, w);
  const Remainder less(lane);
  f32x16 st[4] = {};
  double total = 0.0;
  float next_g = load_decay(0);
  fetch(0);
  const StateTile tile(lds);
  if (start != nullptr) tile.load(start, kept, st);
  if (w == kScalarWave) total += chunk_scalars(lds.scalars[0], next_g, p.scale, lane);
  next_g = load_decay(1);
  put(0);
  fetch(1);
  for (int c = 0; c < chunks; ++c) {
    const ChunkScalars& s = lds.scalars[c & 1];
    const uint8_t* const k_rows = lds.k + (c & 1) * 2 * kRowsBytes;
    const uint8_t* const v_rows = k_rows + kRowsBytes;
    lds_barrier();   // the chunk's rows and scalars are in LDS, the last's read
    const float gamma = s.gamma;
#pragma unroll
    for (int T = 0; T < 4; ++T) st[T] *= gamma;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bf16x8 v[2] = {v_operand(v_rows, vt_at, 2 * i), v_operand(v_rows, vt_at, 2 * i + 1)};
      f32x16 x = decayed(v, s.ek, 32 * i, hi);
      bf16x8 planes[3][2];
#pragma unroll
      for (int n = 0; n < 3; ++n) {
#pragma unroll
        for (int u = 0; u < 2; ++u) planes[n][u] = plane_of(x, u);
        if (n < 2) x = less(x, planes[n][0], planes[n][1]);
      }
      bf16x8 k = k_operand(k_rows, kt_at, 2 * i, 0);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int T = 0; T < 4; ++T) {
          bf16x8 next = k;
          if (T < 3)
            next = k_operand(k_rows, kt_at, 2 * i + u, T + 1);
          else if (u == 0)
            next = k_operand(k_rows, kt_at, 2 * i + 1, 0);
          in_order();
#pragma unroll
          for (int plane = 2; plane >= 0; --plane) st[T] = mfma32(k, planes[plane][u], st[T]);
          in_order();
          k = next;
        }
      if (i == 0) {
        put(c + 1);
        fetch(c + 2);
        if (w == kScalarWave)
          total += chunk_scalars(lds.scalars[(c + 1) & 1], next_g, p.scale, lane);
        next_g = load_decay(c + 2);
      }
    }
  }
  tile.store<kPolPlain>(end, st);
  return total;
}

// One workgroup's walk over `rows` rows from row `bos`: from the state at `start` (zeros if
// null), writing outputs, and the state after the last row to `end` (unless null).
//
// Global memory is reached by buffer loads and stores without branches (past the end a resource
// over 0 bytes or an offset past it: zeros and dropped stores): under a branch the compiler would
// have to wait for every load in flight before it uses any.  Wide: every address is a multiple of
// 4 bytes; else elements move one by one.
// The pool (`end`, and `start` if `joined` is 0) is passed by, the workspace read as the launches
// ahead left it in the caches: `joined` tiles from `start`, with `decays`.
template <bool Wide, bool Gated>
__device__ __forceinline__ void walk(const LinearParams& p, SegmentLds& lds, int64_t bos, int rows,
                                     int head, const float* start, int joined, const float* decays,
                                     float* end) {
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lj = lane & 31;
  const int hi = lane >> 5;
  const int key_head = head / p.group;
  const int chunks = (rows + kTokens - 1) / kTokens;

  // ---- a chunk's rows, in registers on their way to LDS: row 16 i + srow, 16 bytes ----
  struct Staged {
    u32x4 q[4], k[4], v[4];
  } staged;
  const int srow = tid >> 4;
  const int spiece = tid & 15;
  const uint32_t row_bytes = static_cast<uint32_t>(p.qkv_row) * 2;
  uint32_t lane_row = srow * row_bytes + spiece * 16;
  const int q_col = key_head * kTileRow;
  const int k_col = (p.num_k_heads + key_head) * kTileRow;
  const int v_col = (2 * p.num_k_heads + head) * kTileRow;
  const uint32_t width = (2 * p.num_k_heads + p.num_v_heads) * kTileRow;
  // Chunk c's rows of a tensor as a resource: `row` bytes apart, `used` bytes read of each.
  auto chunk_rows = [&](const uint16_t* base, int64_t stride, int c, uint32_t row,
                        uint32_t used) __attribute__((always_inline)) {
    const int live = min(kTokens, rows - c * kTokens);
    return __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t*>(base + (bos + static_cast<int64_t>(c) * kTokens) * stride), 0,
        live > 0 && c >= 0 ? (live - 1) * row + used : 0, 0x00020000);
  };
  // Load i of 12 of a chunk: k and q, then v.  They go out between products: a burst of them would
  // hold the wave until the last is accepted.
  auto source = [&](int c) __attribute__((always_inline)) {
    return chunk_rows(p.qkv, p.qkv_row, c, row_bytes, width);
  };
  auto fetch = [&](__amdgpu_buffer_rsrc_t rs, int c, int i) __attribute__((always_inline)) {
    const int j = i < 8 ? i >> 1 : i - 8;
    const uint32_t at = srow < rows - c * kTokens - 16 * j ? lane_row + 16 * j * row_bytes : 0x7ffff000u;
    if (i >= 8)
      staged.v[j] = load_piece<Wide>(rs, at, v_col);
    else if ((i & 1) == 0)
      staged.k[j] = load_piece<Wide>(rs, at, k_col);
    else
      staged.q[j] = load_piece<Wide>(rs, at, q_col);
  };
  const uint32_t dst = srow * kTileRow + ((spiece ^ swizzle(srow)) << 4);
  auto put = [&](uint8_t* tile, const u32x4 (&x)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<u32x4*>(tile + dst + 16 * i * kTileRow) = x[i];
  };
  auto load_decay = [&](int c) __attribute__((always_inline)) {
    const int live = min(kTokens, rows - c * kTokens);
    const uint32_t step = static_cast<uint32_t>(p.decay_row) * 4;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<float*>(p.log_decay + (bos + static_cast<int64_t>(c) * kTokens) * p.decay_row + head),
        0, live > 0 ? (live - 1) * step + 4 : 0, 0x00020000);
    return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(
                                         rs, lane < live ? lane * step : 0x7ffff000u, 0, 0));
  };

  {
    const __amdgpu_buffer_rsrc_t rs = source(0);
#pragma unroll
    for (int i = 0; i < 12; ++i) fetch(rs, 0, i);
  }
  float next_g = load_decay(0);

  f32x16 st[4] = {};
  const StateTile tile(lds);
  if (start != nullptr) {
    if (joined == 0)
      tile.load(start, nullptr, st);
    else
      tile.load_joined(start, decays, joined, p.num_v_heads, st);
  }
  if (w == kScalarWave) chunk_scalars(lds.scalars[0], next_g, p.scale, lane);
  next_g = load_decay(1);

  // lane addresses of the operands (the parts of the swizzle that depend on the step are XORed in)
  uint32_t a_at = lj * kTileRow + ((hi ^ swizzle(lj)) << 4);       // ^ (step << 5)
  uint32_t kt_at = k_offset(lane);
  const uint32_t vt_at = v_offset(lane, w);
  // P[t][s] of a plane: the quad of s at 16 u + 8 a + 4 hi is half a of row t's 16-byte piece
  // 2 u + hi; the pieces of a row are XORed with t / 2 % 4 (rows of 32 columns) or t % 8
  uint32_t p_upper = lj * 64 + ((hi ^ ((lj >> 1) & 3)) << 4);                // ^ (u << 5)
  uint32_t p_lower = kPlaneUpper + lj * 128 + ((hi ^ (lj & 7)) << 4);        // ^ (u << 5)
  // (between the reads of the last chunk's O and the writes of the next the half behind v is free)
  auto p_plane = [&](int plane) __attribute__((always_inline)) {
    return plane < 2 ? lds.p[plane] : lds.v + kRowsBytes;
  };
  // the wave's 32 x 32 block of P (not the one above the diagonal)
  const int p_rows = w == 0 ? 0 : 1;
  const int p_columns = w == 2 ? 1 : 0;
  // O in LDS: row t's 16-byte pieces XORed with t % 8.  o[tt][4 q + r] is token 32 tt + lj, column
  // 32 w + 8 q + 4 hi + r; a thread finishes columns 8 part + 64 i .. + 7 of rows row and row + 32
  float* const o_rows = reinterpret_cast<float*>(lds.v);
  uint32_t o_put = lj * kDim + ((8 * w + hi) ^ (lj & 7)) * 4;                // ^ (8 q)
  const int row = tid >> 3;
  const int part = tid & 7;
  const uint32_t o_get = row * kDim + ((2 * part) ^ (row & 7)) * 4;   // ^ 4 h, + 64 i
  const uint32_t gate_bytes = static_cast<uint32_t>(p.gate_row) * 2;
  const uint32_t out_bytes = static_cast<uint32_t>(p.num_v_heads) * kTileRow;
  u32x4 gate[2][2];
  auto load_gate = [&](int c) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t rs =
        chunk_rows(p.gate + head * kDim, p.gate_row, c, gate_bytes, kTileRow);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        gate[j][i] = load_piece<Wide>(rs, (row + 32 * j) * gate_bytes + part * 16 + 128 * i, 0);
  };
  auto finish = [&](int c) __attribute__((always_inline)) {   // outputs of chunk c from its O
    const __amdgpu_buffer_rsrc_t rs = chunk_rows(
        p.out + head * kDim, static_cast<int64_t>(p.num_v_heads) * kDim, c, out_bytes, kTileRow);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float y[2][8];
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(o_rows + (o_get ^ (4 * h)) + 64 * i + 32 * j * kDim);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[i][4 * h + e] = x[e];
            if constexpr (Gated) ss = fmaf(x[e], x[e], ss);
          }
        }
      float rstd = 1.0f;
      if constexpr (Gated) {
        ss += dpp<kDppQuadXor1>(ss);
        ss += dpp<kDppQuadXor2>(ss);
        ss += dpp<kDppRowHalfMirror>(ss);
        rstd = fast_rsqrt(ss * (1.0f / kDim) + p.eps);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if constexpr (Gated) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t pair = gate[j][i][e >> 1];
            const float g = __builtin_bit_cast(float, e & 1 ? pair & 0xffff0000u : pair << 16);
            y[i][e] = ((y[i][e] * rstd) * lds.weight[8 * part + 64 * i + e]) * silu(g);
          }
        }
        u32x4 bits;
#pragma unroll
        for (int e = 0; e < 4; ++e) bits[e] = bf16_pair(f32x2{y[i][2 * e], y[i][2 * e + 1]});
        const uint32_t at = (row + 32 * j) * out_bytes + part * 16 + 128 * i;
        if constexpr (Wide) {
          __builtin_amdgcn_raw_buffer_store_b128(bits, rs, at, 0, 0);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            __builtin_amdgcn_raw_buffer_store_b16(static_cast<uint16_t>(bits[e]), rs, at + 4 * e, 0, 0);
            __builtin_amdgcn_raw_buffer_store_b16(static_cast<uint16_t>(bits[e] >> 16), rs, at + 4 * e + 2, 0, 0);
          }
        }
      }
    }
  };

  const Remainder less(lane);
  put(lds.k, staged.k);
  put(lds.q, staged.q);
  for (int c = 0; c < chunks; ++c) {
    const ChunkScalars& s = lds.scalars[c & 1];
    // (opaque here, so that what follows from them is made where it is used, not held in registers
    // over the loop: spilled, it came back with a wait for every load ahead of it, 376 us of 32
    // prompts of 1024 tokens against 360)
    pin(lane_row);
    pin(a_at);
    pin(kt_at);
    pin(p_upper);
    pin(p_lower);
    pin(o_put);
    int here = lane;
    pin(here);
    const int lj = here & 31;
    const int hi = here >> 5;
    lds_barrier();   // k, q and scalars of the chunk are in LDS, O of the last
    f32x16 o[2];
    const __amdgpu_buffer_rsrc_t next_rows = source(c + 1);
    if constexpr (Gated) load_gate(c - 1);
    // ---- O^T = S Q^T: 32 keys at a time, S as three planes; an operand is read again once all
    // of its products are out ----
    bf16x8 q[2][2];
    auto read_q = [&](int T, int u) __attribute__((always_inline)) {
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
        q[u][tt] = *reinterpret_cast<const bf16x8*>(lds.q + 32 * tt * kTileRow +
                                                    (a_at ^ ((2 * T + u) << 5)));
    };
#pragma unroll
    for (int u = 0; u < 2; ++u) read_q(0, u);
#pragma unroll
    for (int T = 0; T < 4; ++T) {
      const bf16x8 high[2] = {plane_of(st[T], 0), plane_of(st[T], 1)};
      f32x16 rest = less(st[T], high[0], high[1]);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        fetch(next_rows, c + 1, 2 * T + u);
        in_order();
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
          o[tt] = mfma32(high[u], q[u][tt], T == 0 && u == 0 ? f32x16{} : o[tt]);
        in_order();
      }
      const bf16x8 middle[2] = {plane_of(rest, 0), plane_of(rest, 1)};
      rest = less(rest, middle[0], middle[1]);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) o[tt] = mfma32(middle[u], q[u][tt], o[tt]);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bf16x8 low = plane_of(rest, u);
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) o[tt] = mfma32(low, q[u][tt], o[tt]);
        in_order();
        if (T < 3) read_q(T + 1, u);
        in_order();
      }
    }
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) o[tt] *= s.eq[32 * tt + lj];
    finish(c - 1);
    lds_barrier();   // O of the last chunk is read
    put(lds.v, staged.v);
    const float gamma = s.gamma;
#pragma unroll
    for (int T = 0; T < 4; ++T) st[T] *= gamma;
    // ---- P ----
    if (w != kScalarWave) {
      f32x16 x = {};
#pragma unroll
      for (int step = 0; step < 8; ++step)
        x = mfma32(*reinterpret_cast<const bf16x8*>(lds.k + 32 * p_columns * kTileRow + (a_at ^ (step << 5))),
                   *reinterpret_cast<const bf16x8*>(lds.q + 32 * p_rows * kTileRow + (a_at ^ (step << 5))),
                   x);
      const float thi = s.hi[32 * p_rows + lj], tlo = s.lo[32 * p_rows + lj];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int first = 8 * q + 4 * hi;
        const f32x4 shi = *reinterpret_cast<const f32x4*>(&s.hi[32 * p_columns + first]);
        const f32x4 slo = *reinterpret_cast<const f32x4*>(&s.lo[32 * p_columns + first]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float d = __builtin_amdgcn_exp2f((thi - shi[r]) + (tlo - slo[r])) * p.scale;
          x[4 * q + r] = p_rows != p_columns || first + r <= lj ? x[4 * q + r] * d : 0.0f;
        }
      }
      auto put_plane = [&](int plane, const bf16x8 (&half)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
          *reinterpret_cast<bf16x8*>(p_plane(plane) + ((p_rows == 0 ? p_upper : p_lower) ^
                                                       ((2 * p_columns + u) << 5))) = half[u];
      };
      const bf16x8 high[2] = {plane_of(x, 0), plane_of(x, 1)};
      put_plane(0, high);
      x = less(x, high[0], high[1]);
      const bf16x8 middle[2] = {plane_of(x, 0), plane_of(x, 1)};
      put_plane(1, middle);
      x = less(x, middle[0], middle[1]);
      const bf16x8 low[2] = {plane_of(x, 0), plane_of(x, 1)};
      put_plane(2, low);
    }
    if (w == kScalarWave) chunk_scalars(lds.scalars[(c + 1) & 1], next_g, p.scale, lane);
    next_g = load_decay(c + 2);
    lds_barrier();   // v and P are in LDS

    auto p_operand = [&](int u, int tt, int plane) __attribute__((always_inline)) {
      return *reinterpret_cast<const bf16x8*>(p_plane(plane) + ((tt == 0 ? p_upper : p_lower) ^ (u << 5)));
    };
    bool nonfinite = false;   // a v of the wave's columns is not finite
    // ---- O^T += V^T P^T and S += K^T (e V): 32 tokens at a time, operands read a product ahead ----
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      bf16x8 v[2] = {v_operand(lds.v, vt_at, 2 * i), v_operand(lds.v, vt_at, 2 * i + 1)};
      f32x16 x = decayed(v, s.ek, 32 * i, hi);
      bf16x8 planes[3][2];
      auto set_planes = [&](int n) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; ++u) planes[n][u] = plane_of(x, u);
      };
      // O's products, between the steps of the split
      auto outputs = [&](int u) __attribute__((always_inline)) {
        bf16x8 ps[2][3];
#pragma unroll
        for (int tt = i; tt < 2; ++tt)
#pragma unroll
          for (int plane = 0; plane < 3; ++plane) ps[tt][plane] = p_operand(2 * i + u, tt, plane);
        in_order();
#pragma unroll
        for (int plane = 2; plane >= 0; --plane)
#pragma unroll
          for (int tt = i; tt < 2; ++tt) o[tt] = mfma32(v[u], ps[tt][plane], o[tt]);
      };
      set_planes(0);
      x = less(x, planes[0][0], planes[0][1]);
      set_planes(1);
      // A v that is not finite, times the zeros of `less`, has made its whole column of x NaN.
      // (4 of the 366 us of 32 prompts of 1024 tokens.)
      if (__builtin_expect(__any(x[0] != x[0]), 0)) {
        int* const from = &lds.nonfinite[32 * w + lj];
        *from = min(nonfinite ? *from : kTokens, take_nonfinite(v, 32 * i, hi));
        nonfinite = true;
      }
      outputs(0);
      x = less(x, planes[1][0], planes[1][1]);
      outputs(1);
      set_planes(2);
      bf16x8 k = k_operand(lds.k, kt_at, 2 * i, 0);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        fetch(next_rows, c + 1, 8 + 2 * i + u);
#pragma unroll
        for (int T = 0; T < 4; ++T) {
          bf16x8 next_k = k;
          if (T < 3)
            next_k = k_operand(lds.k, kt_at, 2 * i + u, T + 1);
          else if (u == 0)
            next_k = k_operand(lds.k, kt_at, 2 * i + 1, 0);
          in_order();
#pragma unroll
          for (int plane = 2; plane >= 0; --plane) st[T] = mfma32(k, planes[plane][u], st[T]);
          in_order();
          k = next_k;
        }
      }
    }
    lds_barrier();   // every read of the chunk's rows and P is done
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(o_rows + (o_put ^ (8 * q)) + 32 * tt * kDim) = quad(o[tt], q);
    if (__builtin_expect(nonfinite, 0)) {   // the outputs behind it are NaN
      lds_order();
      for (int t = lds.nonfinite[32 * w + lj]; t < kTokens; ++t)
        o_rows[t * kDim + (((8 * w + (lj >> 2)) ^ (t & 7)) << 2) + (lj & 3)] = __builtin_nanf("");
    }
    put(lds.k, staged.k);
    put(lds.q, staged.q);
  }
  if (chunks > 0) {
    if constexpr (Gated) load_gate(chunks - 1);
    lds_barrier();
    finish(chunks - 1);
  }

  if (end != nullptr) tile.store<kPolNTSys>(end, st);
}

// A sequence's rows, clamped to those there are.
__device__ __forceinline__ void sequence_rows(const LinearParams& p, int seq, int64_t& bos, int& rows) {
  bos = row_of(p.cu[seq], p.num_tokens);
  rows = static_cast<int>(max(row_of(p.cu[seq + 1], p.num_tokens) - bos, int64_t{0}));
}

// Inclusive sums over the workgroup, and the total; `sums` is free again after a barrier.
__device__ __forceinline__ int inclusive_sum(int mine, int (&sums)[kBlockWaves], int& all) {
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  int sum = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int below = __shfl_up(sum, d);
    if (lane >= d) sum += below;
  }
  if (lane == 63) sums[wave] = sum;
  __syncthreads();
  all = 0;
#pragma unroll
  for (int v = 0; v < kBlockWaves; ++v) {
    if (v < wave) sum += sums[v];
    all += sums[v];
  }
  return sum;
}

// A sequence of `rows` rows is cut into as few segments as `most` rows a segment (a multiple of a
// chunk's) allow, each but the last of the same whole chunks: no workgroup walks longer than the
// sequence needs.
__device__ __forceinline__ int later_of(int rows, int most) {
  return rows > 0 ? static_cast<int>(static_cast<uint32_t>(rows - 1) / static_cast<uint32_t>(most)) : 0;
}
__device__ __forceinline__ int segment_rows(int rows, int later) {
  const uint32_t count = static_cast<uint32_t>(later) + 1;
  return static_cast<int>((rows + count - 1) / count + kTokens - 1) / kTokens * kTokens;
}

// Later segments (all but the first) of the sequences are numbered in order: finds the j-th, i.e.
// its sequence, which of the sequence's later segments it is, and how many that has.  False past
// the last.  By the whole workgroup.
__device__ bool find_segment(const LinearParams& p, SearchLds& lds, int num_sequences, int most,
                             int j, int& seq, int& index, int& count) {
  const int tid = threadIdx.x;
  int base = 0;
  for (int first = 0; first < num_sequences; first += kBlock) {
    const int n = first + tid;
    int mine = 0;
    if (n < num_sequences) {
      int64_t bos;
      int rows;
      sequence_rows(p, n, bos, rows);
      mine = later_of(rows, most);
    }
    int all;
    const int sum = inclusive_sum(mine, lds.wave_sums, all);
    const int at = j - base;
    if (at < sum && at >= sum - mine) {
      lds.found[0] = n;
      lds.found[1] = at - (sum - mine);
      lds.found[2] = mine;
    }
    __syncthreads();
    if (at < all) {
      seq = __builtin_amdgcn_readfirstlane(lds.found[0]);
      index = __builtin_amdgcn_readfirstlane(lds.found[1]);
      count = __builtin_amdgcn_readfirstlane(lds.found[2]);
      return true;
    }
    base += all;
  }
  return false;
}

constexpr int kAhead = 16;

struct Segments {
  int num_sequences;
  int most;         // tokens of a segment, at most
  int later;        // at most this many later segments
  // Each segment sums the states ahead of it by itself, without the second launch: up to kAhead of
  // them, or twice that among several sequences, most of which have far fewer (us, with the second launch and
  // without: 13 prompts of 1 to 3000 tokens 140 / 131, 16 of 64 to 1024 107 / 100, one of 4096 80 / 78;
  // one of 8192 with 8 heads, 31 ahead of the last, 56 / 63, of 16384 85 / 127).  Among several one that
  // has nearly all of the tokens loses by it, as one alone would (8192 and an empty one 56 / 62).
  bool direct;
  // per (later segment, head): the state after the segment ahead of it, for a sequence's first one
  // from the state that the sequence starts from, for the others from zeros (behind the join: the
  // state that the segment starts from)
  float* tiles;
  float* firsts;    // in the places of the first later segments: the state the sequence starts
                    // from, as its last segment replaces it in the pool
  float* decays;    // per (later segment, head): the decay over the segment ahead of it
};

// Workgroups go to the 8 XCDs round-robin by id; the v-heads of one k-head read the same q and k,
// so they are given ids on one XCD.  False past the last unit.
__device__ __forceinline__ bool unit_of(const LinearParams& p, int items, int& item, int& head) {
  const int xcd = blockIdx.x & 7;
  const int rank = blockIdx.x >> 3;
  const int unit = (rank / p.group) * 8 + xcd;
  if (unit >= items * p.num_k_heads) return false;
  item = unit / p.num_k_heads;
  head = (unit - item * p.num_k_heads) * p.group + rank % p.group;
  return true;
}

__device__ __forceinline__ int64_t tile_of(const LinearParams& p, int segment, int head) {
  return static_cast<int64_t>(segment) * p.num_v_heads + head;
}

// The first launch: item j reduces the segment ahead of later segment j to the state after it and
// its decay.
template <bool Wide>
__global__ __launch_bounds__(kBlock) __attribute__((amdgpu_waves_per_eu(2, 2)))
void linear_reduce_kernel(const LinearParams p, const Segments g) {
  __shared__ SegmentLds lds;
  __shared__ SearchLds search;
  int item, head, seq, index, count;
  if (!unit_of(p, g.later, item, head) ||
      !find_segment(p, search, g.num_sequences, g.most, item, seq, index, count))
    return;
  int64_t bos;
  int rows;
  sequence_rows(p, seq, bos, rows);
  const int64_t at = tile_of(p, item, head);
  const int each = segment_rows(rows, count);
  const int slot = p.indices[seq];
  const float* start = index == 0 && live_slot(slot, p.num_slots) && p.has_initial[seq] != 0
                           ? p.state + slot * p.state_slot + head * kTileFloats
                           : nullptr;
  const double total = reduce<Wide>(p, lds, bos + index * each, each, head, start,
                                    g.firsts + at * kTileFloats, g.tiles + at * kTileFloats);
  if (threadIdx.x == 64 * kScalarWave) g.decays[at] = __builtin_amdgcn_exp2f(static_cast<float>(total));
}

// The second, unless direct: the state at every later segment's start, along each sequence.  A
// workgroup takes a sixteenth of one head's tile through every fourth of the sequences of several
// segments: they wait for memory side by side.
constexpr int kJoinParts = kTileFloats / 4 / kBlock;
constexpr int kJoinSequences = 4;
__global__ __launch_bounds__(kBlock) void linear_join_kernel(const LinearParams p, const Segments g) {
  __shared__ int counts[kBlock], bases[kBlock];   // of the sequences of several segments
  __shared__ int sums[2][kBlockWaves];
  const int tid = threadIdx.x;
  const int part = blockIdx.x % kJoinParts;
  const int head = blockIdx.x / kJoinParts;
  const int64_t at = (part * kBlock + tid) * 4;
  const int64_t step = p.num_v_heads * kTileFloats;
  int base = 0;
  for (int first = 0; first < g.num_sequences; first += kBlock) {
    // later segments of each of kBlock sequences, and of those ahead of it
    const int n = first + tid;
    int mine = 0;
    if (n < g.num_sequences) {
      int64_t bos;
      int rows;
      sequence_rows(p, n, bos, rows);
      mine = later_of(rows, g.most);
    }
    int all, several;
    const int sum = inclusive_sum(mine, sums[0], all);
    const int place = inclusive_sum(mine > 0 ? 1 : 0, sums[1], several) - 1;
    if (mine > 0) {
      counts[place] = mine;
      bases[place] = base + sum - mine;
    }
    __syncthreads();
    base += all;
    for (int i = blockIdx.y; i < several; i += gridDim.y) {
      const int j = __builtin_amdgcn_readfirstlane(bases[i]);
      const int count = min(__builtin_amdgcn_readfirstlane(counts[i]), g.later - j);
      if (count <= 1) continue;
      f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
      float* tile = g.tiles + tile_of(p, j, head) * kTileFloats + at;
      const float* decay = g.decays + tile_of(p, j, head);
      constexpr int kFlight = 8;   // updates and decays in flight
      f32x4 update[kFlight];
      float by[kFlight];
      auto load = [&](int a, int k) __attribute__((always_inline)) {   // (past the last, that again)
        const int64_t from = min(k, count - 1);
        update[a] = *reinterpret_cast<const f32x4*>(tile + from * step);
        by[a] = from == 0 ? 0.0f : decay[from * p.num_v_heads];
      };
#pragma unroll
      for (int a = 0; a < kFlight; ++a) load(a, a);
      for (int k = 0; k < count; k += kFlight) {
#pragma unroll
        for (int a = 0; a < kFlight; ++a) {
          s = s * by[a] + update[a];
          load(a, k + a + kFlight);
          if (k + a > 0 && k + a < count) *reinterpret_cast<f32x4*>(tile + (k + a) * step) = s;
        }
      }
    }
    __syncthreads();
  }
}

// The third: every segment's outputs, and the sequences' last states.  Item j < later is later
// segment j; item later + j the first segment of its sequence, if j is the sequence's first later
// one; item 2 later + n sequence n, if it is a single segment (the shortest last).
// Two workgroups a CU; one where elements are loaded one by one, whose 96 loads in flight take a
// register each: with the registers of two, 49 of them spilled (32 prompts of 1024 tokens with a norm
// 926 us against 797, without 735 against 682).
template <bool Wide, bool Gated>
__global__ __launch_bounds__(kBlock) __attribute__((amdgpu_waves_per_eu(Wide ? 2 : 1, Wide ? 2 : 1)))
void linear_walk_kernel(const LinearParams p, const Segments g) {
  __shared__ SegmentLds lds;
  __shared__ SearchLds search;
  int item, head, seq, index = -1, count = 0;
  if (!unit_of(p, 2 * g.later + g.num_sequences, item, head)) return;
  const bool single = item >= 2 * g.later;
  if (single) {
    seq = item - 2 * g.later;
  } else {
    const bool is_first = item >= g.later;
    if (is_first) item -= g.later;
    if (!find_segment(p, search, g.num_sequences, g.most, item, seq, index, count) ||
        (is_first && index != 0))
      return;
    if (is_first) index = -1;
  }
  int64_t bos;
  int rows;
  sequence_rows(p, seq, bos, rows);
  if (single && later_of(rows, g.most) != 0) return;
  if (p.gate != nullptr && threadIdx.x < kDim)
    lds.weight[threadIdx.x] = load_param(p.norm_weight, threadIdx.x, p.weight_bf16);
  const int each = segment_rows(rows, count);
  const int done = (index + 1) * each;
  const int slot = p.indices[seq];
  const bool live = live_slot(slot, p.num_slots);
  float* const home = p.state + static_cast<int64_t>(live ? slot : 0) * p.state_slot + head * kTileFloats;
  const bool initial = live && p.has_initial[seq] != 0;
  // later segments: the tile that the join left, or all of the sequence's up to theirs
  const int joined = single ? 0 : index < 0 || !g.direct ? 1 : index + 1;
  const int64_t at = tile_of(p, item - (index < 0 ? 0 : joined - 1), head);
  const float* start = g.tiles + at * kTileFloats;
  if (single) start = initial ? home : nullptr;
  if (!single && index < 0) start = initial ? g.firsts + at * kTileFloats : nullptr;
  walk<Wide, Gated>(p, lds, bos + done, min(rows - done, each), head, start, joined, g.decays + at,
                    live && index + 1 == count ? home : nullptr);
}

// A segment's tokens, at most, in whole chunks: the share of a workgroup where 512 run at once (two
// a CU), and at least 256, as a segment is walked twice.  Rounded to a power of two the share leaves
// CUs idle (32 heads, us: 5000 tokens 105 / 88, 9000 173 / 147, 20000 375 / 301, 16 prompts of 64 to
// 1024 119 / 100).
// One prompt is cut finer, to 128 tokens, while a CU gets one workgroup and a segment has 16 ahead
// of it (us: 512 tokens of 32 heads 42 / 32, 1024 46 / 37; to 128 in any case 2048 55 against 51, 8192 of
// 8 heads 62 against 56, though 4096 of those 43 against 53).  Several of 512 tokens in all are left whole: most likely none is long, and a
// reduction in vain takes 5 us of their 20.
int64_t segment_tokens(int64_t num_tokens, int32_t num_sequences, int32_t num_v_heads) {
  if (num_sequences > 1 && num_tokens <= 512) return 512;
  const auto share = [](int64_t tokens, int64_t parts) {
    const int64_t each = (tokens + parts - 1) / parts;
    return (each + kTokens - 1) / kTokens * kTokens;
  };
  int64_t least = 256;
  if (num_sequences == 1)
    least = std::clamp<int64_t>(
        std::max(share(num_tokens * num_v_heads, 256), share(num_tokens, kAhead + 1)), 128, least);
  return std::clamp<int64_t>(share(num_tokens * num_v_heads, 512), least, 1 << 30);
}

// Sequences of more than a segment have at most this many later ones.
int64_t later_segments(int64_t num_tokens, int32_t num_sequences, int32_t num_v_heads) {
  return num_tokens > 0 ? (num_tokens - 1) / segment_tokens(num_tokens, num_sequences, num_v_heads) : 0;
}

template <bool Wide>
void launch_segments(const LinearParams& p, const Segments& g, uint32_t reduced, uint32_t walked,
                     hipStream_t s) {
  if (g.later > 0)
    hipLaunchKernelGGL((linear_reduce_kernel<Wide>), dim3(reduced), dim3(kBlock), 0, s, p, g);
  if (g.later > 0 && !g.direct) {
    const dim3 parts(p.num_v_heads * kJoinParts,
                     std::min({g.num_sequences, g.later, kJoinSequences}));
    hipLaunchKernelGGL(linear_join_kernel, parts, dim3(kBlock), 0, s, p, g);
  }
  const auto walk = p.gate != nullptr ? linear_walk_kernel<Wide, true> : linear_walk_kernel<Wide, false>;
  hipLaunchKernelGGL(walk, dim3(walked), dim3(kBlock), 0, s, p, g);
}

void launch_linear_prefill(const LinearParams& p, const Segments& g, uint32_t reduced,
                           uint32_t walked, hipStream_t s) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(p.qkv) | reinterpret_cast<uintptr_t>(p.gate) |
                         reinterpret_cast<uintptr_t>(p.out) | (p.qkv_row * 2) | (p.gate_row * 2);
  if ((bits & 3) == 0)
    launch_segments<true>(p, g, reduced, walked, s);
  else
    launch_segments<false>(p, g, reduced, walked, s);
}

}  // namespace
}  // namespace ld

extern "C" int64_t ld_linear_prefill_workspace_bytes(int64_t num_tokens, int32_t num_sequences,
                                                     int32_t num_v_heads) {
  if (num_tokens < 0 || num_tokens > 0x7fffffff || num_sequences <= 0 || num_v_heads <= 0) return 0;
  return ld::later_segments(num_tokens, num_sequences, num_v_heads) * num_v_heads *
         static_cast<int64_t>((2 * ld::kTileFloats + 4) * sizeof(float));
}

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
  if (a.num_tokens <= 1) p.qkv_row = p.gate_row = p.decay_row = 0;   // (the distance to no other row)
  if (p.qkv_row < 0 || p.qkv_row > kMaxRow || p.gate_row < 0 || p.gate_row > kMaxRow ||
      p.decay_row < 0 || p.decay_row > kMaxRow || a.num_v_heads > kMaxRow / kDim)
    return fail(LD_ERR_INVALID_ARGUMENT, "qkv, log_decay, gate and out rows must be at most 2^23 elements apart");
  if (a.num_tokens > 0x7fffffff) return fail(LD_ERR_INVALID_ARGUMENT, "too many tokens");
  p.indices = a.slots;
  p.cu = a.cu_seqlens;
  p.has_initial = a.has_initial;
  const int64_t later = later_segments(a.num_tokens, a.num_sequences, a.num_v_heads);
  if (later > 0 && (!aligned16(a.workspace) || a.workspace == nullptr ||
                    a.workspace_bytes < ld_linear_prefill_workspace_bytes(
                                            a.num_tokens, a.num_sequences, a.num_v_heads)))
    return fail(LD_ERR_INVALID_ARGUMENT, "ld_linear_prefill: workspace missing or too small");
  // grids in multiples of 8 XCDs times the group; a grid's threads stay below 2^32
  auto blocks_of = [&](int64_t items) {
    return (items * a.num_k_heads + 7) / 8 * 8 * p.group;
  };
  if (blocks_of(2 * later + a.num_sequences) > 0x7fffff || a.num_v_heads > 0x7fffff / kJoinParts)
    return fail(LD_ERR_INVALID_ARGUMENT, "too many (sequence, head) tiles");
  Segments g{};
  g.num_sequences = a.num_sequences;
  g.most = static_cast<int>(segment_tokens(a.num_tokens, a.num_sequences, a.num_v_heads));
  g.later = static_cast<int>(later);
  g.direct = later <= (a.num_sequences == 1 ? kAhead : 2 * kAhead);
  g.tiles = static_cast<float*>(a.workspace);
  g.firsts = g.tiles + later * a.num_v_heads * kTileFloats;
  g.decays = g.firsts + later * a.num_v_heads * kTileFloats;
  launch_linear_prefill(p, g, static_cast<uint32_t>(blocks_of(later)),
                        static_cast<uint32_t>(blocks_of(2 * later + a.num_sequences)),
                        static_cast<hipStream_t>(stream));
  return check_launch("ld_linear_prefill");
}
