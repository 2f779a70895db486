// Prefill of linear attention with a decay for each head, for gfx950:
//   S <- exp(g) S + v k^T ;  o = scale * S q ;  out = o, or its gated RMSNorm
// in chunks of 64 tokens.  With c_t the sum of g over the chunk's tokens up to t:
//   o_t = scale (e^(c_t) S q_t + sum over s <= t of e^(c_t - c_s) (k_s . q_t) v_s)
//   S'  = e^(c_63) S + sum over s of k_s (e^(c_63 - c_s) v_s)^T
//
// A workgroup of eight waves walks the chunks of one (sequence, v-head).  Wave w owns state rows
// v = 16 w .. 16 w + 15 as S^T in the accumulators of v_mfma_f32_16x16x32_bf16: for lane l,
// li = l % 16 and lg = l / 16, an accumulator holds rows 4 lg + r, r < 4, of column li, an operand
// A[i = li][k = 8 lg + e] or B[k = 8 lg + e][j = li], e < 8.  The summation index may be assigned
// to (step, lg, e) freely as long as both operands agree, so two accumulators, split into bf16
// planes, are directly the operand of a step of the next product:
//   keys     row 4 lg + r of accumulators (n, a) is k = 32 n + 8 lg + 4 a + r, so that step n takes
//            16 consecutive bytes of a q row
//   tokens   step i takes token 32 i + 16 (e / 4) + 4 lg + e % 4
//   O = Q S^T          S as two planes
//   P = (K Q^T) . D    16 x 16 blocks over the waves, two planes, exchanged through LDS
//   O = diag(e^c) O + P V
//   S' = e^(c_63) S + K^T (e^(c_63 - c) V)    e V as three planes
// and O crosses LDS in fp32 to whole rows, for the norm and 16-byte stores.  The transposed
// operands come by ds_read_b64_tr_b16.
//
// Decays come from differences of 64-bit prefix sums: their error over thousands of tokens would
// be the state's.  Roundings to fewer than 32 bits, each of operands of the bf16 matrix cores
// whose sums are fp32: the state's update takes its operand exactly (three planes hold fp32's 24
// bits), what only reaches bf16 outputs takes two planes (relative error 2^-17 a term, against
// 2^-9 of the output's own rounding).
//
// A sequence longer than a segment is cut into segments, since the recurrence over them is
// associative: one launch runs every first segment and reduces the middle ones to their update
// and decay, a second joins these along each sequence, a third runs the later segments from the
// states the second left.
#include "linear_common.h"
#include "matrix_common.h"

namespace ld {
namespace {

constexpr int kBlockWaves = 8;
constexpr int kBlock = 64 * kBlockWaves;
constexpr int kTokens = 64;                     // tokens per chunk
constexpr int kRowsBytes = kTokens * kTileRow;  // q, k or v of a chunk
constexpr int64_t kTileFloats = kDim * kDim;

// Per-token scalars of a chunk: c in units of log 2 as a sum of two floats, scale * e^c and
// e^(c_63 - c); and e^(c_63).
struct alignas(16) ChunkScalars {
  float hi[kTokens], lo[kTokens], eq[kTokens], ek[kTokens];
  float gamma;
};

struct SegmentLds {
  // k, then q (behind them, in their place, the chunk's O in fp32); v; the two planes of P
  alignas(16) uint8_t k[kRowsBytes];
  alignas(16) uint8_t q[kRowsBytes];
  alignas(16) uint8_t v[kRowsBytes];
  alignas(16) uint8_t p[2][kTokens * kTokens * 2];
  ChunkScalars scalars[2];
  alignas(16) float weight[kDim];
};
struct SearchLds {
  int wave_sums[kBlockWaves];
  int found[3];
};
static_assert(2 * (sizeof(SegmentLds) + sizeof(SearchLds)) <= 160 * 1024, "two workgroups a CU");
static_assert(2 * kRowsBytes == kTokens * kDim * 4, "O takes the place of k and q");

// x = sum of N bf16 planes (exactly, for three), eight values as an operand each.
template <int N>
struct Planes {
  u32x4 w[N];
  __device__ __forceinline__ explicit Planes(float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[i][j] = bf16_pair(f32x2{x[2 * j], x[2 * j + 1]});
        if (i + 1 < N) {
          x[2 * j] -= __builtin_bit_cast(float, w[i][j] << 16);
          x[2 * j + 1] -= __builtin_bit_cast(float, w[i][j] & 0xffff0000u);
        }
      }
    }
  }
  __device__ __forceinline__ bf16x8 operator[](int i) const {
    return __builtin_bit_cast(bf16x8, w[i]);
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

__device__ __forceinline__ bf16x8 join(bf16x4 a, bf16x4 b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// One workgroup's walk over `rows` rows from row `bos`: from the state at `start` (zeros if
// null), writing outputs if Out, and the state after the last row to `end` (unless null).  Without
// Out the state is the segment's update; either way returns, on wave 0, the sum of log decays in
// units of log 2.
template <bool Out>
__device__ __forceinline__ double walk(const LinearParams& p, SegmentLds& lds, int64_t bos, int rows,
                                       int head, const float* start, float* end) {
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 15;
  const int lg = lane >> 4;
  const int key_head = head / p.group;
  const int chunks = (rows + kTokens - 1) / kTokens;

  // ---- a chunk's rows, in registers on their way to LDS: row 32 i + srow, 16 bytes ----
  struct Staged {
    u32x4 q[2], k[2], v[2];
  } staged;
  const int srow = tid >> 4;
  const int spiece = tid & 15;
  const uint16_t* const columns = p.qkv + 8 * spiece + key_head * kDim;
  const int k_col = p.num_k_heads * kDim;
  const int v_col = (2 * p.num_k_heads + head - key_head) * kDim;
  auto fetch = [&](int c) __attribute__((always_inline)) {
    const int live = min(kTokens, rows - c * kTokens);
    const int64_t first = bos + static_cast<int64_t>(c) * kTokens;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint16_t* const row = columns + (first + min(srow + 32 * i, live - 1)) * p.qkv_row;
      __builtin_memcpy(&staged.k[i], row + k_col, 16);
      __builtin_memcpy(&staged.v[i], row + v_col, 16);
      if constexpr (Out) __builtin_memcpy(&staged.q[i], row, 16);
    }
    if (live < kTokens) {   // rows past the end are zeros
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (srow + 32 * i >= live) {
          staged.k[i] = staged.v[i] = u32x4{0u, 0u, 0u, 0u};
          if constexpr (Out) staged.q[i] = u32x4{0u, 0u, 0u, 0u};
        }
    }
  };
  const uint32_t dst = srow * kTileRow + ((spiece ^ swizzle(srow)) << 4);
  auto put = [&](uint8_t* tile, const u32x4 (&x)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) *reinterpret_cast<u32x4*>(tile + dst + 32 * i * kTileRow) = x[i];
  };
  auto load_decay = [&](int c) __attribute__((always_inline)) {
    const int t = c * kTokens + lane;
    return t < rows ? p.log_decay[(bos + t) * p.decay_row + head] : 0.0f;
  };

  double total = 0.0;
  if (chunks > 0) {
    fetch(0);
    if (w == 0) total += chunk_scalars(lds.scalars[0], load_decay(0), p.scale, lane);
  }

  // st[n][a][r] = S[16 w + li][32 n + 8 lg + 4 a + r]
  f32x4 st[4][2];
  const int tile_at = (16 * w + li) * kDim + 8 * lg;
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      st[n][a] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (start != nullptr)
        st[n][a] = *reinterpret_cast<const f32x4*>(start + tile_at + 32 * n + 4 * a);
    }

  // lane addresses of the operands (the parts of the swizzle that depend on the step are XORed in)
  uint32_t a_at = li * kTileRow + ((lg ^ swizzle(li)) << 4);       // ^ (step << 6)
  const int quad = li >> 2;
  const uint32_t tr_row = (4 * lg + quad) * kTileRow;
  // transposed k: rows 32 s + 16 h + .., columns 32 n + 8 (i / 4) + 4 a + i % 4   ^ (n << 6)
  uint32_t kt_at = tr_row + (((li & 3) ^ (quad << 2) ^ lg) << 4);
  // transposed v: rows 32 s + 16 h + .., the wave's columns
  const uint32_t vt_at = tr_row + (((2 * w + ((li & 3) >> 1)) ^ (quad << 2) ^ lg) << 4) + (li & 1) * 8;
  // P[t][s] of a plane: the quad of s at 32 i + 16 a + 4 lg is half a of row t's 16-byte piece
  // 4 i + lg, the pieces of a row XORed with t % 8
  uint32_t p_at = li * (2 * kTokens) + ((lg ^ (li & 7)) << 4);     // ^ (i << 6)
  // the wave's part of P: rows of strip w / 2; columns 16 w % 2 of the first two, 32 (w % 2) and
  // 16 more of the others
  const int strip = w >> 1;
  // O in fp32: row t's 16-byte pieces XORed with 4 (t / 4 % 4)
  const int row = tid >> 3;
  const int part = tid & 7;
  const int o_at = row * kDim + (((2 * part) ^ (((row >> 2) & 3) << 2)) << 2);

  if (chunks > 0) {
    put(lds.k, staged.k);
    put(lds.v, staged.v);
    if constexpr (Out) put(lds.q, staged.q);
  }
  for (int c = 0; c < chunks; ++c) {
    const ChunkScalars& s = lds.scalars[c & 1];
    const bool more = c + 1 < chunks;
    float next_g = 0.0f;
    // (opaque here, so that their XORed forms are made where they are used, not held in registers
    // over the loop)
    pin(a_at);
    pin(kt_at);
    pin(p_at);
    lds_barrier();   // the chunk's rows and scalars are in LDS
    if (more) fetch(c + 1);
    if (more && w == 0) next_g = load_decay(c + 1);
    f32x4 o[4];
    const float gamma = s.gamma;
    if constexpr (Out) {
      // ---- P ----
      bf16x8 qf[4];
#pragma unroll
      for (int step = 0; step < 4; ++step)
        qf[step] = *reinterpret_cast<const bf16x8*>(lds.q + 16 * strip * kTileRow +
                                                    (a_at ^ (step << 6)));
      const float thi = s.hi[16 * strip + li], tlo = s.lo[16 * strip + li];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (i == 1 && strip < 2) break;
        const int j = strip < 2 ? w & 1 : 2 * (w & 1) + i;
        f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
        if (j <= strip) {
#pragma unroll
          for (int step = 0; step < 4; ++step)
            x = mfma16(*reinterpret_cast<const bf16x8*>(lds.k + 16 * j * kTileRow +
                                                        (a_at ^ (step << 6))),
                       qf[step], x);
          const f32x4 shi = *reinterpret_cast<const f32x4*>(&s.hi[16 * j + 4 * lg]);
          const f32x4 slo = *reinterpret_cast<const f32x4*>(&s.lo[16 * j + 4 * lg]);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float d = __builtin_amdgcn_exp2f((thi - shi[r]) + (tlo - slo[r])) * p.scale;
            x[r] = j < strip || 4 * lg + r <= li ? x[r] * d : 0.0f;
          }
        }
        uint8_t* const at = lds.p[0] + (16 * strip + li) * (2 * kTokens) +
                            (((4 * (j >> 1) + lg) ^ (li & 7)) << 4) + (j & 1) * 8;
#pragma unroll
        for (int plane = 0; plane < 2; ++plane) {
          const uint2 bits = {bf16_pair(f32x2{x[0], x[1]}), bf16_pair(f32x2{x[2], x[3]})};
          *reinterpret_cast<uint2*>(at + plane * sizeof(lds.p[0])) = bits;
          x[0] -= __builtin_bit_cast(float, bits.x << 16);
          x[1] -= __builtin_bit_cast(float, bits.x & 0xffff0000u);
          x[2] -= __builtin_bit_cast(float, bits.y << 16);
          x[3] -= __builtin_bit_cast(float, bits.y & 0xffff0000u);
        }
      }
      // ---- O = Q S^T ----
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) o[tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = st[n][e >> 2][e & 3];
        const Planes<2> split(x);
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          const bf16x8 a = *reinterpret_cast<const bf16x8*>(lds.q + 16 * tt * kTileRow +
                                                            (a_at ^ (n << 6)));
          o[tt] = mfma16(a, split[1], o[tt]);
          o[tt] = mfma16(a, split[0], o[tt]);
        }
      }
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        const f32x4 eq = *reinterpret_cast<const f32x4*>(&s.eq[16 * tt + 4 * lg]);
        o[tt] *= eq;
      }
    }
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int a = 0; a < 2; ++a) st[n][a] *= gamma;
    if constexpr (Out) lds_barrier();   // P is in LDS
    if (more && w == 0)
      total += chunk_scalars(lds.scalars[(c + 1) & 1], next_g, p.scale, lane);

    // ---- O += P V and S += K^T (e V), 32 tokens a step ----
    u32x4 gate[2];
    const int64_t token = bos + static_cast<int64_t>(c) * kTokens + row;
    const bool stored = c * kTokens + row < rows;
    if constexpr (Out) {
      if (p.gate != nullptr && stored) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          __builtin_memcpy(&gate[i], p.gate + token * p.gate_row + head * kDim + 8 * part + 64 * i, 16);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bf16x8 v = join(read_tr(lds.v + vt_at + 32 * i * kTileRow),
                            read_tr(lds.v + vt_at + (32 * i + 16) * kTileRow));
      if constexpr (Out) {
#pragma unroll
        for (int tt = 2 * i; tt < 4; ++tt)
#pragma unroll
          for (int plane = 1; plane >= 0; --plane)
            o[tt] = mfma16(*reinterpret_cast<const bf16x8*>(
                               lds.p[plane] + 16 * tt * (2 * kTokens) + (p_at ^ (i << 6))),
                           v, o[tt]);
      }
      float x[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 ek = *reinterpret_cast<const f32x4*>(&s.ek[32 * i + 16 * h + 4 * lg]);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[4 * h + r] = static_cast<float>(v[4 * h + r]) * ek[r];
      }
      const Planes<3> split(x);
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const uint8_t* const at = lds.k + (kt_at ^ (n << 6)) + 8 * a;
          const bf16x8 k = join(read_tr(at + 32 * i * kTileRow), read_tr(at + (32 * i + 16) * kTileRow));
#pragma unroll
          for (int plane = 2; plane >= 0; --plane) st[n][a] = mfma16(k, split[plane], st[n][a]);
        }
    }
    lds_barrier();   // every read of the chunk's rows and P is done
    if constexpr (Out) {
      float* const o_rows = reinterpret_cast<float*>(lds.k);
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          o_rows[(16 * tt + 4 * lg + r) * kDim + (((4 * w + (li >> 2)) ^ (lg << 2)) << 2) + (li & 3)] =
              o[tt][r];
      if (more) put(lds.v, staged.v);
      lds_barrier();   // O is in LDS
      // ---- an eighth of one row a thread: columns 8 part + 64 i .. + 7 ----
      float y[2][8];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(
              o_rows + o_at + 64 * i + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) y[i][4 * h + e] = x[e];
        }
      if (p.gate != nullptr) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) ss = fmaf(y[i][e], y[i][e], ss);
        ss += dpp<kDppQuadXor1>(ss);
        ss += dpp<kDppQuadXor2>(ss);
        ss += dpp<kDppRowHalfMirror>(ss);
        const float rstd = fast_rsqrt(ss * (1.0f / kDim) + p.eps);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t pair = gate[i][e >> 1];
            const float g = __builtin_bit_cast(float, e & 1 ? pair & 0xffff0000u : pair << 16);
            y[i][e] = ((y[i][e] * rstd) * lds.weight[8 * part + 64 * i + e]) * silu(g);
          }
      }
      if (stored) {
        uint16_t* const to = p.out + (token * p.num_v_heads + head) * kDim + 8 * part;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          u32x4 bits;
#pragma unroll
          for (int e = 0; e < 4; ++e) bits[e] = bf16_pair(f32x2{y[i][2 * e], y[i][2 * e + 1]});
          __builtin_memcpy(to + 64 * i, &bits, 16);
        }
      }
      lds_barrier();   // O is read
      if (more) {
        put(lds.k, staged.k);
        put(lds.q, staged.q);
      }
    } else if (more) {
      put(lds.k, staged.k);
      put(lds.v, staged.v);
    }
  }

  if (end != nullptr) {
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int a = 0; a < 2; ++a)
        *reinterpret_cast<f32x4*>(end + tile_at + 32 * n + 4 * a) = st[n][a];
  }
  return total;
}

// A sequence's rows, clamped to those there are.
__device__ __forceinline__ void sequence_rows(const LinearParams& p, int seq, int64_t& bos, int& rows) {
  bos = row_of(p.cu[seq], p.num_tokens);
  rows = static_cast<int>(max(row_of(p.cu[seq + 1], p.num_tokens) - bos, int64_t{0}));
}

// Later segments (all but the first) of the sequences are numbered in order: finds the j-th, i.e.
// its sequence, which of the sequence's later segments it is, and how many that has.  False past
// the last.  By the whole workgroup.
__device__ bool find_segment(const LinearParams& p, SearchLds& lds, int num_sequences, int shift,
                             int j, int& seq, int& index, int& count) {
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  int base = 0;
  for (int first = 0; first < num_sequences; first += kBlock) {
    const int n = first + tid;
    int mine = 0;
    if (n < num_sequences) {
      int64_t bos;
      int rows;
      sequence_rows(p, n, bos, rows);
      mine = rows > 0 ? (rows - 1) >> shift : 0;
    }
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int below = __shfl_up(sum, d);
      if (lane >= d) sum += below;
    }
    if (lane == 63) lds.wave_sums[tid >> 6] = sum;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int v = 0; v < kBlockWaves; ++v) {
      if (v < tid >> 6) sum += lds.wave_sums[v];
      all += lds.wave_sums[v];
    }
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

struct Segments {
  int num_sequences;
  int shift;        // log2 of a segment's tokens
  int later;        // at most this many later segments
  float* tiles;     // per (later segment, head): the state it starts from, S or (before the
                    // second launch) the update of the segment ahead of it
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

__device__ __forceinline__ void load_weight(const LinearParams& p, SegmentLds& lds) {
  if (p.gate != nullptr && threadIdx.x < kDim)
    lds.weight[threadIdx.x] = load_param(p.norm_weight, threadIdx.x, p.weight_bf16);
}

// The first launch.  Item j < later is later segment j's predecessor: the sequence's first
// segment, walked from its state, or a middle one, reduced to its update; item later + n is
// sequence n if it is a single segment.
__global__ __launch_bounds__(kBlock) __attribute__((amdgpu_waves_per_eu(4, 4)))
void linear_first_kernel(const LinearParams p, const Segments g) {
  __shared__ SegmentLds lds;
  __shared__ SearchLds search;
  int item, head;
  if (!unit_of(p, g.later + g.num_sequences, item, head)) return;
  int seq = item - g.later, index = 0, count = 0;
  const bool whole = item >= g.later;
  if (!whole && !find_segment(p, search, g.num_sequences, g.shift, item, seq, index, count)) return;
  int64_t bos;
  int rows;
  sequence_rows(p, seq, bos, rows);
  if (whole && rows > 0 && (rows - 1) >> g.shift != 0) return;
  load_weight(p, lds);
  float* const tile = whole ? nullptr : g.tiles + (static_cast<int64_t>(item) * p.num_v_heads + head) * kTileFloats;
  if (index > 0) {
    const double total = walk<false>(p, lds, bos + (static_cast<int64_t>(index) << g.shift),
                                     1 << g.shift, head, nullptr, tile);
    if (threadIdx.x == 0)
      g.decays[static_cast<int64_t>(item) * p.num_v_heads + head] =
          __builtin_amdgcn_exp2f(static_cast<float>(total));
    return;
  }
  const int slot = p.indices[seq];
  const bool live = live_slot(slot, p.num_slots);
  float* const home = p.state + static_cast<int64_t>(live ? slot : 0) * p.state_slot + head * kTileFloats;
  walk<true>(p, lds, bos, whole ? rows : 1 << g.shift, head,
             live && p.has_initial[seq] != 0 ? home : nullptr, whole ? (live ? home : nullptr) : tile);
}

// The second: the state at every later segment's start, along each sequence; an eighth of a tile
// a workgroup.
constexpr int kJoinParts = kTileFloats / 4 / kBlock;
__global__ __launch_bounds__(kBlock) void linear_join_kernel(const LinearParams p, const Segments g) {
  __shared__ SearchLds search;
  const int part = blockIdx.x % kJoinParts;
  const int pair = blockIdx.x / kJoinParts;
  const int j = pair / p.num_v_heads;
  const int head = pair - j * p.num_v_heads;
  int seq, index, count;
  if (!find_segment(p, search, g.num_sequences, g.shift, j, seq, index, count) || index != 0) return;
  count = min(count, g.later - j);
  const int64_t step = p.num_v_heads * kTileFloats;
  float* at = g.tiles + (static_cast<int64_t>(j) * p.num_v_heads + head) * kTileFloats +
              (part * kBlock + threadIdx.x) * 4;
  const float* decay = g.decays + static_cast<int64_t>(j) * p.num_v_heads + head;
  f32x4 s = *reinterpret_cast<const f32x4*>(at);
  for (int i = 1; i < count; ++i) {
    at += step;
    decay += p.num_v_heads;
    s = s * *decay + *reinterpret_cast<const f32x4*>(at);
    *reinterpret_cast<f32x4*>(at) = s;
  }
}

// The third: the later segments, each from its state.
__global__ __launch_bounds__(kBlock) __attribute__((amdgpu_waves_per_eu(4, 4)))
void linear_later_kernel(const LinearParams p, const Segments g) {
  __shared__ SegmentLds lds;
  __shared__ SearchLds search;
  int item, head, seq, index, count;
  if (!unit_of(p, g.later, item, head) ||
      !find_segment(p, search, g.num_sequences, g.shift, item, seq, index, count))
    return;
  int64_t bos;
  int rows;
  sequence_rows(p, seq, bos, rows);
  load_weight(p, lds);
  const int done = (index + 1) << g.shift;
  const int slot = p.indices[seq];
  float* const home = p.state + static_cast<int64_t>(slot) * p.state_slot + head * kTileFloats;
  walk<true>(p, lds, bos + done, min(rows - done, 1 << g.shift), head,
             g.tiles + (static_cast<int64_t>(item) * p.num_v_heads + head) * kTileFloats,
             index + 1 == count && live_slot(slot, p.num_slots) ? home : nullptr);
}

// log2 of a segment's tokens: the share of a workgroup where about 512 run at once (two a CU),
// at least 256.
int segment_shift(int64_t num_tokens, int32_t num_v_heads) {
  int shift = 8;
  while (shift < 30 && (int64_t{512} << shift) < num_tokens * num_v_heads) ++shift;
  return shift;
}

// Sequences of more than a segment have at most this many later ones.
int64_t later_segments(int64_t num_tokens, int32_t num_v_heads) {
  return num_tokens > 0 ? (num_tokens - 1) >> segment_shift(num_tokens, num_v_heads) : 0;
}

}  // namespace
}  // namespace ld

extern "C" int64_t ld_linear_prefill_workspace_bytes(int64_t num_tokens, int32_t num_sequences,
                                                     int32_t num_v_heads) {
  if (num_tokens < 0 || num_sequences <= 0 || num_v_heads <= 0) return 0;
  return ld::later_segments(num_tokens, num_v_heads) * num_v_heads *
         static_cast<int64_t>((ld::kTileFloats + 4) * sizeof(float));
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
  if (a.num_tokens > 0x7fffffff) return fail(LD_ERR_INVALID_ARGUMENT, "too many tokens");
  p.indices = a.slots;
  p.cu = a.cu_seqlens;
  p.has_initial = a.has_initial;
  const int64_t later = later_segments(a.num_tokens, a.num_v_heads);
  if (later > 0 && (!aligned16(a.workspace) || a.workspace == nullptr ||
                    a.workspace_bytes < ld_linear_prefill_workspace_bytes(
                                            a.num_tokens, a.num_sequences, a.num_v_heads)))
    return fail(LD_ERR_INVALID_ARGUMENT, "ld_linear_prefill: workspace missing or too small");
  // grids in multiples of 8 XCDs times the group; a grid's threads stay below 2^32
  auto blocks_of = [&](int64_t items) {
    return (items * a.num_k_heads + 7) / 8 * 8 * p.group;
  };
  if (blocks_of(later + a.num_sequences) > 0x7fffff || later * a.num_v_heads * kJoinParts > 0x7fffff)
    return fail(LD_ERR_INVALID_ARGUMENT, "too many (sequence, head) tiles");
  Segments g{};
  g.num_sequences = a.num_sequences;
  g.shift = segment_shift(a.num_tokens, a.num_v_heads);
  g.later = static_cast<int>(later);
  g.tiles = static_cast<float*>(a.workspace);
  g.decays = g.tiles + later * a.num_v_heads * kTileFloats;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(linear_first_kernel, dim3(static_cast<uint32_t>(blocks_of(later + a.num_sequences))),
                     dim3(kBlock), 0, s, p, g);
  if (later > 1)   // (a lone later segment starts from what the first launch left)
    hipLaunchKernelGGL(linear_join_kernel, dim3(static_cast<uint32_t>(later * a.num_v_heads * kJoinParts)),
                       dim3(kBlock), 0, s, p, g);
  if (later > 0)
    hipLaunchKernelGGL(linear_later_kernel, dim3(static_cast<uint32_t>(blocks_of(later))),
                       dim3(kBlock), 0, s, p, g);
  return check_launch("ld_linear_prefill");
}
