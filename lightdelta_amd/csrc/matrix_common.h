// Device helpers of the kernels that keep a whole head's state in the accumulators of
// v_mfma_f32_32x32x16_bf16 (prefill_heads.hip, linear_prefill.hip): matrix instructions, exact
// splits of their registers into operands, transposed LDS reads and 64-bit lane moves.
#pragma once

#include "chunk_common.h"

namespace ld {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kTileRow = kDim * 2;             // bytes of a q, k, v or raw-output row in LDS

// 16-byte pieces of row r are stored at piece ^ swizzle(r): a column of pieces over 16 rows
// (operand A of the products with S) and 4 x 4 element blocks of 4 rows (transposed reads)
// each cover every bank once.
__device__ __forceinline__ constexpr int swizzle(int row) {
  return ((row & 3) << 2) | ((row >> 2) & 3);
}

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Fixes the order of pure operations: a value is defined ahead of this point and not used
// before it, and the points keep their order in the program.  (Left to itself the compiler
// lines the splits up ahead of the matrix instructions that should run beside them; it
// emits nothing for a pin.)
template <typename T>
__device__ __forceinline__ void pin(T& x) {
  asm volatile("" : "+v"(x));
}

// The exact split of eight values (a lane's registers 8 u .. 8 u + 7 of an accumulator) into
// planes that are B operands, in five stages: 0, 2, 4 round (4 instructions), 1, 3 take the
// remainders (16: each value less its plane's, exact).  split4's remainder is one v_dot2c, but
// that does not run beside a matrix instruction: with 8 of them behind each, a matrix
// instruction of 32 cycles took 81 (78 with two waves a SIMD); with 8 of these, 46 (42).
struct Split8 {
  float r[8];
  u32x4 w[3];
  __device__ __forceinline__ void set(f32x4 lo, f32x4 hi) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      r[e] = lo[e];
      r[4 + e] = hi[e];
    }
  }
  __device__ __forceinline__ void stage(int i) {  // 0 .. 4
    if (i & 1) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t pair = w[i >> 1][j];
        r[2 * j] -= __builtin_bit_cast(float, pair << 16);
        r[2 * j + 1] -= __builtin_bit_cast(float, pair & 0xffff0000u);
      }
      asm volatile("" : "+v"(r[0]), "+v"(r[1]), "+v"(r[2]), "+v"(r[3]), "+v"(r[4]), "+v"(r[5]),
                   "+v"(r[6]), "+v"(r[7]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[i >> 1][j] = bf16_pair(f32x2{r[2 * j], r[2 * j + 1]});
      pin(w[i >> 1]);
    }
  }
  __device__ __forceinline__ void all() {
#pragma unroll
    for (int i = 0; i < 5; ++i) stage(i);
  }
  __device__ __forceinline__ bf16x8 plane(int i) const {
    return __builtin_bit_cast(bf16x8, w[i]);
  }
};
__device__ __forceinline__ f32x4 quad(const f32x16& x, int q) {
  return f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
}

// 4 x 16 block of bf16 transposed on the way from LDS: within 16 lanes, lane m gives the
// address of row m / 4, elements 4 (m % 4) .. + 3, and receives rows 0 .. 3 of column m.
__device__ __forceinline__ bf16x4 read_tr(const uint8_t* at) {
  const auto p = (__attribute__((address_space(3))) s16x4*)(at);
  return __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p));
}

// Sixteen bytes of a row at a lane's byte offset + a uniform one: one load, or (rows not at
// 16-byte boundaries) eight of one element.
template <bool Wide>
__device__ __forceinline__ u32x4 load_piece(__amdgpu_buffer_rsrc_t rs, uint32_t offset,
                                            int uniform) {
  if constexpr (Wide) return load16u(rs, offset, uniform);
  u32x4 out;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = __builtin_amdgcn_raw_buffer_load_b16(rs, static_cast<int>(offset + 4 * i), uniform, 0);
    const uint32_t hi = __builtin_amdgcn_raw_buffer_load_b16(rs, static_cast<int>(offset + 4 * i + 2), uniform, 0);
    out[i] = (lo & 0xffffu) | (hi << 16);
  }
  return out;
}

// The 64-bit value of the lane that Ctrl names (zero where it names none).
template <int Ctrl>
__device__ __forceinline__ double dpp64(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), Ctrl, 0xF, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), Ctrl, 0xF, 0xF, false);
  return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}

}  // namespace
}  // namespace ld
