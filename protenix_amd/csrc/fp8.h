// Values of 8 bits with a scale per block of 128 (fp8quant.hip, rmsnorm.hip; read by fp8gemm.hip).
//
// A block with the largest magnitude a has the scale s = max(a / 448, 2^-126) and, with i = 1 / s, the values
// q = e4m3(v i): 1 sign, 4 exponent and 3 mantissa bits, largest 448, rounded to the nearest, ties to even.  s, i and v i are each
// rounded once to 32 bits, so that every kernel has the same bits; |v i| is at most 448 (1 + 2^-22), which rounds to 448.  2^-126 keeps
// i finite and normal for blocks of zeros and of tiny values.  An infinity or a NaN makes the block's scale that, and so
// every product of the block is infinite or NaN.
//
// Layout of a matrix [rows][cols]: values in rows of fp8_pitch(cols) bytes, zeros behind the last column; scales by block of columns
// first, [blocks][fp8_scale_pitch(rows)], so that the rows of a tile of the product lie side by side (a scale per 128 x 128 values:
// [blocks of rows][blocks of columns]).
#pragma once
#include "common.h"

namespace ptx {

constexpr int kFp8Block = 128;

__host__ __device__ __forceinline__ int64_t fp8_blocks(int64_t n) { return (n + kFp8Block - 1) / kFp8Block; }
__host__ __device__ __forceinline__ int64_t fp8_pitch(int64_t cols) { return fp8_blocks(cols) * kFp8Block; }
__host__ __device__ __forceinline__ int64_t fp8_scale_pitch(int64_t rows) { return (rows + 3) / 4 * 4; }

// Magnitudes as whole numbers: in their order, with infinities and NaN above all (a maximum of floats would lose the NaN).
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t magnitude(const f32x8& v) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, magnitude(v[e]));
  return m;
}

// The largest of 16 neighbouring lanes, in all of them, on the vector pipe (moves within rows of 16 lanes).
template <int CTRL> __device__ __forceinline__ uint32_t lane_moved(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true);
}
__device__ __forceinline__ uint32_t largest16(uint32_t v) {
  v = max(v, lane_moved<0xB1>(v));        // lane ^ 1 (within four: 1 0 3 2)
  v = max(v, lane_moved<0x4E>(v));        // lane ^ 2 (2 3 0 1)
  v = max(v, lane_moved<0x141>(v));       // 7 - lane within 8: the other four
  return max(v, lane_moved<0x140>(v));    // 15 - lane within 16: the other eight
}

struct Fp8Scale {
  float s, i;
};
// Both quotients rounded once, in three operations each where a division takes ten: an approximation and a correction from its exact
// remainder (Markstein: Computation of elementary functions on the IBM RISC System/6000 processor, 1990).  One correction of 1 / s is rounded
// rightly from this instruction's approximations, at each of the 2^23 mantissas (compared; tests/test_gpu_fp8_contract.py holds the bits); from
// others off by a unit it would not be at some.  Where top / 448 would be subnormal the result is 2^-126 either way.
__device__ __forceinline__ Fp8Scale fp8_scale(uint32_t top) {
  const float a = __uint_as_float(top), least = 1.1754943508222875e-38f, r = 1.0f / 448.0f;
  float s = a * r;
  s = __builtin_fmaf(__builtin_fmaf(-448.0f, s, a), r, s);
  float i = __builtin_amdgcn_rcpf(s < least ? least : s);
  i = __builtin_fmaf(__builtin_fmaf(-(s < least ? least : s), i, 1.0f), i, i);
  const bool infinite = top == 0x7f800000u;      // (its remainder is no number)
  Fp8Scale q;
  q.s = infinite ? a : s < least ? least : s;      // (a NaN stays)
  q.i = infinite ? 0.0f : i;
  return q;
}

typedef __attribute__((ext_vector_type(2))) uint32_t u32x2_t;
__device__ __forceinline__ u32x2_t fp8_pack8(const f32x8& v, float i) {
  u32x2_t q;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    int p = 0;
    p = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * w] * i, v[4 * w + 1] * i, p, false);
    p = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * w + 2] * i, v[4 * w + 3] * i, p, true);
    q[w] = (uint32_t)p;
  }
  return q;
}

}  // namespace ptx
