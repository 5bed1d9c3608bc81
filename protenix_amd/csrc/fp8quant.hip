// Matrices into 8-bit blocks of 128 (fp8.h): along their rows, along their columns (the result is the transposed matrix's, as a
// product over the rows reads it), or both in one pass; a scale per 128 values or, for weights, per 128 x 128.
//
// Bound by memory: an element is read once and written once per direction.  Rows alone: 16 lanes hold a block in registers.  Else
// a workgroup holds a tile of 128 x 128 in its registers, 8 x 8 per thread, takes the largest magnitudes of its rows among 16 lanes
// and of its columns through LDS, and turns the bytes round in LDS, from where the transposed rows go out in whole lines of 128 bytes.
// 16384 x 4096 bf16 both ways 55.7 us among other passes (4.9 TB/s; a plain copy 5.8), its rows alone 39 (5.3); 8192 x 4096 square both
// ways 29.1, in a training pass 35.  On the same tensors again 49, with tiles in one run per XCD 51 - 56, with loads past the caches 49 - 55.
#include "fp8.h"
#include "dropout.h"
#include "kernels.h"

namespace ptx {

// x [rows][cols] -> q [rows][fp8_pitch(cols)], scales [blocks][fp8_scale_pitch(rows)]
template <typename T, bool SHORT>
__global__ __launch_bounds__(256) void fp8_rows_kernel(const T* __restrict__ x, uint8_t* __restrict__ q, float* __restrict__ scales,
                                                       uint32_t rows, int cols, uint32_t n_blocks) {
  const uint32_t per_row = (uint32_t)fp8_blocks(cols), at = blockIdx.x * 16u + threadIdx.x / 16;
  // (blocks beyond the end: the last one once more, not written)
  const bool ok = at < n_blocks;
  const uint32_t block = ok ? at : n_blocks - 1, row = block / per_row, kb = block - row * per_row;
  const int col = (int)(kb * kFp8Block + threadIdx.x % 16 * 8), n = max(min(cols - col, 8), 0);
  f32x8 v = used_cols<SHORT, T>(load_cols<SHORT>(x + (int64_t)row * cols, col, cols), n);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = e < n ? v[e] : 0.0f;
  const Fp8Scale s = fp8_scale(largest16(magnitude(v)));
  if (!ok) return;
  *reinterpret_cast<u32x2_t*>(q + (int64_t)row * fp8_pitch(cols) + col) = fp8_pack8(v, s.i);
  if (threadIdx.x % 16 == 0) scales[(int64_t)kb * fp8_scale_pitch(rows) + row] = s.s;
}

// Largest magnitudes of 8 values at a time, as whole numbers: for 16-bit types in pairs, on the bits as they come.
template <typename T> struct Tops {
  typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
  static constexpr int kWords = 4;      // per 8 values, as they travel between lanes
  u16x8 v;
  __device__ __forceinline__ explicit Tops(const Raw8<T>& raw) : v(__builtin_bit_cast(u16x8, raw) & (unsigned short)0x7fff) {}
  __device__ __forceinline__ void take(const Tops& o) { v = __builtin_elementwise_max(v, o.v); }
  __device__ __forceinline__ uint32_t word(int k) const { return (uint32_t)v[2 * k] | (uint32_t)v[2 * k + 1] << 16; }
  __device__ __forceinline__ void take_word(int k, uint32_t w) {
    v[2 * k] = max(v[2 * k], (unsigned short)w);
    v[2 * k + 1] = max(v[2 * k + 1], (unsigned short)(w >> 16));
  }
  // one of them, or the largest, as the bits of a float
  __device__ __forceinline__ uint32_t bits(int e) const {
    const unsigned short m = v[e];      // (by way of a variable: a cast of a vector's element takes the first one)
    return __float_as_uint((float)__builtin_bit_cast(T, m));
  }
  __device__ __forceinline__ uint32_t largest_bits() const {
    unsigned short m = v[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) m = max(m, v[e]);
    return __float_as_uint((float)__builtin_bit_cast(T, m));
  }
};
template <> struct Tops<float> {
  static constexpr int kWords = 8;
  uint32_t v[8];
  __device__ __forceinline__ explicit Tops(const Raw8<float>& raw) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = magnitude(raw[e]);
  }
  __device__ __forceinline__ void take(const Tops& o) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = max(v[e], o.v[e]);
  }
  __device__ __forceinline__ uint32_t word(int k) const { return v[k]; }
  __device__ __forceinline__ void take_word(int k, uint32_t w) { v[k] = max(v[k], w); }
  __device__ __forceinline__ uint32_t bits(int e) const { return v[e]; }
  __device__ __forceinline__ uint32_t largest_bits() const {
    uint32_t m = v[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) m = max(m, v[e]);
    return m;
  }
};

// One tile of 128 x 128 per workgroup.  q, qt: either may be null.  part: null, or the tile's column sums of x, [tiles of rows][cols].
template <typename T, bool SHORT, bool SQUARE>
__global__ __launch_bounds__(256) void fp8_tile_kernel(const T* __restrict__ x, uint8_t* __restrict__ q, float* __restrict__ scales,
                                                       uint8_t* __restrict__ qt, float* __restrict__ scales_t, float* __restrict__ part,
                                                       int64_t rows, int cols) {
  // (column 8 l + e of the tile at e 16 + l of the arrays by column: neighbouring lanes then use neighbouring banks)
  __shared__ __align__(16) uint8_t turned[kFp8Block * kFp8Block];
  __shared__ uint32_t tops[4][Tops<T>::kWords][16];
  __shared__ float inverse[kFp8Block], sums[4][kFp8Block];
  __shared__ uint32_t top_of_all[4];
  const int tiles = (int)fp8_blocks(cols), tid = threadIdx.x, wave = tid >> 6, l = tid & 15, g = tid >> 4;
  // (tiles go down BAND rows of them before the next column's, so that the lines of 128 bytes that neighbouring tiles write of a transposed row
  // go out together: 16384 x 4096 bf16 59 -> 55.7 us, with 2, 4 or 32 58, 57, 57, with 8 columns' tiles side by side in a band 58.5; of fp32, which reads more than it writes, 44.7 -> 45.7,
  // and 8192 x 2048 square 11.3 -> 11.8)
  constexpr uint32_t BAND = sizeof(T) == 2 && !SQUARE ? 8 : 1;
  const uint32_t of_band = BAND * (uint32_t)tiles, band = blockIdx.x / of_band, in = blockIdx.x - band * of_band;
  const uint32_t high = min(BAND, (uint32_t)fp8_blocks(rows) - band * BAND);
  const int64_t row_tile = band * BAND + in % high;
  const int col_tile = (int)(in / high);
  const int64_t row0 = row_tile * kFp8Block + 8 * g;      // this thread's rows row0 .. row0 + 7
  const int col = col_tile * kFp8Block + 8 * l, n = max(min(cols - col, 8), 0);
  Raw8<T> raw[8];
#pragma unroll
  for (int p = 0; p < 8; ++p) raw[p] = load_cols<SHORT>(x + min(row0 + p, rows - 1) * cols, col, cols);
  if (SHORT || (row_tile + 1) * kFp8Block > rows || (col_tile + 1) * kFp8Block > cols) {
    // (zeros beyond the end; the values are T's own, and so their rounding to T is none)
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      f32x8 v = used_cols<SHORT, T>(raw[p], n);
      const int have = row0 + p < rows ? n : 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < have ? v[e] : 0.0f;
      raw[p] = rounded<T>(v);
    }
  }
  uint32_t row_top[8];
  Tops<T> col_top(raw[0]);
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const Tops<T> t(raw[p]);
    if (p > 0) col_top.take(t);
    if (!SQUARE) row_top[p] = largest16(t.largest_bits());
  }
  // the largest of each column's 8 rows, then over the four groups of rows of a wave, then over the waves
#pragma unroll
  for (int k = 0; k < Tops<T>::kWords; ++k) {
    col_top.take_word(k, (uint32_t)__shfl_xor((int)col_top.word(k), 16, 64));
    col_top.take_word(k, (uint32_t)__shfl_xor((int)col_top.word(k), 32, 64));
  }
  f32x8 v[8];
#pragma unroll
  for (int p = 0; p < 8; ++p) v[p] = widened<T>(raw[p]);
  if (part) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float s = 0.0f;
#pragma unroll
      for (int p = 0; p < 8; ++p) s += v[p][e];
      s += __shfl_xor(s, 16, 64);
      s += __shfl_xor(s, 32, 64);
      if ((tid & 63) < 16) sums[wave][16 * e + l] = s;
    }
  }
  if constexpr (SQUARE) {
    const uint32_t m = largest16(col_top.largest_bits());
    if ((tid & 63) == 0) top_of_all[wave] = m;
  } else if ((tid & 63) < 16) {
#pragma unroll
    for (int k = 0; k < Tops<T>::kWords; ++k) tops[wave][k][l] = col_top.word(k);
  }
  __syncthreads();
  Fp8Scale all;
  if constexpr (SQUARE) all = fp8_scale(max(max(top_of_all[0], top_of_all[1]), max(top_of_all[2], top_of_all[3])));
  if (part && tid < kFp8Block && col_tile * kFp8Block + tid < cols) {
    const int at = 16 * (tid & 7) + (tid >> 3);
    part[row_tile * cols + col_tile * kFp8Block + tid] = (sums[0][at] + sums[1][at]) + (sums[2][at] + sums[3][at]);
  }
  if (!SQUARE && qt && tid < 16) {
    // the columns' scales, once: 8 of them per thread of 16
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int k = 0; k < Tops<T>::kWords; ++k) col_top.take_word(k, tops[w][k][l]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const Fp8Scale s = fp8_scale(col_top.bits(e));
      inverse[16 * e + l] = s.i;
      if (e < n) scales_t[row_tile * fp8_scale_pitch(cols) + col + e] = s.s;
    }
  }
  const int64_t pitch = fp8_pitch(cols), row_tiles = fp8_blocks(rows);
  if (q) {
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      if (row0 + p >= rows) break;
      const Fp8Scale s = SQUARE ? all : fp8_scale(row_top[p]);
      *reinterpret_cast<u32x2_t*>(q + (row0 + p) * pitch + col) = fp8_pack8(v[p], s.i);
      if (!SQUARE && l == 0) scales[(int64_t)col_tile * fp8_scale_pitch(rows) + row0 + p] = s.s;
    }
    if (SQUARE && tid == 0) scales[row_tile * tiles + col_tile] = all.s;
  }
  if (!qt) return;
  if (!SQUARE) __syncthreads();
  // Column 8 l + e of the tile as row of `turned`, its rows 8 g .. 8 g + 7 as 8 bytes in place g ^ l (of 16): the 64 lanes of a wave
  // write to, and 16 bytes later read from, all banks alike.
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    f32x8 t;
#pragma unroll
    for (int p = 0; p < 8; ++p) t[p] = v[p][e];
    *reinterpret_cast<u32x2_t*>(turned + (8 * l + e) * kFp8Block + ((g ^ l) << 3)) = fp8_pack8(t, SQUARE ? all.i : inverse[16 * e + l]);
  }
  if (SQUARE && tid == 0) scales_t[(int64_t)col_tile * row_tiles + row_tile] = all.s;
  __syncthreads();
  const int64_t pitch_t = fp8_pitch(rows);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = 32 * i + (tid >> 3), j = tid & 7, turn = c >> 3;      // bytes 16 j .. 16 j + 15 of the column: places 2 j and 2 j + 1, each ^ turn
    const u32x4_t b = *reinterpret_cast<const u32x4_t*>(turned + c * kFp8Block + ((j ^ (turn >> 1)) << 4));
    const u32x4_t o = turn & 1 ? u32x4_t{b[2], b[3], b[0], b[1]} : b;
    if (col_tile * kFp8Block + c < cols)
      *reinterpret_cast<u32x4_t*>(qt + (int64_t)(col_tile * kFp8Block + c) * pitch_t + row_tile * kFp8Block + 16 * j) = o;
  }
}

template <typename T>
int fp8_quantize(const T* x, void* q, float* scales, void* qt, float* scales_t, float* part, int64_t rows, int cols, bool square,
                 hipStream_t stream) {
  const int64_t row_blocks = rows * fp8_blocks(cols), tiles = fp8_blocks(rows) * fp8_blocks(cols);
  if (!qt && !square && !part) {
    auto* kernel = cols < 8 ? fp8_rows_kernel<T, true> : fp8_rows_kernel<T, false>;
    kernel<<<dim3((unsigned)((row_blocks + 15) / 16)), dim3(256), 0, stream>>>(x, (uint8_t*)q, scales, (uint32_t)rows, cols, (uint32_t)row_blocks);
    return 0;
  }
  auto* kernel = cols < 8 ? (square ? fp8_tile_kernel<T, true, true> : fp8_tile_kernel<T, true, false>)
                          : (square ? fp8_tile_kernel<T, false, true> : fp8_tile_kernel<T, false, false>);
  kernel<<<dim3((unsigned)tiles), dim3(256), 0, stream>>>(x, (uint8_t*)q, scales, (uint8_t*)qt, scales_t, part, rows, cols);
  return 0;
}

#define PTX_FP8_TYPES(T) template int fp8_quantize(const T*, void*, float*, void*, float*, float*, int64_t, int, bool, hipStream_t);
PTX_FP8_TYPES(float)
PTX_FP8_TYPES(bf16_t)
PTX_FP8_TYPES(f16_t)

}  // namespace ptx
