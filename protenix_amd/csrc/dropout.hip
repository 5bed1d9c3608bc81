// out = residual + dropout(x), and the gradient of x: the same kernel on the gradient, without a residual.
//
// One pass: x, the residual and the sum are moved once, the mask costs no memory.  A thread owns one block of 8 columns of a mask
// row and four of the rows that share it (one, where a row has a mask row of its own): the mask is drawn once for them.  Bound by
// memory; [768, 768, 128] bf16 onto fp32 rows 127 us, its gradient 82 (5.9 and 5.5 TB/s), 65536 x 768 bf16 with a mask for
// every row 51 and 37 us (5.9 and 5.5), where a plain copy reaches 5.8.
#include <algorithm>

#include "dropout.h"
#include "kernels.h"

namespace ptx {

// TI: type of x; TO: of the residual and the sum.  ROWS: of a mask row in a thread.  SHORT: fewer than 8 columns.
template <typename TI, typename TO, bool RES, int ROWS, bool SHORT>
__global__ __launch_bounds__(256) void dropout_add_kernel(const TI* __restrict__ x, const TO* __restrict__ res, TO* __restrict__ out,
                                                          int cols, uint32_t n_vec, int64_t n_blocks, Dropout drop) {
  drop = with_key(drop);
  for (int64_t block = (int64_t)blockIdx.x * 256 + threadIdx.x; block < n_blocks; block += (int64_t)gridDim.x * 256) {
    // (a 64-bit division costs as much as the mask)
    const uint32_t mask_row = n_blocks >> 32 ? (uint32_t)(block / n_vec) : (uint32_t)block / n_vec;
    const uint32_t k = (uint32_t)(block - (int64_t)mask_row * n_vec);
    const uint32_t outer = ROWS == 1 ? mask_row : mask_row / drop.inner, in = ROWS == 1 ? 0 : mask_row - outer * drop.inner;
    const uint32_t shared = ROWS == 1 ? 1 : drop.shared;
    const int n = min(cols - (int)(k * 8), 8);
    // (before the loads: waves that draw while others load take 51 us where all loads first take 63, on 65536 x 768 bf16)
    const uint32_t keeps = dropout_keeps(drop, mask_row, k);
    const int64_t step = (int64_t)(ROWS == 1 ? 1 : drop.inner) * cols;
    for (uint32_t s = ROWS == 1 ? 0 : blockIdx.y * ROWS; s < shared; s += ROWS == 1 ? 1 : gridDim.y * ROWS) {
      const int64_t at = (((int64_t)outer * shared + s) * (ROWS == 1 ? 1 : drop.inner) + in) * cols;
      Raw8<TI> raw[ROWS];
      Raw8<TO> raw_res[ROWS];
#pragma unroll
      for (uint32_t r = 0; r < ROWS; ++r) {
        const int64_t row = at + min(r, shared - 1 - s) * step;      // (beyond the last: that one once more, not used)
        raw[r] = load_cols<SHORT>(x + row, k * 8, cols);
        if (RES) raw_res[r] = load_cols<SHORT>(res + row, k * 8, cols);
      }
#pragma unroll
      for (uint32_t r = 0; r < ROWS; ++r) {
        if (s + r >= shared) break;
        f32x8 v = used_cols<SHORT, TI>(raw[r], n), y = f32x8{};
        if (RES) y = used_cols<SHORT, TO>(raw_res[r], n);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          v[e] = RES ? __builtin_fmaf(kept(v[e], keeps, e), drop.scale, y[e]) : kept(v[e], keeps, e) * drop.scale;
        store_cols(out + at + r * step + k * 8, v, n);
      }
    }
  }
}

template <typename TI, typename TO, bool RES>
static void launch(const TI* x, const TO* res, TO* out, int64_t rows, int cols, const Dropout& drop, hipStream_t stream) {
  constexpr int kRows = 4;      // us of the pair tensor above, forward and gradient, in one sweep: two 126 and 84, four 127 and 83, eight 137 and 87
  const uint32_t n_vec = (uint32_t)((cols + 7) / 8);
  const int64_t n_blocks = rows / drop.shared * n_vec;
  // (2^32 threads at most along a grid's axis)
  const dim3 grid((unsigned)std::min<int64_t>((n_blocks + 255) / 256, 1 << 23), std::min<uint32_t>((drop.shared + kRows - 1) / kRows, 65535));
  auto* kernel = drop.shared == 1 ? (cols < 8 ? dropout_add_kernel<TI, TO, RES, 1, true> : dropout_add_kernel<TI, TO, RES, 1, false>)
                                  : (cols < 8 ? dropout_add_kernel<TI, TO, RES, kRows, true> : dropout_add_kernel<TI, TO, RES, kRows, false>);
  kernel<<<grid, dim3(256), 0, stream>>>(x, res, out, cols, n_vec, n_blocks, drop);
}

template <typename TI, typename TO>
int dropout_add(const TI* x, const TO* res, TO* out, int64_t rows, int cols, const Dropout& drop, hipStream_t stream) {
  if (rows == 0) return 0;
  if (res) launch<TI, TO, true>(x, res, out, rows, cols, drop, stream);
  else launch<TI, TO, false>(x, nullptr, out, rows, cols, drop, stream);
  return 0;
}

template int dropout_add(const float*, const float*, float*, int64_t, int, const Dropout&, hipStream_t);
template int dropout_add(const bf16_t*, const bf16_t*, bf16_t*, int64_t, int, const Dropout&, hipStream_t);
template int dropout_add(const f16_t*, const f16_t*, f16_t*, int64_t, int, const Dropout&, hipStream_t);
template int dropout_add(const bf16_t*, const float*, float*, int64_t, int, const Dropout&, hipStream_t);
template int dropout_add(const f16_t*, const float*, float*, int64_t, int, const Dropout&, hipStream_t);
template int dropout_add(const float*, const bf16_t*, bf16_t*, int64_t, int, const Dropout&, hipStream_t);
template int dropout_add(const float*, const f16_t*, f16_t*, int64_t, int, const Dropout&, hipStream_t);

}  // namespace ptx
