// out = residual + dropout(x), and the gradient of x: the same kernel on the gradient, without a residual.
//
// One pass: x, the residual and the sum are moved once, the mask costs no memory.  A thread owns one block of 8 columns
// of a mask row and walks the rows that share it: the mask is drawn once per block and used for every one of them.
#include <algorithm>

#include "dropout.h"
#include "kernels.h"

namespace ptx {

// TI: type of x; TO: of the residual and the sum.  AHEAD: rows requested before the first is worked on (1: a mask row is
// one row).  SHORT: fewer than 8 columns.
template <typename TI, typename TO, bool RES, int AHEAD, bool SHORT>
__global__ __launch_bounds__(256) void dropout_add_kernel(const TI* __restrict__ x, const TO* __restrict__ res, TO* __restrict__ out,
                                                          int cols, uint32_t n_vec, int64_t n_blocks, uint32_t rows_at_once, Dropout drop) {
  drop = with_key(drop);
  for (int64_t block = (int64_t)blockIdx.x * 256 + threadIdx.x; block < n_blocks; block += (int64_t)gridDim.x * 256) {
    // (a 64-bit division costs as much as the mask)
    const uint32_t mask_row = n_blocks >> 32 ? (uint32_t)(block / n_vec) : (uint32_t)block / n_vec;
    const uint32_t k = (uint32_t)(block - (int64_t)mask_row * n_vec);
    const uint32_t outer = AHEAD == 1 ? mask_row : mask_row / drop.inner, in = AHEAD == 1 ? 0 : mask_row - outer * drop.inner;
    const uint32_t s0 = AHEAD == 1 ? 0 : blockIdx.y * rows_at_once, s1 = AHEAD == 1 ? 1 : min(s0 + rows_at_once, drop.shared);
    const int n = min(cols - (int)(k * 8), 8);
    const int64_t step = AHEAD == 1 ? 0 : (int64_t)drop.inner * cols;
    int64_t at = AHEAD == 1 ? (int64_t)mask_row * cols : (((int64_t)outer * drop.shared + s0) * drop.inner + in) * cols;
    // (before the loads: waves that draw while others load take 52 us where 63 on 65536 x 768 bf16 with a residual, all loads first)
    const uint32_t keeps = dropout_keeps(drop, mask_row, k);
    for (uint32_t s = s0; s < s1; s += AHEAD) {
      Raw8<TI> raw[AHEAD];
      Raw8<TO> raw_res[AHEAD];
#pragma unroll
      for (uint32_t r = 0; r < AHEAD; ++r) {
        const int64_t row = at + (s + r < s1 ? r : s1 - 1 - s) * step;      // (beyond the last: that one once more)
        raw[r] = load_cols<SHORT>(x + row, k * 8, cols);
        if (RES) raw_res[r] = load_cols<SHORT>(res + row, k * 8, cols);
      }
#pragma unroll
      for (uint32_t r = 0; r < AHEAD; ++r) {
        if (s + r >= s1) break;
        f32x8 v = used_cols<SHORT, TI>(raw[r], n);
        if (RES) {
          const f32x8 y = used_cols<SHORT, TO>(raw_res[r], n);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(kept(v[e], keeps, e), drop.scale, y[e]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = kept(v[e], keeps, e) * drop.scale;
        }
        store_cols(out + at + k * 8, v, n);
        at += step;
      }
    }
  }
}

template <typename TI, typename TO, bool RES>
static void launch(const TI* x, const TO* res, TO* out, int64_t rows, int cols, const Dropout& drop, hipStream_t stream) {
  const uint32_t n_vec = (uint32_t)((cols + 7) / 8);
  const int64_t n_blocks = rows / drop.shared * n_vec;
  const uint32_t at_once = std::min<uint32_t>(drop.shared, std::max<uint32_t>(8, (drop.shared + 65534) / 65535));
  // (2^32 threads at most along a grid's axis)
  const dim3 grid((unsigned)std::min<int64_t>((n_blocks + 255) / 256, 1 << 23), (drop.shared + at_once - 1) / at_once);
  if (cols < 8 && drop.shared == 1)
    dropout_add_kernel<TI, TO, RES, 1, true><<<grid, dim3(256), 0, stream>>>(x, res, out, cols, n_vec, n_blocks, at_once, drop);
  else if (cols < 8)
    dropout_add_kernel<TI, TO, RES, 4, true><<<grid, dim3(256), 0, stream>>>(x, res, out, cols, n_vec, n_blocks, at_once, drop);
  else if (drop.shared == 1)
    dropout_add_kernel<TI, TO, RES, 1, false><<<grid, dim3(256), 0, stream>>>(x, res, out, cols, n_vec, n_blocks, at_once, drop);
  else
    dropout_add_kernel<TI, TO, RES, 4, false><<<grid, dim3(256), 0, stream>>>(x, res, out, cols, n_vec, n_blocks, at_once, drop);
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
