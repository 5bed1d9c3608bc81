// out = residual + dropout(x), and the gradient of x: the same kernel on the gradient, without a residual.
//
// One pass: x, the residual and the sum are moved once, the mask costs no memory.  A thread owns one block of 8 columns
// of a mask row and walks the rows that share it: the mask is drawn once per block and used for every one of them.
#include <algorithm>

#include "dropout.h"
#include "kernels.h"

namespace ptx {

// TI: type of x; TO: of the residual and the sum.
template <typename TI, typename TO, bool RES>
__global__ __launch_bounds__(256) void dropout_add_kernel(const TI* __restrict__ x, const TO* __restrict__ res, TO* __restrict__ out,
                                                          int cols, uint32_t n_vec, int64_t n_blocks, int rows_at_once, Dropout drop) {
  const bool masked = (drop.hi | drop.lo) != 0;
  drop = with_key(drop);
  for (int64_t block = (int64_t)blockIdx.x * 256 + threadIdx.x; block < n_blocks; block += (int64_t)gridDim.x * 256) {
    const uint32_t mask_row = (uint32_t)(block / n_vec), k = (uint32_t)(block - (int64_t)mask_row * n_vec);
    const uint32_t outer = mask_row / drop.inner, in = mask_row - outer * drop.inner;
    const uint32_t s0 = blockIdx.y * rows_at_once, s1 = min(s0 + rows_at_once, drop.shared);
    const int n = min(cols - (int)(k * 8), 8);
    float factor[8] = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
    if (masked) dropout_factors(drop, mask_row, k, factor);
    const int64_t step = (int64_t)drop.inner * cols;
    int64_t at = (((int64_t)outer * drop.shared + s0) * drop.inner + in) * cols + k * 8;
    for (uint32_t s = s0; s < s1; ++s, at += step) {
      f32x8 v = load_cols(x + at, n);
      if (RES) {
        const f32x8 r = load_cols(res + at, n);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = dropped_add(v[e], factor[e], r[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = dropped(v[e], factor[e]);
      }
      store_cols(out + at, v, n);
    }
  }
}

template <typename TI, typename TO>
int dropout_add(const TI* x, const TO* res, TO* out, int64_t rows, int cols, const Dropout& drop, hipStream_t stream) {
  if (rows == 0) return 0;
  const uint32_t n_vec = (uint32_t)((cols + 7) / 8);
  const int64_t n_blocks = rows / drop.shared * n_vec, groups = (n_blocks + 255) / 256;
  const int at_once = std::min<int>(drop.shared, std::max(8, (int)((drop.shared + 65534) / 65535)));
  // (2^32 threads at most along a grid's axis)
  const dim3 grid((unsigned)std::min<int64_t>(groups, 1 << 23), (drop.shared + at_once - 1) / at_once);
  if (res)
    dropout_add_kernel<TI, TO, true><<<grid, dim3(256), 0, stream>>>(x, res, out, cols, n_vec, n_blocks, at_once, drop);
  else
    dropout_add_kernel<TI, TO, false><<<grid, dim3(256), 0, stream>>>(x, nullptr, out, cols, n_vec, n_blocks, at_once, drop);
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
