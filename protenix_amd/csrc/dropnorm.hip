// h = residual + dropout(x) and y = LayerNorm(h), with their gradients, in one pass over the rows each.
//
//   forward    h = res + m x,  y = (h - mean) rstd gamma + beta             m = 1 / (1 - p) or 0 (dropout.h)
//   backward   with g = gamma dy, xh = (h - mean) rstd:
//              dres = rstd (g - avg(g) - xh avg(g xh)) + dh,  dx = m dres,
//              dgamma = sum_rows dy xh,  dbeta = sum_rows dy
//
// A row lies over its lanes in registers, one block of 8 columns per lane (= one draw of the mask, see dropout.h), two for
// rows of more than 8192 columns: 1 to 64 lanes of a wave for up to 512 columns, as many waves of a workgroup as hold it
// beyond, whose sums meet in LDS.  Statistics are fp32 and taken in two passes over the registers, from the sum before it is rounded to h.
// The backward pass takes h from memory where it is fp32, and forms it again from x and the residual where the stream
// has 16 bits: xh of a rounded h would leave dgamma with an error of 2^-8 instead of 2^-24, for the sake of one
// 16-bit read.  Bound by memory: 16384 rows of 2048 bf16 forward 49 us (5.5 TB/s), backward 83 and 5 for the sums (4.9 TB/s of its
// 12 bytes an element; 75 where its tensors are partly in the caches); 147456 rows of 128 bf16 on fp32 44 and 51 us; a plain
// copy reaches 5.8 TB/s.  dgamma and dbeta: column sums in registers over the rows a workgroup walks, one row of fp32 partial sums per
// workgroup, added in a fixed order by layernorm_bwd_reduce (no atomics).
#include "kernels.h"
#include "normrows.h"

namespace ptx {

__device__ __forceinline__ uint32_t mask_row_of(const Dropout& d, uint32_t row) {
  if (d.shared == 1) return row;
  const uint32_t o = row / (d.shared * d.inner);
  return o * d.inner + row % d.inner;
}

// TX: type of x and y; TR: of the residual and h.  SHORT: fewer than 8 columns.  RES: with a residual.
template <typename TX, typename TR, int G, int WAVES, int NC, bool SHORT, bool RES>
__global__ __launch_bounds__((Lay<G, WAVES>::kThreads)) void dropnorm_fwd_kernel(
    const TX* __restrict__ x, const TR* __restrict__ res, NormParam gamma, NormParam beta, TX* __restrict__ y, TR* __restrict__ h,
    float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t rows, int cols, float eps, Dropout drop) {
  typedef Lay<G, WAVES> L;
  __shared__ Slots<WAVES> slots;
  clear(slots);
  const int span = L::span(), lane = L::lane(), sub_row = L::sub_row();
  const float inv_n = 1.0f / (float)cols;
  drop = with_key(drop);
  f32x8 gm[NC], bt[NC];
  int n[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = (c * span + lane) * 8;
    n[c] = max(min(cols - col, 8), 0);
    gm[c] = load_param<SHORT>(gamma, col, cols, n[c], 1.0f);
    bt[c] = load_param<SHORT>(beta, col, cols, n[c], 0.0f);
  }
  int turn = 0;
  // (every wave of a workgroup makes the same number of turns: the sums hold barriers)
  for (int64_t row0 = (int64_t)blockIdx.x * L::kRows; row0 < rows; row0 += (int64_t)gridDim.x * L::kRows) {
    // (rows and columns beyond the end: the last ones once more, not used)
    const int64_t row = min(row0 + sub_row, rows - 1);
    const bool ok = row0 + sub_row < rows;
    // The mask first: waves that draw while others load keep the memory busier than loads that run ahead of it, or a row ahead, do
    // (4110 rows of 1035 fp32: 15.6 us, 17.5 and 18.6).
    uint32_t keeps[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) keeps[c] = dropout_keeps(drop, mask_row_of(drop, (uint32_t)row), c * span + lane);
    Raw8<TX> raw_x[NC];
    Raw8<TR> raw_res[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      raw_x[c] = load_cols<SHORT>(x + row * cols, (c * span + lane) * 8, cols);
      if (RES) raw_res[c] = load_cols<SHORT>(res + row * cols, (c * span + lane) * 8, cols);
    }
    f32x8 v[NC];
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      f32x8 r = f32x8{};
      if (RES) r = used_cols<SHORT, TR>(raw_res[c], n[c]);
      v[c] = used_cols<SHORT, TX>(raw_x[c], n[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[c][e] = __builtin_fmaf(kept(v[c][e], keeps[c], e), drop.scale, r[e]);
        s[0] += e < n[c] ? v[c][e] : 0.0f;
      }
      if (ok && n[c]) store_cols(h + row * cols + (c * span + lane) * 8, v[c], n[c]);
    }
    row_sums<G, WAVES>(s, slots, turn);
    const float mean = s[0] * inv_n;
    float q[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[c][e] -= mean;
        // (selected, then squared: a lane without columns holds the row's last ones under another block's mask, and an infinity that is
        // dropped there times 0 is NaN)
        const float t = e < n[c] ? v[c][e] : 0.0f;
        q[0] = __builtin_fmaf(t, t, q[0]);
      }
    row_sums<G, WAVES>(q, slots, turn);
    const float rstd = rsqrtf(q[0] * inv_n + eps);
    if (!ok) continue;
    if (lane == 0) {
      if (mean_out) mean_out[row] = mean;
      if (rstd_out) rstd_out[row] = rstd;
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (!n[c]) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = __builtin_fmaf(v[c][e] * rstd, gm[c][e], bt[c][e]);
      store_cols(y + row * cols + (c * span + lane) * 8, v[c], n[c]);
    }
  }
}

// dy, dh, dx, dres may be null (a gradient that is not there is zero; one that is not wanted is not written).  With a stream of
// 16 bits h is formed again from x and the residual (null: none), else it is read and x and res are not.
template <typename TX, typename TR, int G, int WAVES, int NC, bool SHORT>
__global__ __launch_bounds__((Lay<G, WAVES>::kThreads)) void dropnorm_bwd_kernel(
    const TX* __restrict__ dy, const TR* __restrict__ dh, const TX* __restrict__ x, const TR* __restrict__ res,
    const TR* __restrict__ h, const float* __restrict__ mean, const float* __restrict__ rstd, NormParam gamma, TX* __restrict__ dx,
    TR* __restrict__ dres, float* __restrict__ part, int64_t rows, int cols, Dropout drop) {
  typedef Lay<G, WAVES> L;
  constexpr bool AGAIN = sizeof(TR) == 2;
  __shared__ Slots<WAVES> slots;
  clear(slots);
  const int span = L::span(), lane = L::lane(), sub_row = L::sub_row();
  const float inv_n = 1.0f / (float)cols;
  drop = with_key(drop);
  // (what is not there is read from where something is, and not used: loads without a branch wait for one another least)
  const TR* some = AGAIN ? (const TR*)x : h;
  const bool have_dy = dy, have_dh = dh, have_res = res;
  if (!have_dy) dy = (const TX*)some;
  if (!have_dh) dh = some;
  const TR* stream = AGAIN ? (have_res ? res : some) : h;
  f32x8 gm[NC], dg[NC], db[NC];
  int n[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = (c * span + lane) * 8;
    n[c] = max(min(cols - col, 8), 0);
    gm[c] = load_param<SHORT>(gamma, col, cols, n[c], 1.0f);
    dg[c] = db[c] = f32x8{};
  }
  int turn = 0;
  for (int64_t row0 = (int64_t)blockIdx.x * L::kRows; row0 < rows; row0 += (int64_t)gridDim.x * L::kRows) {
    const int64_t row = min(row0 + sub_row, rows - 1);
    const bool ok = row0 + sub_row < rows;
    Raw8<TX> raw_dy[NC], raw_x[NC];
    Raw8<TR> raw_dh[NC], raw_stream[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * span + lane) * 8;
      raw_stream[c] = load_cols<SHORT>(stream + row * cols, col, cols);
      if (AGAIN) raw_x[c] = load_cols<SHORT>(x + row * cols, col, cols);
      raw_dy[c] = load_cols<SHORT>(dy + row * cols, col, cols);
      raw_dh[c] = load_cols<SHORT>(dh + row * cols, col, cols);
    }
    const float mu = mean[row], rs = rstd[row];
    f32x8 xh[NC], d[NC];
    uint32_t keeps[NC];
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      keeps[c] = dropout_keeps(drop, mask_row_of(drop, (uint32_t)row), c * span + lane);
      // (columns and rows beyond the end, and all of them without dy: dy = 0 and a deviation of 0 keep them out of every sum)
      const int have = ok && have_dy ? n[c] : 0;
      xh[c] = used_cols<SHORT, TR>(raw_stream[c], n[c]);
      d[c] = used_cols<SHORT, TX>(raw_dy[c], n[c]);
      if (AGAIN) {
        const f32x8 u = used_cols<SHORT, TX>(raw_x[c], n[c]);
        if (!have_res) xh[c] = f32x8{};
#pragma unroll
        for (int e = 0; e < 8; ++e) xh[c][e] = __builtin_fmaf(kept(u[e], keeps[c], e), drop.scale, xh[c][e]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        xh[c][e] = e < have ? (xh[c][e] - mu) * rs : 0.0f;
        d[c][e] = e < have ? d[c][e] : 0.0f;
        const float g = gm[c][e] * d[c][e];
        s[0] += g;
        s[1] = __builtin_fmaf(g, xh[c][e], s[1]);
        dg[c][e] = __builtin_fmaf(d[c][e], xh[c][e], dg[c][e]);
        db[c][e] += d[c][e];
      }
    }
    row_sums<G, WAVES>(s, slots, turn);
    const float a = s[0] * inv_n, b = s[1] * inv_n;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (!ok || !n[c]) continue;
      const int64_t at = row * cols + (c * span + lane) * 8;
      const f32x8 up = used_cols<SHORT, TR>(raw_dh[c], n[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float of_h = have_dh ? up[e] : 0.0f;
        // (without dy dh alone: a zero times the rstd of a row that has none would be NaN)
        d[c][e] = have_dy ? __builtin_fmaf(gm[c][e] * d[c][e] - a - xh[c][e] * b, rs, of_h) : of_h;
      }
      if (dres) store_cols(dres + at, d[c], n[c]);
      if (dx) {
#pragma unroll
        for (int e = 0; e < 8; ++e) d[c][e] = kept(d[c][e], keeps[c], e) * drop.scale;
        store_cols(dx + at, d[c], n[c]);
      }
    }
  }
  if (!part) return;
  const int64_t parts = gridDim.x;
  float* out[2] = {part + (int64_t)blockIdx.x * cols, part + (parts + blockIdx.x) * cols};
  if constexpr (WAVES > 1) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * span + lane) * 8;
      if (!n[c]) continue;
      store_cols(out[0] + col, dg[c], n[c]);
      store_cols(out[1] + col, db[c], n[c]);
    }
  } else {
    // lanes that hold the same columns of other rows, then the four waves in order
    __shared__ float red[2][4][G * 8];
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float a = dg[0][e], b = db[0][e];
#pragma unroll
      for (int m = G; m < kWave; m <<= 1) {
        a += __shfl_xor(a, m, 64);
        b += __shfl_xor(b, m, 64);
      }
      if ((threadIdx.x & 63) < G) {
        red[0][wave][lane * 8 + e] = a;
        red[1][wave][lane * 8 + e] = b;
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * cols; i += 256) {
      const int which = i >= cols, col = i - which * cols;
      out[which][col] = (red[which][0][col] + red[which][1][col]) + (red[which][2][col] + red[which][3][col]);
    }
  }
}

constexpr int kDropnormCols = 16384;

int dropnorm_max_cols() { return kDropnormCols; }

// Waves of a compute unit that walk the forward pass (24 fit).  TB/s of 64 M bf16 elements with 16, 32 and 64 of them, and with as many
// as there are rows: rows of 128 4.9, 4.9, 5.0 and 5.6, of 512 5.1, 5.0, 4.9 and 5.6, but of 384 (lanes without columns) 4.8, 4.6, 4.9
// and 4.4, of 65 3.0, 3.0, 3.2 and 2.0; several waves to a row: of 2048 5.3, 5.0, 5.3 and 5.2, of 4096 5.5, 4.9, 5.2 and 5.2, of 5000
// with two, three, six workgroups and all 5.0, 4.3, 4.3 and 3.7.
template <int G, int WAVES> static int fwd_waves(int cols) { return WAVES > 1 ? 16 : cols == 8 * G ? 1 << 15 : 64; }

template <typename TX, typename TR>
int dropnorm_fwd(const TX* x, const TR* res, const void* gamma, const void* beta, int param_type, TX* y, TR* h, float* mean,
                 float* rstd, int64_t rows, int cols, float eps, const Dropout& drop, hipStream_t stream) {
  if (rows == 0) return 0;
  const int n_vec = (cols + 7) / 8;
#define PTX_DN_CASE(G, WAVES, NC, SHORT)                                                                              \
  if (PTX_DN_FITS(G, WAVES, NC, SHORT)) {                                                                             \
    const Walk w = walk<G, WAVES, NC>(rows, n_vec, fwd_waves<G, WAVES>(cols), 1);                                    \
    auto* kernel = res ? dropnorm_fwd_kernel<TX, TR, G, WAVES, NC, SHORT, true> : dropnorm_fwd_kernel<TX, TR, G, WAVES, NC, SHORT, false>; \
    kernel<<<dim3(w.groups), dim3(w.threads), 0, stream>>>(x, res, NormParam{gamma, param_type}, NormParam{beta, param_type}, y, h,    \
                                                           mean, rstd, rows, cols, eps, drop);                        \
    return 0;                                                                                                         \
  }
  PTX_DN_LAYOUTS(PTX_DN_CASE)
#undef PTX_DN_CASE
  return 1;
}

// Backward: waves per compute unit, and turns of a workgroup at the least, which leaves a row of partial sums each.  Us with the sums, the
// same tensors again and again, of 16384 rows of 2048 bf16: 16 waves 89, 12 85, 8 82, 4 106; of 700 rows of 2048 fp32 with at least one
// turn 16.5, two 14.7, four 13.4; but where a wave holds whole rows, of 6000 rows of 384 with one 13.2, two 13.2, four 15.4.
constexpr int kDropnormBwdWaves = 8;
template <int WAVES> constexpr int kDropnormBwdTurns = WAVES == 1 ? 1 : 4;

int64_t dropnorm_bwd_workspace_elems(int64_t rows, int cols) {
  if (rows <= 0 || cols <= 0) return 0;
  // (a row of partial sums per workgroup, for dgamma and dbeta: of two waves and one row, or of four, at the least)
  return 2 * std::min<int64_t>(rows, 256 * kDropnormBwdWaves / 2) * cols;
}

template <typename TX, typename TR>
int dropnorm_bwd(const TX* dy, const TR* dh, const TX* x, const TR* res, const TR* h, const float* mean, const float* rstd,
                 const void* gamma, int param_type, TX* dx, TR* dres, void* dgamma, void* dbeta, float* workspace, int64_t rows,
                 int cols, const Dropout& drop, hipStream_t stream) {
  float* part = dgamma || dbeta ? workspace : nullptr;
  const int n_vec = (cols + 7) / 8;
  int parts = 0;
  auto launch = [&]() {
#define PTX_DN_CASE(G, WAVES, NC, SHORT)                                                               \
  if (PTX_DN_FITS(G, WAVES, NC, SHORT)) {                                                              \
    const Walk w = walk<G, WAVES, NC>(rows, n_vec, kDropnormBwdWaves, kDropnormBwdTurns<WAVES>);        \
    parts = w.groups;                                                                                  \
    dropnorm_bwd_kernel<TX, TR, G, WAVES, NC, SHORT><<<dim3(parts), dim3(w.threads), 0, stream>>>(     \
        dy, dh, x, res, h, mean, rstd, NormParam{gamma, param_type}, dx, dres, part, rows, cols, drop); \
    return 0;                                                                                          \
  }
    PTX_DN_LAYOUTS(PTX_DN_CASE)
#undef PTX_DN_CASE
    return 1;
  };
  if (rows > 0 && launch()) return 1;
  // (no rows: the sums are zero, and written by the same kernel)
  if (dgamma || dbeta) column_sums(part, parts, cols, param_type, dgamma, dbeta, stream);
  return 0;
}

#define PTX_DN_TYPES(TX, TR)                                                                                                     \
  template int dropnorm_fwd(const TX*, const TR*, const void*, const void*, int, TX*, TR*, float*, float*, int64_t, int, float,  \
                            const Dropout&, hipStream_t);                                                                        \
  template int dropnorm_bwd(const TX*, const TR*, const TX*, const TR*, const TR*, const float*, const float*, const void*, int, \
                            TX*, TR*, void*, void*, float*, int64_t, int, const Dropout&, hipStream_t);
PTX_DN_TYPES(float, float)
PTX_DN_TYPES(bf16_t, bf16_t)
PTX_DN_TYPES(f16_t, f16_t)
PTX_DN_TYPES(bf16_t, float)
PTX_DN_TYPES(f16_t, float)

}  // namespace ptx
