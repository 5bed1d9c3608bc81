// h = residual + dropout(x) and y = LayerNorm(h), with their gradients, in one pass over the rows each.
//
//   forward    h = res + m x,  y = (h - mean) rstd gamma + beta             m = 1 / (1 - p) or 0 (dropout.h)
//   backward   with g = gamma dy, xh = (h - mean) rstd:
//              dres = rstd (g - avg(g) - xh avg(g xh)) + dh,  dx = m dres,
//              dgamma = sum_rows dy xh,  dbeta = sum_rows dy
//
// A row lies over its lanes in registers, one block of 8 columns per lane (= one draw of the mask, see dropout.h), two or
// four blocks for rows of more than 8192 columns: G lanes of a wave for up to 512 columns, WPR waves of a workgroup beyond, whose sums
// meet in LDS.  Statistics are fp32 and taken in two passes over the registers, from the sum before it is rounded to h.
// The backward pass takes h from memory where it is fp32, and forms it again from x and the residual where the stream
// has 16 bits: xh of a rounded h would leave dgamma with an error of 2^-9 instead of 2^-24, for the sake of one
// 16-bit read.  dgamma and dbeta: column sums in registers over the rows a workgroup walks, one row of fp32 partial sums
// per workgroup, added in a fixed order by layernorm_bwd_reduce (no atomics).
#include <algorithm>

#include "dropout.h"
#include "kernels.h"

namespace ptx {

// gamma / beta have a type of their own (fp32 parameters beside 16-bit rows): told apart at run time, these are read
// once per workgroup.
struct NormParam {
  const void* p;
  int type;   // ptx_dtype
};
constexpr int kF32 = 0, kBF16 = 1;

template <bool SHORT> __device__ __forceinline__ f32x8 load_param(NormParam w, int col, int cols, int n, float absent) {
  if (n == 0) return f32x8{};
  if (!w.p) return f32x8{absent, absent, absent, absent, absent, absent, absent, absent};
  if (w.type == kF32) return used_cols<SHORT, float>(load_cols<SHORT>((const float*)w.p, col, cols), n);
  if (w.type == kBF16) return used_cols<SHORT, bf16_t>(load_cols<SHORT>((const bf16_t*)w.p, col, cols), n);
  return used_cols<SHORT, f16_t>(load_cols<SHORT>((const f16_t*)w.p, col, cols), n);
}

template <int G> __device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int m = G / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}

// Sums over the lanes of a row: within G lanes, or over the WPR waves of a workgroup through one of the slots (a slot is
// used again two exchanges later, when every wave has passed the barrier of the exchange between).
template <int G, int WPR, int N> __device__ __forceinline__ void row_sums(float (&v)[N], float (*slots)[16][2], int& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lanes_sum<G>(v[i]);
  if constexpr (WPR > 1) {
    float(*s)[2] = slots[turn];
    turn ^= 1;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) s[threadIdx.x >> 6][i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float t = 0.0f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) t += s[w][i];
      v[i] = t;
    }
  }
}

template <int G, int WPR> struct Lay {
  static constexpr int kThreads = WPR == 1 ? 256 : 64 * WPR;
  static constexpr int kRows = WPR == 1 ? 256 / G : 1;       // rows a workgroup holds at once
  static constexpr int kSpan = WPR == 1 ? G : 64 * WPR;      // lanes of a row
};

__device__ __forceinline__ uint32_t mask_row_of(const Dropout& d, uint32_t row) {
  if (d.shared == 1) return row;
  const uint32_t o = row / (d.shared * d.inner);
  return o * d.inner + row % d.inner;
}

// TX: type of x and y; TR: of the residual and h.  SHORT: fewer than 8 columns.
template <typename TX, typename TR, int G, int WPR, int NC, bool SHORT>
__global__ __launch_bounds__((Lay<G, WPR>::kThreads)) void dropnorm_fwd_kernel(
    const TX* __restrict__ x, const TR* __restrict__ res, NormParam gamma, NormParam beta, TX* __restrict__ y, TR* __restrict__ h,
    float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t rows, int cols, float eps, Dropout drop) {
  typedef Lay<G, WPR> L;
  __shared__ float slots[2][16][2];
  const int lane = threadIdx.x % L::kSpan, sub_row = threadIdx.x / L::kSpan;
  const float inv_n = 1.0f / (float)cols;
  const bool masked = (drop.hi | drop.lo) != 0;
  drop = with_key(drop);
  struct Raw {
    Raw8<TX> x[NC];
    Raw8<TR> res[NC];
  };
  // (rows and columns beyond the end: the last ones once more, not used)
  auto load = [&](Raw& raw, int64_t row) {
    const int64_t at = min(row, rows - 1) * cols;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      raw.x[c] = load_cols<SHORT>(x + at, (c * L::kSpan + lane) * 8, cols);
      raw.res[c] = Raw8<TR>{};
      if (res) raw.res[c] = load_cols<SHORT>(res + at, (c * L::kSpan + lane) * 8, cols);
    }
  };
  const int64_t step = (int64_t)gridDim.x * L::kRows;
  int64_t row0 = (int64_t)blockIdx.x * L::kRows;
  Raw cur;
  load(cur, row0 + sub_row);
  f32x8 gm[NC], bt[NC];
  int n[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = (c * L::kSpan + lane) * 8;
    n[c] = max(min(cols - col, 8), 0);
    gm[c] = load_param<SHORT>(gamma, col, cols, n[c], 1.0f);
    bt[c] = load_param<SHORT>(beta, col, cols, n[c], 0.0f);
  }
  int turn = 0;
  // (every wave of a workgroup makes the same number of turns: the sums hold barriers)
  for (; row0 < rows; row0 += step) {
    const int64_t row = row0 + sub_row;
    const bool ok = row < rows;
    Raw next;
    if (row0 + step < rows) load(next, row + step);
    f32x8 v[NC];
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int k = c * L::kSpan + lane;
      float factor[8];
      if (masked) dropout_factors(drop, mask_row_of(drop, (uint32_t)min(row, rows - 1)), k, factor);
      const f32x8 r = used_cols<SHORT, TR>(cur.res[c], n[c]);
      v[c] = used_cols<SHORT, TX>(cur.x[c], n[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[c][e] = masked ? dropped_add(v[c][e], factor[e], r[e]) : v[c][e] + r[e];
        s[0] += e < n[c] ? v[c][e] : 0.0f;
      }
      if (ok && n[c]) store_cols(h + row * cols + k * 8, v[c], n[c]);
    }
    row_sums<G, WPR>(s, slots, turn);
    const float mean = s[0] * inv_n;
    float q[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[c][e] -= mean;
        q[0] = __builtin_fmaf(v[c][e], e < n[c] ? v[c][e] : 0.0f, q[0]);
      }
    row_sums<G, WPR>(q, slots, turn);
    const float rstd = rsqrtf(q[0] * inv_n + eps);
    if (ok) {
      if (lane == 0) {
        if (mean_out) mean_out[row] = mean;
        if (rstd_out) rstd_out[row] = rstd;
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (!n[c]) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[c][e] = __builtin_fmaf(v[c][e] * rstd, gm[c][e], bt[c][e]);
        store_cols(y + row * cols + (c * L::kSpan + lane) * 8, v[c], n[c]);
      }
    }
    cur = next;
  }
}

// dy, dh, dx, dres may be null (a gradient that is not there is zero; one that is not wanted is not written); h is null
// where the sum is to be formed again from x and the residual (null: none).
template <typename TX, typename TR, int G, int WPR, int NC, bool SHORT>
__global__ __launch_bounds__((Lay<G, WPR>::kThreads)) void dropnorm_bwd_kernel(
    const TX* __restrict__ dy, const TR* __restrict__ dh, const TX* __restrict__ x, const TR* __restrict__ res,
    const TR* __restrict__ h, const float* __restrict__ mean, const float* __restrict__ rstd, NormParam gamma, TX* __restrict__ dx,
    TR* __restrict__ dres, float* __restrict__ part, int64_t rows, int cols, Dropout drop) {
  typedef Lay<G, WPR> L;
  __shared__ float slots[2][16][2];
  const int lane = threadIdx.x % L::kSpan, sub_row = threadIdx.x / L::kSpan;
  const float inv_n = 1.0f / (float)cols;
  drop = with_key(drop);
  const bool masked = (drop.hi | drop.lo) != 0, again = h == nullptr;
  const TR* stream = again ? res : h;
  struct Raw {
    Raw8<TX> dy[NC], x[NC];
    Raw8<TR> dh[NC], stream[NC];
    float mean, rstd;
  };
  auto load = [&](Raw& raw, int64_t row) {
    row = min(row, rows - 1);
    const int64_t at = row * cols;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * L::kSpan + lane) * 8;
      raw.dy[c] = raw.x[c] = Raw8<TX>{};
      raw.dh[c] = raw.stream[c] = Raw8<TR>{};
      if (dy) raw.dy[c] = load_cols<SHORT>(dy + at, col, cols);
      if (dh) raw.dh[c] = load_cols<SHORT>(dh + at, col, cols);
      if (again) raw.x[c] = load_cols<SHORT>(x + at, col, cols);
      if (stream) raw.stream[c] = load_cols<SHORT>(stream + at, col, cols);
    }
    raw.mean = mean[row];
    raw.rstd = rstd[row];
  };
  const int64_t step = (int64_t)gridDim.x * L::kRows;
  int64_t row0 = (int64_t)blockIdx.x * L::kRows;
  Raw cur;
  load(cur, row0 + sub_row);
  f32x8 gm[NC], dg[NC], db[NC];
  int n[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = (c * L::kSpan + lane) * 8;
    n[c] = max(min(cols - col, 8), 0);
    gm[c] = load_param<SHORT>(gamma, col, cols, n[c], 1.0f);
    dg[c] = db[c] = f32x8{};
  }
  int turn = 0;
  for (; row0 < rows; row0 += step) {
    const int64_t row = row0 + sub_row;
    const bool ok = row < rows;
    Raw next;
    if (row0 + step < rows) load(next, row + step);
    f32x8 xh[NC], d[NC];
    float factor[NC][8];
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int k = c * L::kSpan + lane;
      if (masked) dropout_factors(drop, mask_row_of(drop, (uint32_t)min(row, rows - 1)), k, factor[c]);
      // (columns and rows beyond the end: dy = 0 and a deviation of 0 keep them out of every sum)
      const int have = ok ? n[c] : 0;
      xh[c] = used_cols<SHORT, TR>(cur.stream[c], n[c]);
      d[c] = used_cols<SHORT, TX>(cur.dy[c], n[c]);
      if (again) {
        const f32x8 u = used_cols<SHORT, TX>(cur.x[c], n[c]);
#pragma unroll
        for (int e = 0; e < 8; ++e) xh[c][e] = masked ? dropped_add(u[e], factor[c][e], xh[c][e]) : u[e] + xh[c][e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        xh[c][e] = e < have ? (xh[c][e] - cur.mean) * cur.rstd : 0.0f;
        d[c][e] = e < have ? d[c][e] : 0.0f;
        const float g = gm[c][e] * d[c][e];
        s[0] += g;
        s[1] = __builtin_fmaf(g, xh[c][e], s[1]);
        dg[c][e] = __builtin_fmaf(d[c][e], xh[c][e], dg[c][e]);
        db[c][e] += d[c][e];
      }
    }
    row_sums<G, WPR>(s, slots, turn);
    const float a = s[0] * inv_n, b = s[1] * inv_n;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (!ok || !n[c]) continue;
      const int64_t at = row * cols + (c * L::kSpan + lane) * 8;
      const f32x8 up = used_cols<SHORT, TR>(cur.dh[c], n[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) d[c][e] = __builtin_fmaf(gm[c][e] * d[c][e] - a - xh[c][e] * b, cur.rstd, up[e]);
      if (dres) store_cols(dres + at, d[c], n[c]);
      if (dx) {
        if (masked) {
#pragma unroll
          for (int e = 0; e < 8; ++e) d[c][e] = dropped(d[c][e], factor[c][e]);
        }
        store_cols(dx + at, d[c], n[c]);
      }
    }
    cur = next;
  }
  if (!part) return;
  const int64_t parts = gridDim.x;
  float* out[2] = {part + (int64_t)blockIdx.x * cols, part + (parts + blockIdx.x) * cols};
  if constexpr (WPR > 1) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * L::kSpan + lane) * 8;
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

// The first layout that holds a row's blocks of 8 columns: (lanes, waves, blocks per lane, fewer than 8 columns).
#define PTX_DN_LAYOUTS(X) \
  X(8, 1, 1, true) X(8, 1, 1, false) X(16, 1, 1, false) X(32, 1, 1, false) X(64, 1, 1, false) X(64, 2, 1, false) X(64, 4, 1, false) \
  X(64, 8, 1, false) X(64, 16, 1, false) X(64, 16, 2, false) X(64, 16, 4, false)
constexpr int kDropnormCols = 32768;

int dropnorm_max_cols() { return kDropnormCols; }

// Workgroups that walk the rows: rows of up to 512 columns a wave or less each, 8 workgroups of four waves per compute unit; longer ones
// as many waves.
template <int G, int WPR> static int walkers(int64_t rows, int waves_per_cu) {
  const int64_t most = std::max(1, 256 * waves_per_cu / (Lay<G, WPR>::kThreads / 64));
  return (int)std::min<int64_t>((rows + Lay<G, WPR>::kRows - 1) / Lay<G, WPR>::kRows, most);
}

template <typename TX, typename TR>
int dropnorm_fwd(const TX* x, const TR* res, const void* gamma, const void* beta, int param_type, TX* y, TR* h, float* mean,
                 float* rstd, int64_t rows, int cols, float eps, const Dropout& drop, hipStream_t stream) {
  if (rows == 0) return 0;
  const int n_vec = (cols + 7) / 8;
#define PTX_DN_CASE(G, WPR, NC, SHORT)                                                                                              \
  if (SHORT ? cols < 8 : n_vec <= Lay<G, WPR>::kSpan * (NC)) {                                                                                  \
    dropnorm_fwd_kernel<TX, TR, G, WPR, NC, SHORT><<<dim3(walkers<G, WPR>(rows, 32)), dim3(Lay<G, WPR>::kThreads), 0, stream>>>(    \
        x, res, NormParam{gamma, param_type}, NormParam{beta, param_type}, y, h, mean, rstd, rows, cols, eps, drop);                 \
    return 0;                                                                                                                \
  }
  PTX_DN_LAYOUTS(PTX_DN_CASE)
#undef PTX_DN_CASE
  return 1;
}

constexpr int kDropnormBwdWaves = 16;   // waves per compute unit = 4096 at most in all

int64_t dropnorm_bwd_workspace_elems(int64_t rows, int cols) {
  if (rows <= 0 || cols <= 0) return 0;
  // (one row of partial sums per workgroup, for dgamma and dbeta: four waves to a workgroup at the least, or one row
  // of more than 512 columns in two)
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
#define PTX_DN_CASE(G, WPR, NC, SHORT)                                                                                               \
  if (SHORT ? cols < 8 : n_vec <= Lay<G, WPR>::kSpan * (NC)) {                                                                                   \
    parts = walkers<G, WPR>(rows, kDropnormBwdWaves);                                                                         \
    dropnorm_bwd_kernel<TX, TR, G, WPR, NC, SHORT><<<dim3(parts), dim3(Lay<G, WPR>::kThreads), 0, stream>>>(                         \
        dy, dh, x, res, h, mean, rstd, NormParam{gamma, param_type}, dx, dres, part, rows, cols, drop);                           \
    return 0;                                                                                                                 \
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
