// h = residual + x and y = RMSNorm(h), with their gradients, in one pass over the rows each; y in x's type or in 8 bits.
//
//   forward    h = res + x,  r = 1 / sqrt(mean(h^2) + eps),  y = h r gamma
//   backward   with g = gamma dy, xh = h r:  dres = dx = r (g - xh avg(g xh)) + dh,  dgamma = sum_rows dy xh
//
// Rows lie over lanes as in normrows.h, in registers.  The norm is that of the fp32 sum before it is rounded to h; the backward pass
// reads h where it is fp32 and forms it again from x and the residual where it has 16 bits (one 16-bit read, and dgamma keeps 24 bits).
// In 8 bits y goes from the fp32 registers into blocks of 128 columns, 16 lanes each, which find their largest magnitude among themselves
// (fp8.h): neither y in 16 bits nor a second launch.
// dgamma: column sums in registers over the rows a workgroup walks, one row of partial sums each, added in a fixed order.
// Bound by memory: 8192 rows of 4096 bf16 into 8 bits 45 us (5.2 TB/s); 147456 rows of 128 bf16 on fp32 forward 43, backward 49 us and 4
// for the sums (5.5 TB/s).
#include "fp8.h"
#include "kernels.h"
#include "normrows.h"

namespace ptx {

// TX: type of x and y; TR: of the residual and h.  RES: with a residual; without one h is x and is not written.
// QUANT: y as 8-bit values [rows][fp8_pitch(cols)] with scales [blocks][fp8_scale_pitch(rows)]; 16 lanes of a row or more.
template <typename TX, typename TR, int G, int WAVES, int NC, bool SHORT, bool RES, bool QUANT>
__global__ __launch_bounds__((Lay<G, WAVES>::kThreads)) void rmsnorm_fwd_kernel(
    const TX* __restrict__ x, const TR* __restrict__ res, NormParam gamma, void* __restrict__ y, float* __restrict__ scales,
    TR* __restrict__ h, float* __restrict__ rstd_out, int64_t rows, int cols, float eps) {
  typedef Lay<G, WAVES> L;
  __shared__ Slots<WAVES> slots;
  clear(slots);
  const int span = L::span(), lane = L::lane(), sub_row = L::sub_row();
  const float inv_n = 1.0f / (float)cols;
  const int pitch = (int)fp8_pitch(cols);
  f32x8 gm[NC];
  int n[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = (c * span + lane) * 8;
    n[c] = max(min(cols - col, 8), 0);
    gm[c] = load_param<SHORT>(gamma, col, cols, n[c], 1.0f);
  }
  int turn = 0;
  // (every wave of a workgroup makes the same number of turns: the sums hold barriers)
  for (int64_t row0 = (int64_t)blockIdx.x * L::kRows; row0 < rows; row0 += (int64_t)gridDim.x * L::kRows) {
    // (rows and columns beyond the end: the last ones once more, not used)
    const int64_t row = min(row0 + sub_row, rows - 1);
    const bool ok = row0 + sub_row < rows;
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
      v[c] = used_cols<SHORT, TX>(raw_x[c], n[c]);
      if (RES) v[c] += used_cols<SHORT, TR>(raw_res[c], n[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[c][e] = e < n[c] ? v[c][e] : 0.0f;
        s[0] = __builtin_fmaf(v[c][e], v[c][e], s[0]);
      }
      if (RES && ok && n[c]) store_cols(h + row * cols + (c * span + lane) * 8, v[c], n[c]);
    }
    row_sums<G, WAVES>(s, slots, turn);
    const float rstd = rsqrtf(s[0] * inv_n + eps);
    if (lane == 0 && ok && rstd_out) rstd_out[row] = rstd;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * span + lane) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = v[c][e] * rstd * gm[c][e];
      if constexpr (QUANT) {
        // (columns beyond the end are zeros, and a NaN among the others must not reach them: their block has its scale already)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[c][e] = e < n[c] ? v[c][e] : 0.0f;
        const Fp8Scale q = fp8_scale(largest16(magnitude(v[c])));
        if (ok && col < pitch) {
          *reinterpret_cast<u32x2_t*>((uint8_t*)y + row * pitch + col) = fp8_pack8(v[c], q.i);
          if ((lane & 15) == 0) scales[(int64_t)(col / kFp8Block) * fp8_scale_pitch(rows) + row] = q.s;
        }
      } else if (ok && n[c]) {
        store_cols((TX*)y + row * cols + col, v[c], n[c]);
      }
    }
  }
}

// dy, dh, dx, dres may be null (a gradient that is not there is zero; one that is not wanted is not written).  With a stream of
// 16 bits h is formed again from x and the residual (null: none), else h is read (x itself where there was no residual).
template <typename TX, typename TR, int G, int WAVES, int NC, bool SHORT>
__global__ __launch_bounds__((Lay<G, WAVES>::kThreads)) void rmsnorm_bwd_kernel(
    const TX* __restrict__ dy, const TR* __restrict__ dh, const TX* __restrict__ x, const TR* __restrict__ res,
    const TR* __restrict__ h, const float* __restrict__ rstd, NormParam gamma, TX* __restrict__ dx, TR* __restrict__ dres,
    float* __restrict__ part, int64_t rows, int cols) {
  typedef Lay<G, WAVES> L;
  constexpr bool AGAIN = sizeof(TR) == 2;
  __shared__ Slots<WAVES> slots;
  clear(slots);
  const int span = L::span(), lane = L::lane(), sub_row = L::sub_row();
  const float inv_n = 1.0f / (float)cols;
  // (what is not there is read from where something is, and not used: loads without a branch wait for one another least)
  const TR* some = AGAIN ? (const TR*)x : h;
  const bool have_dy = dy, have_dh = dh, have_res = res;
  if (!have_dy) dy = (const TX*)some;
  if (!have_dh) dh = some;
  const TR* stream = AGAIN ? (have_res ? res : some) : h;
  f32x8 gm[NC], dg[NC];
  int n[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = (c * span + lane) * 8;
    n[c] = max(min(cols - col, 8), 0);
    gm[c] = load_param<SHORT>(gamma, col, cols, n[c], 1.0f);
    dg[c] = f32x8{};
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
    const float rs = rstd[row];
    f32x8 xh[NC], d[NC];
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      // (columns and rows beyond the end, and all of them without dy: dy = 0 and xh = 0 keep them out of every sum)
      const int have = ok && have_dy ? n[c] : 0;
      xh[c] = used_cols<SHORT, TR>(raw_stream[c], n[c]);
      d[c] = used_cols<SHORT, TX>(raw_dy[c], n[c]);
      if (AGAIN) {
        const f32x8 u = used_cols<SHORT, TX>(raw_x[c], n[c]);
        if (have_res) xh[c] += u; else xh[c] = u;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        xh[c][e] = e < have ? xh[c][e] * rs : 0.0f;
        d[c][e] = e < have ? d[c][e] : 0.0f;
        s[0] = __builtin_fmaf(gm[c][e] * d[c][e], xh[c][e], s[0]);
        dg[c][e] = __builtin_fmaf(d[c][e], xh[c][e], dg[c][e]);
      }
    }
    row_sums<G, WAVES>(s, slots, turn);
    const float b = s[0] * inv_n;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (!ok || !n[c]) continue;
      const int64_t at = row * cols + (c * span + lane) * 8;
      const f32x8 up = used_cols<SHORT, TR>(raw_dh[c], n[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float of_h = have_dh ? up[e] : 0.0f;
        // (without dy dh alone: a zero times the rstd of a row that has none would be NaN)
        d[c][e] = have_dy ? __builtin_fmaf(gm[c][e] * d[c][e] - xh[c][e] * b, rs, of_h) : of_h;
      }
      if (dres) store_cols(dres + at, d[c], n[c]);
      if (dx) store_cols(dx + at, d[c], n[c]);
    }
  }
  if (!part) return;
  float* out = part + (int64_t)blockIdx.x * cols;
  if constexpr (WAVES > 1) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (n[c]) store_cols(out + (c * span + lane) * 8, dg[c], n[c]);
  } else {
    // lanes that hold the same columns of other rows, then the four waves in order
    __shared__ float red[4][G * 8];
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float a = dg[0][e];
#pragma unroll
      for (int m = G; m < kWave; m <<= 1) a += __shfl_xor(a, m, 64);
      if ((threadIdx.x & 63) < G) red[wave][lane * 8 + e] = a;
    }
    __syncthreads();
    for (int col = threadIdx.x; col < cols; col += 256) out[col] = (red[0][col] + red[1][col]) + (red[2][col] + red[3][col]);
  }
}

constexpr int kRmsnormCols = 16384;
int rmsnorm_max_cols() { return kRmsnormCols; }

// Waves of a compute unit that walk the rows: as in dropnorm.hip, whose passes these are but for the mask and the mean.
template <int G, int WAVES> static int rms_fwd_waves(int cols) { return WAVES > 1 ? 16 : cols == 8 * G ? 1 << 15 : 64; }
constexpr int kRmsBwdWaves = 8;
template <int WAVES> constexpr int kRmsBwdTurns = WAVES == 1 ? 1 : 4;

template <typename TX, typename TR>
int rmsnorm_fwd(const TX* x, const TR* res, const void* gamma, int param_type, void* y, float* scales, TR* h, float* rstd,
                int64_t rows, int cols, float eps, hipStream_t stream) {
  if (rows == 0) return 0;
  const int n_vec = (cols + 7) / 8;
  const bool quant = scales;
#define PTX_RMS_LAUNCH(G, WAVES, NC, SHORT, QUANT)                                                                              \
  {                                                                                                                             \
    const Walk w = walk<G, WAVES, NC>(rows, n_vec, rms_fwd_waves<G, WAVES>(cols), 1);                                           \
    auto* kernel = res ? rmsnorm_fwd_kernel<TX, TR, G, WAVES, NC, SHORT, true, QUANT> : rmsnorm_fwd_kernel<TX, TR, G, WAVES, NC, SHORT, false, QUANT>; \
    kernel<<<dim3(w.groups), dim3(w.threads), 0, stream>>>(x, res, NormParam{gamma, param_type}, y, scales, h, rstd, rows, cols, eps); \
    return 0;                                                                                                                   \
  }
#define PTX_RMS_CASE(G, WAVES, NC, SHORT) \
  if (!quant && PTX_DN_FITS(G, WAVES, NC, SHORT)) PTX_RMS_LAUNCH(G, WAVES, NC, SHORT, false)
#define PTX_RMS_QUANT_CASE(G, WAVES, NC, SHORT) \
  if (quant && PTX_DN_FITS(G, WAVES, NC, SHORT)) PTX_RMS_LAUNCH(G, WAVES, NC, SHORT, true)
  PTX_DN_LAYOUTS(PTX_RMS_CASE)
  // (a block of 128 columns has 16 lanes, also where a row has fewer columns)
  PTX_RMS_QUANT_CASE(16, 1, 1, true)
  PTX_RMS_QUANT_CASE(16, 1, 1, false)
  PTX_RMS_QUANT_CASE(32, 1, 1, false)
  PTX_RMS_QUANT_CASE(64, 1, 1, false)
  PTX_RMS_QUANT_CASE(64, 8, 1, false)
  PTX_RMS_QUANT_CASE(64, 16, 1, false)
  PTX_RMS_QUANT_CASE(64, 16, 2, false)
#undef PTX_RMS_CASE
#undef PTX_RMS_QUANT_CASE
#undef PTX_RMS_LAUNCH
  return 1;
}

int64_t rmsnorm_bwd_workspace_elems(int64_t rows, int cols) {
  if (rows <= 0 || cols <= 0) return 0;
  // (a row of partial sums per workgroup: of two waves and one row, or of four, at the least)
  return std::min<int64_t>(rows, 256 * kRmsBwdWaves / 2) * cols;
}

template <typename TX, typename TR>
int rmsnorm_bwd(const TX* dy, const TR* dh, const TX* x, const TR* res, const TR* h, const float* rstd, const void* gamma,
                int param_type, TX* dx, TR* dres, void* dgamma, float* workspace, int64_t rows, int cols, hipStream_t stream) {
  float* part = dgamma ? workspace : nullptr;
  const int n_vec = (cols + 7) / 8;
  int parts = 0;
  auto launch = [&]() {
#define PTX_RMS_CASE(G, WAVES, NC, SHORT)                                                               \
  if (PTX_DN_FITS(G, WAVES, NC, SHORT)) {                                                               \
    const Walk w = walk<G, WAVES, NC>(rows, n_vec, kRmsBwdWaves, kRmsBwdTurns<WAVES>);                   \
    parts = w.groups;                                                                                   \
    rmsnorm_bwd_kernel<TX, TR, G, WAVES, NC, SHORT><<<dim3(parts), dim3(w.threads), 0, stream>>>(       \
        dy, dh, x, res, h, rstd, NormParam{gamma, param_type}, dx, dres, part, rows, cols);             \
    return 0;                                                                                           \
  }
    PTX_DN_LAYOUTS(PTX_RMS_CASE)
#undef PTX_RMS_CASE
    return 1;
  };
  if (rows > 0 && launch()) return 1;
  // (no rows: the sums are zero, and written by the same kernel)
  if (dgamma) column_sums(part, parts, cols, param_type, dgamma, nullptr, stream);
  return 0;
}

#define PTX_RMS_TYPES(TX, TR)                                                                                                      \
  template int rmsnorm_fwd(const TX*, const TR*, const void*, int, void*, float*, TR*, float*, int64_t, int, float, hipStream_t);  \
  template int rmsnorm_bwd(const TX*, const TR*, const TX*, const TR*, const TR*, const float*, const void*, int, TX*, TR*, void*, \
                           float*, int64_t, int, hipStream_t);
PTX_RMS_TYPES(float, float)
PTX_RMS_TYPES(bf16_t, bf16_t)
PTX_RMS_TYPES(f16_t, f16_t)
PTX_RMS_TYPES(bf16_t, float)
PTX_RMS_TYPES(f16_t, float)

}  // namespace ptx
