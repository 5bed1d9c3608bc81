// Rows of norms over the lanes of a wave or the waves of a workgroup (dropnorm.hip, rmsnorm.hip): where a row's blocks of 8 columns
// lie, its sums, its parameters, and how many workgroups walk the rows.
#pragma once
#include <algorithm>

#include "dropout.h"

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

// Sums over the lanes of a row: within G lanes, or (WAVES > 1) over the waves of a workgroup through one of the slots (a slot is
// used again two exchanges later, when every wave has passed the barrier of the exchange between).
template <int WAVES> struct Slots {
  f32x4 sum[2][2][WAVES > 1 ? WAVES / 4 : 1];   // [exchange][value][wave]
};
// (waves that a workgroup does not have count as 0)
template <int WAVES> __device__ __forceinline__ void clear(Slots<WAVES>& s) {
  if (WAVES > 1 && threadIdx.x < 4 * WAVES && (int)(threadIdx.x % WAVES) >= (int)(blockDim.x >> 6)) ((float*)s.sum)[threadIdx.x] = 0.0f;
}
template <int G, int WAVES, int N> __device__ __forceinline__ void row_sums(float (&v)[N], Slots<WAVES>& slots, int& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lanes_sum<G>(v[i]);
  if constexpr (WAVES > 1) {
    f32x4(*s)[WAVES / 4] = slots.sum[turn];
    turn ^= 1;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) ((float*)s[i])[threadIdx.x >> 6] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float t = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES / 4; ++w) t += (s[i][w][0] + s[i][w][1]) + (s[i][w][2] + s[i][w][3]);
      v[i] = t;
    }
  }
}

// WAVES = 1: four waves to a workgroup, 64 / G rows to a wave.  Else a row to a workgroup of up to WAVES waves.
template <int G, int WAVES> struct Lay {
  static constexpr int kThreads = WAVES == 1 ? 256 : 64 * WAVES;
  static constexpr int kRows = WAVES == 1 ? 256 / G : 1;       // rows a workgroup holds at once
  static __device__ __forceinline__ int span() { return WAVES == 1 ? G : (int)blockDim.x; }      // lanes of a row
  static __device__ __forceinline__ int lane() { return WAVES == 1 ? threadIdx.x % G : threadIdx.x; }
  static __device__ __forceinline__ int sub_row() { return WAVES == 1 ? threadIdx.x / G : 0; }
};

// The first layout that holds a row's blocks of 8 columns: (lanes, waves at most, blocks per lane, fewer than 8 columns).
#define PTX_DN_LAYOUTS(X) \
  X(1, 1, 1, true) X(1, 1, 1, false) X(2, 1, 1, false) X(4, 1, 1, false) X(8, 1, 1, false) X(16, 1, 1, false) X(32, 1, 1, false) \
  X(64, 1, 1, false) X(64, 8, 1, false) X(64, 16, 1, false) X(64, 16, 2, false)
// A launch's shape: workgroups of one row in the fewest waves that hold it, or of four waves of rows, which walk the rows: the same number
// of them for each of the 256 compute units, the first that holds `waves` waves, or as many fewer as leave each `turns` turns (rounded
// down, so that some make one more; but one per compute unit).  (With 256 waves / w of them, whatever that leaves over, some units walk two shares one after the other: 64 M bf16
// elements in rows of 2800 backward 4.0 TB/s, with 2 for each 4.9.)
struct Walk {
  int groups, threads;
};
template <int G, int WAVES, int NC> static Walk walk(int64_t rows, int n_vec, int waves, int turns) {
  Walk w;
  w.threads = WAVES == 1 ? 256 : (n_vec + 64 * NC - 1) / (64 * NC) * 64;
  const int64_t batches = (rows + Lay<G, WAVES>::kRows - 1) / Lay<G, WAVES>::kRows;
  const int own = w.threads / 64, per_cu = (waves + own - 1) / own;
  w.groups = (int)std::min<int64_t>({batches, std::max<int64_t>(256, batches / turns), (int64_t)256 * per_cu});
  return w;
}
#define PTX_DN_FITS(G, WAVES, NC, SHORT) (SHORT ? cols < 8 : n_vec <= G * WAVES * NC)

}  // namespace ptx
