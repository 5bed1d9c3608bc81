// A learned bias per head and bucket of relative position, and the gradient of its table.
//
//   out[b][h][i][j] = table[bucket(kpos[b][j] - qpos[b][i])][h]          dtable[u][h] = sum over the elements of bucket u
//
// Bound by the memory of the bias (written, and its gradient read); the buckets cost no memory.  A workgroup has a
// byte per distance in LDS (differences beyond max_distance stand for it), made from the distances at which the buckets start, so that
// an element costs one look-up for its bucket, shared by the heads, and one for its value.
//
// Gradient: sums of millions of elements in a few buckets.  Every lane has bins of its own in LDS, [bucket][lane], and adds to
// them in its program's order: no two lanes ever meet in a bin (nor, a bin's bank being its lane's, in a bank), so nothing
// depends on scheduling.  Lanes, waves and workgroups are added in a fixed order at the end.
#include <algorithm>

#include "../../include/protenix_amd.h"
#include "dropout.h"
#include "kernels.h"

namespace ptx {

typedef ptx_relative_buckets Buckets;

struct Axis {
  const int64_t* pos;     // [batch][n], or null: first + index
  const int64_t* group;   // [batch][n], or null
  int64_t first;
  __device__ __forceinline__ int64_t at(int64_t base, int i) const { return pos ? pos[base + i] : first + i; }
};

// min(|k - q|, most) with the sign of k - q, whatever the two are
__device__ __forceinline__ int clamped(int64_t k, int64_t q, int most) {
  const uint64_t n = k > q ? (uint64_t)k - (uint64_t)q : (uint64_t)q - (uint64_t)k;
  const int m = n < (uint64_t)most ? (int)n : most;
  return k > q ? m : -m;
}

// lut[max_distance + d]: the bucket of the difference d
__device__ __forceinline__ void fill_lut(const Buckets& bk, uint8_t* lut, int threads) {
  for (int i = threadIdx.x; i <= 2 * bk.max_distance; i += threads) {
    const int d = i - bk.max_distance, n = d < 0 ? -d : d;
    int lo = 0, hi = bk.side - 1;   // the last bucket that starts at n or before
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (bk.starts[mid] <= n) lo = mid; else hi = mid - 1;
    }
    lut[i] = (uint8_t)(d > 0 ? bk.pos_base + bk.pos_step * lo : bk.neg_base + bk.neg_step * lo);
  }
}

__device__ __forceinline__ float table_at(const void* table, int type, int64_t i) {
  return type == PTX_F32 ? ((const float*)table)[i] : type == PTX_BF16 ? (float)((const bf16_t*)table)[i] : (float)((const f16_t*)table)[i];
}

template <typename T>
__global__ __launch_bounds__(256) void relative_bias_fwd_kernel(Buckets bk, int n_buckets, const void* __restrict__ table, int table_type,
                                                                T* __restrict__ out, int heads, int heads_at_once, int q_len, int k_len,
                                                                int n_vec, int chunk, int chunks, Axis qa, Axis ka) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  uint8_t* lut = (uint8_t*)lds;
  T* tab = (T*)(lds + ((2 * bk.max_distance + 16) & ~15));
  const int batch = blockIdx.x / chunks;
  const int h0 = blockIdx.y * heads_at_once, nh = min(heads_at_once, heads - h0);
  fill_lut(bk, lut, 256);
  for (int i = threadIdx.x; i < nh * n_buckets; i += 256) {
    const int h = i / n_buckets, u = i - h * n_buckets;
    tab[i] = from_f32<T>(table_at(table, table_type, (int64_t)u * heads + h0 + h));
  }
  __syncthreads();
  const int64_t pairs = (int64_t)q_len * n_vec, end = min((int64_t)(blockIdx.x % chunks + 1) * chunk, pairs);
  const int64_t qb = (int64_t)batch * q_len, kb = (int64_t)batch * k_len;
  for (int64_t p = (int64_t)(blockIdx.x % chunks) * chunk + threadIdx.x; p < end; p += 256) {
    const int i = (int)(p / n_vec), j = (int)(p - (int64_t)i * n_vec) * 8, n = min(k_len - j, 8);
    const int64_t q = qa.at(qb, i), qg = qa.group ? qa.group[qb + i] : 0;
    int bucket[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int je = min(j + e, k_len - 1);
      bucket[e] = lut[bk.max_distance + clamped(ka.at(kb, je), q, bk.max_distance)];
      if (ka.group && ka.group[kb + je] != qg) bucket[e] = bk.count;
    }
    T* o = out + (((int64_t)batch * heads + h0) * q_len + i) * k_len + j;
    for (int h = 0; h < nh; ++h, o += (int64_t)q_len * k_len) {
      f32x8 v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (float)tab[h * n_buckets + bucket[e]];
      store_cols(o, v, n);
    }
  }
}

// bins: [waves][n_buckets][64]
template <typename T>
__global__ __launch_bounds__(256) void relative_bias_bwd_kernel(Buckets bk, int n_buckets, const T* __restrict__ dout,
                                                                float* __restrict__ part, int heads, int q_len, int k_len, int n_vec,
                                                                int64_t pairs, int64_t chunk, Axis qa, Axis ka) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int waves = blockDim.x >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, h = blockIdx.y;
  uint8_t* lut = (uint8_t*)lds;
  float* bins = (float*)(lds + ((2 * bk.max_distance + 16) & ~15));
  fill_lut(bk, lut, blockDim.x);
  for (int i = threadIdx.x; i < waves * n_buckets * 64; i += blockDim.x) bins[i] = 0.0f;
  __syncthreads();
  float* own = bins + wave * n_buckets * 64 + lane;
  const int64_t per_batch = (int64_t)q_len * n_vec, end = min((blockIdx.x + 1) * chunk, pairs);
  for (int64_t p = blockIdx.x * chunk + threadIdx.x; p < end; p += blockDim.x) {
    const int64_t batch = p / per_batch, r = p - batch * per_batch;
    const int i = (int)(r / n_vec), j = (int)(r - (int64_t)i * n_vec) * 8, n = min(k_len - j, 8);
    const f32x8 v = load_cols(dout + ((batch * heads + h) * q_len + i) * k_len + j, n);
    const int64_t qb = batch * q_len, kb = batch * k_len;
    const int64_t q = qa.at(qb, i), qg = qa.group ? qa.group[qb + i] : 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (e >= n) continue;
      int u = lut[bk.max_distance + clamped(ka.at(kb, j + e), q, bk.max_distance)];
      if (ka.group && ka.group[kb + j + e] != qg) u = bk.count;
      own[u * 64] += v[e];
    }
  }
  __syncthreads();
  for (int u = wave; u < n_buckets; u += waves) {
    float s = 0.0f;
    for (int w = 0; w < waves; ++w) s += bins[(w * n_buckets + u) * 64 + lane];
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) s += __shfl_xor(s, m, 64);
    if (lane == 0) part[((int64_t)blockIdx.x * n_buckets + u) * heads + h] = s;
  }
}

static int lut_bytes(const Buckets& bk) { return (2 * bk.max_distance + 16) & ~15; }

template <typename T>
int relative_bias_fwd(const Buckets& bk, const void* table, int table_type, T* out, int batch, int heads, int q_len, int k_len,
                      const int64_t* q_pos, const int64_t* k_pos, int64_t q_first, int64_t k_first, const int64_t* q_group,
                      const int64_t* k_group, hipStream_t stream) {
  const int n_buckets = bk.count + (q_group != nullptr), n_vec = (k_len + 7) / 8;
  const int at_once = std::min(heads, std::max(1, 16384 / (n_buckets * (int)sizeof(T))));
  const int64_t pairs = (int64_t)q_len * n_vec;
  const int chunk = 1024;
  const int64_t chunks = (pairs + chunk - 1) / chunk;
  if (chunks * batch > 0x7fffffff) return 1;
  const int lds = lut_bytes(bk) + at_once * n_buckets * (int)sizeof(T);
  relative_bias_fwd_kernel<T><<<dim3((unsigned)(chunks * batch), (heads + at_once - 1) / at_once), dim3(256), lds, stream>>>(
      bk, n_buckets, table, table_type, out, heads, at_once, q_len, k_len, n_vec, chunk, (int)chunks, Axis{q_pos, q_group, q_first},
      Axis{k_pos, k_group, k_first});
  return 0;
}

// Slices of the elements, one row of partial sums each.
constexpr int kRelBwdGroups = 1024;   // workgroups of all heads together
static int bwd_slices(int heads) { return std::max(1, kRelBwdGroups / heads); }

int64_t relative_bias_bwd_workspace_elems(int heads, int n_buckets) {
  return heads <= 0 || n_buckets <= 0 ? 0 : (int64_t)bwd_slices(heads) * heads * n_buckets;
}

template <typename T>
int relative_bias_bwd(const Buckets& bk, const T* dout, void* dtable, int table_type, float* workspace, int batch, int heads, int q_len,
                      int k_len, const int64_t* q_pos, const int64_t* k_pos, int64_t q_first, int64_t k_first, const int64_t* q_group,
                      const int64_t* k_group, hipStream_t stream) {
  const int n_buckets = bk.count + (q_group != nullptr), n_vec = (k_len + 7) / 8;
  const int64_t pairs = (int64_t)batch * q_len * n_vec;
  int slices = 0;
  if (pairs > 0) {
    const int waves = n_buckets <= 64 ? 4 : n_buckets <= 128 ? 2 : 1, threads = 64 * waves;
    const int64_t chunk = ((pairs + bwd_slices(heads) - 1) / bwd_slices(heads) + threads - 1) / threads * threads;
    slices = (int)((pairs + chunk - 1) / chunk);
    relative_bias_bwd_kernel<T><<<dim3(slices, heads), dim3(threads), lut_bytes(bk) + waves * n_buckets * 256, stream>>>(
        bk, n_buckets, dout, workspace, heads, q_len, k_len, n_vec, pairs, chunk, Axis{q_pos, q_group, q_first},
        Axis{k_pos, k_group, k_first});
  }
  column_sums(workspace, slices, n_buckets * heads, table_type, dtable, nullptr, stream);
  return 0;
}

#define PTX_REL_TYPES(T)                                                                                                          \
  template int relative_bias_fwd(const Buckets&, const void*, int, T*, int, int, int, int, const int64_t*, const int64_t*,        \
                                 int64_t, int64_t, const int64_t*, const int64_t*, hipStream_t);                                  \
  template int relative_bias_bwd(const Buckets&, const T*, void*, int, float*, int, int, int, int, const int64_t*,                \
                                 const int64_t*, int64_t, int64_t, const int64_t*, const int64_t*, hipStream_t);
PTX_REL_TYPES(float)
PTX_REL_TYPES(bf16_t)
PTX_REL_TYPES(f16_t)

}  // namespace ptx
