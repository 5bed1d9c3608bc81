// A learned bias per head and bucket of relative position, and the gradient of its table.
//
//   out[b][h][i][j] = table[bucket(kpos[b][j] - qpos[b][i])][h]          dtable[u][h] = sum over the elements of bucket u
//
// Bound by the memory of the bias (written, and its gradient read); the buckets cost no memory.  A workgroup has a
// byte per distance in LDS (differences beyond max_distance stand for it), made from the distances at which the buckets start.
// A thread owns 8 neighbouring keys, kept as 32-bit offsets from a query of the workgroup's (whole 64-bit differences where some
// position is 2^30 or more away), and walks the rows of queries.  The differences that share a bucket are an interval (schemes of
// other buckets are refused at the C entry): where a thread's keys are consecutive numbers of one group and the first and the last of
// them fall into the same bucket, all do, and two look-ups stand for eight.  The rest is a look-up per element, shared by the heads.
//
// Gradient: sums of millions of elements in a few buckets.  Every lane has bins of its own in LDS, [bucket][lane], and adds to
// them in its program's order, without waiting for the sums: no two lanes ever meet in a bin (nor, a bin's bank being its lane's, in a
// bank), so nothing depends on scheduling.  Lanes, waves and workgroups are added in a fixed order at the end.  An addition takes
// about two cycles a lane, so a step of 8 queries by 8 keys makes few: one where all its differences share a bucket, one per difference
// (and not even that where neighbours share one) along the diagonal, one per element only where positions jump.
//
// Us of [2, 16, 2048, 2048] bf16, 32 buckets to a distance of 128: forward 59 (4.5 TB/s; 48 into memory that is in the caches); gradient
// with its sums 204 with an addition per element, 103 with one per step or query, 55 (4.9 TB/s) with those along the diagonal.
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
};

// How the elements lie over workgroups: units of queries by `chunk` vectors of 8 keys, a thread to a vector and `at_once` queries
// (by_head: heads) side by side, per_lane of them in a row.  A unit's queries are blocks of at_once * per_lane in a row, row_units
// blocks apart: the diagonal, whose neighbourhood takes the most look-ups, then passes through all waves of a workgroup in turn.
struct Tiling {
  int q_len, k_len, n_vec;
  int chunk, chunks;        // vectors of a unit, units along the keys
  int at_once, per_lane, block, row_units;      // block = at_once * per_lane
  int units;                // of all batches together
  int threads;
  bool by_head;
};

// min(|k - q|, most) with the sign of k - q, whatever the two are
__device__ __forceinline__ int clamped(int64_t k, int64_t q, int most) {
  const uint64_t n = k > q ? (uint64_t)k - (uint64_t)q : (uint64_t)q - (uint64_t)k;
  const int m = n < (uint64_t)most ? (int)n : most;
  return k > q ? m : -m;
}
// |a - base| < 2^30 (without a branch)
__device__ __forceinline__ bool near(int64_t a, int64_t base) {
  const uint64_t d = (uint64_t)a - (uint64_t)base;
  const bool wrapped = (int64_t)(((uint64_t)a ^ (uint64_t)base) & ((uint64_t)a ^ d)) < 0;
  return !wrapped & (d + (1u << 30) < (uint64_t)1 << 31);
}
__device__ __forceinline__ int offset(int64_t a, int64_t base) { return (int)(uint32_t)((uint64_t)a - (uint64_t)base); }   // (where near)

__host__ __device__ __forceinline__ int lut_bytes(const Buckets& bk) { return (2 * bk.max_distance + 16) & ~15; }
constexpr int kStartsBytes = 512;

// lut[max_distance + d]: the bucket of the difference d (-max_distance .. max_distance), by all threads of the workgroup (which
// have left starts[] in LDS; the caller's next barrier ends it)
__device__ __forceinline__ void fill_lut(const Buckets& bk, const uint16_t* starts, uint8_t* lut) {
  for (int n = threadIdx.x; n <= bk.max_distance; n += blockDim.x) {
    int lo = 0, hi = bk.side - 1;   // the last bucket that starts at n or before
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (starts[mid] <= n) lo = mid; else hi = mid - 1;
    }
    if (n > 0) lut[bk.max_distance + n] = (uint8_t)(bk.pos_base + bk.pos_step * lo);
    lut[bk.max_distance - n] = (uint8_t)(bk.neg_base + bk.neg_step * lo);
  }
}

__device__ __forceinline__ float table_at(const void* table, int type, int64_t i) {
  return type == PTX_F32 ? ((const float*)table)[i] : type == PTX_BF16 ? (float)((const bf16_t*)table)[i] : (float)((const f16_t*)table)[i];
}

constexpr int kUnitRows = 256;   // most queries of a unit

// A unit as a thread sees it.
struct Unit {
  int batch, rows;         // rows: queries of the unit; what is numbered 0 .. rows - 1 below
  int i0, gap;             // the first one; from the end of a block to the next one's first
  int j, n;                // keys j .. j + n - 1 (n = 0: none); the last vector of 8 or more keys ends with them,
  int again;               // and its first `again` keys are the vector's before
  int64_t p[8], g[8], base, gbase;      // positions and groups of the keys and of query i0, as loaded
  bool one_group, run;     // the keys are of one group; and have consecutive numbers
  bool narrow;             // (the whole workgroup's) offsets are good
  int off[8], goff[8];     // positions and groups of the keys, from those of query i0; the queries' own are in LDS
};

// Asks for what the thread's part of a unit is made from (and waits for nothing).
__device__ __forceinline__ void request_unit(Unit& k, const Tiling& t, const Axis& qa, const Axis& ka, int unit, int col) {
  const int rest = unit / t.row_units;
  k.batch = rest / t.chunks;
  const int phase = unit - rest * t.row_units, q_blocks = (t.q_len + t.block - 1) / t.block;
  const int blocks = (q_blocks - phase + t.row_units - 1) / t.row_units;      // (the last of all may be shorter, and is then the unit's last)
  k.i0 = phase * t.block;
  k.gap = (t.row_units - 1) * t.block;
  k.rows = blocks * t.block - max((phase + (blocks - 1) * t.row_units + 1) * t.block - t.q_len, 0);
  const int64_t qb = (int64_t)k.batch * t.q_len + k.i0, kb = (int64_t)k.batch * t.k_len;
  const int v = (rest - k.batch * t.chunks) * t.chunk + col;
  k.j = max(min(v * 8, t.k_len - 8), 0);
  k.n = v < t.n_vec ? min(t.k_len, 8) : 0;
  k.again = k.n ? v * 8 - k.j : 0;
  k.base = qa.first + k.i0;
  k.gbase = 0;
  if (qa.pos) k.base = qa.pos[qb];
  if (qa.group) k.gbase = qa.group[qb];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    k.p[e] = ka.first + min(k.j + e, t.k_len - 1);      // (fewer than 8 keys: the last one once more)
    k.g[e] = 0;
  }
  if (ka.pos)
#pragma unroll
    for (int e = 0; e < 8; ++e) k.p[e] = ka.pos[kb + min(k.j + e, t.k_len - 1)];
  if (ka.group)
#pragma unroll
    for (int e = 0; e < 8; ++e) k.g[e] = ka.group[kb + min(k.j + e, t.k_len - 1)];
}

// Every thread of the workgroup takes part; query_offsets are whole behind the barrier at the end.
__device__ __forceinline__ void enter_unit(Unit& k, const Tiling& t, const Axis& qa, const Axis& ka, int2* query_offsets) {
  const int64_t qb = (int64_t)k.batch * t.q_len + k.i0;
  bool fits = true;
  for (int l = threadIdx.x; l < k.rows; l += blockDim.x) {
    const int i = l + l / t.block * k.gap;
    const int64_t q = qa.pos ? qa.pos[qb + i] : qa.first + k.i0 + i, qg = qa.group ? qa.group[qb + i] : 0;
    fits = fits & near(q, k.base) & near(qg, k.gbase);
    query_offsets[l] = int2{offset(q, k.base), offset(qg, k.gbase)};
  }
  k.run = k.one_group = true;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    fits = fits & near(k.p[e], k.base) & near(k.g[e], k.gbase);
    k.off[e] = offset(k.p[e], k.base);
    k.goff[e] = offset(k.g[e], k.gbase);
    k.run = k.run & (k.off[e] == k.off[0] + e);
    k.one_group = k.one_group & (k.goff[e] == k.goff[0]);
  }
  k.run = k.run & k.one_group;
  k.narrow = !__syncthreads_or(!fits);
}

// Calls f(l, i) for the queries of a thread whose place among those side by side is `sub`: l in the unit, i from its first.
template <typename F> __device__ __forceinline__ void for_queries(const Unit& k, const Tiling& t, int sub, F f) {
  if (t.by_head) {      // (one block; all of it for every thread)
    for (int l = 0; l < k.rows; ++l) f(l, l);
    return;
  }
  for (int l0 = sub * t.per_lane, i0 = l0; l0 < k.rows; l0 += t.block, i0 += t.block + k.gap)
    for (int r = 0; r < t.per_lane && l0 + r < k.rows; ++r) f(l0 + r, i0 + r);
}

// Calls one(u) where all of the thread's keys have bucket u from the query, else each(u[8]).
template <typename One, typename Each>
__device__ __forceinline__ void at_query(const Buckets& bk, const uint8_t* mid, const Unit& k, int2 query, One one, Each each) {
  const int top = bk.max_distance;
  auto look = [&](int e) {
    const int u = mid[max(min(k.off[e] - query.x, top), -top)];
    return k.goff[e] == query.y ? u : bk.count;
  };
  int u[8];
  u[0] = look(0);
  u[7] = look(7);
  if (k.run && u[0] == u[7]) {
    one(u[0]);
  } else {
#pragma unroll
    for (int e = 1; e < 7; ++e) u[e] = look(e);
    each(u);
  }
}
// The same where the offsets do not hold the differences: from the positions themselves.  i: the query, from the unit's first.
template <typename Each>
__device__ __forceinline__ void at_far_query(const Buckets& bk, const uint8_t* mid, const Tiling& t, const Axis& qa, const Axis& ka, const Unit& k,
                                             int i, Each each) {
  const int64_t qi = (int64_t)k.batch * t.q_len + k.i0 + i, kb = (int64_t)k.batch * t.k_len;
  const int64_t q = qa.pos ? qa.pos[qi] : qa.first + k.i0 + i, g = qa.group ? qa.group[qi] : 0;
  int u[8];
  for (int e = 0; e < 8; ++e) {
    const int j = min(k.j + e, t.k_len - 1);
    u[e] = (ka.group ? ka.group[kb + j] : 0) == g ? (int)mid[clamped(ka.pos ? ka.pos[kb + j] : ka.first + j, q, bk.max_distance)] : bk.count;
  }
  each(u);
}

template <typename T>
__global__ __launch_bounds__(256) void relative_bias_fwd_kernel(Buckets bk, int n_buckets, const void* __restrict__ table, int table_type,
                                                                T* __restrict__ out, int heads, int heads_at_once, Tiling t, Axis qa, Axis ka) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  uint16_t* starts = (uint16_t*)lds;
  uint8_t* lut = (uint8_t*)lds + kStartsBytes;
  T* tab = (T*)(lds + kStartsBytes + lut_bytes(bk));
  __shared__ int2 queries[kUnitRows];
  const int h0 = blockIdx.y * heads_at_once, nh = min(heads_at_once, heads - h0);
  const int sub = threadIdx.x / t.chunk, col = threadIdx.x - sub * t.chunk;
  Unit k;
  request_unit(k, t, qa, ka, blockIdx.x, col);
  for (int i = threadIdx.x; i < bk.side; i += blockDim.x) starts[i] = bk.starts[i];
  for (int i = threadIdx.x; i < nh * n_buckets; i += blockDim.x) {
    const int u = i / nh, h = i - u * nh;
    tab[h * n_buckets + u] = from_f32<T>(table_at(table, table_type, (int64_t)u * heads + h0 + h));
  }
  __syncthreads();
  fill_lut(bk, starts, lut);
  const int64_t plane = (int64_t)t.q_len * t.k_len;
  const int head_step = t.by_head ? t.at_once : 1, first_head = t.by_head ? sub : 0;
  const uint8_t* mid = lut + bk.max_distance;
  for (int unit = blockIdx.x; unit < t.units; unit += gridDim.x) {
    if (unit != (int)blockIdx.x) {
      request_unit(k, t, qa, ka, unit, col);
      __syncthreads();      // (the queries of the unit before are done with)
    }
    enter_unit(k, t, qa, ka, queries);
    if (sub >= t.at_once || k.n == 0) continue;
    T* o = out + ((int64_t)k.batch * heads + h0) * plane + (int64_t)k.i0 * t.k_len + k.j;
    for_queries(k, t, sub, [&](int l, int i) {
      T* oi = o + (int64_t)i * t.k_len;
      auto one = [&](int u) {
        for (int h = first_head; h < nh; h += head_step) {
          const float v = (float)tab[h * n_buckets + u];
          store_cols(oi + h * plane, f32x8{v, v, v, v, v, v, v, v}, k.n);
        }
      };
      auto each = [&](const int(&u)[8]) {
        for (int h = first_head; h < nh; h += head_step) {
          f32x8 v;
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = (float)tab[h * n_buckets + u[e]];
          store_cols(oi + h * plane, v, k.n);
        }
      };
      if (k.narrow) at_query(bk, mid, k, queries[l], one, each);
      else at_far_query(bk, mid, t, qa, ka, k, i, each);
    });
  }
}

__device__ __forceinline__ void bin_add(float* bin, float v) {
  __hip_atomic_fetch_add((__attribute__((address_space(3))) float*)bin, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}

// Queries of a step in a lane, requested a step ahead: 128 bytes.  Read past the caches (NT): behind the forward pass, whose bias lies
// there still to be written to memory, reads that take its place wait for that (94 against 55 us at the size above).
template <typename T> constexpr int kAhead = sizeof(T) == 2 ? 8 : 4;

// bins: [waves][n_buckets][64].  SHORT: fewer than 8 keys.
template <typename T, bool SHORT>
__global__ __launch_bounds__(256) void relative_bias_bwd_kernel(Buckets bk, int n_buckets, const T* __restrict__ dout,
                                                                float* __restrict__ part, int heads, Tiling t, Axis qa, Axis ka) {
  constexpr int AHEAD = kAhead<T>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ int2 queries[kUnitRows];
  const int waves = blockDim.x >> 6, h = blockIdx.y;
  uint16_t* starts = (uint16_t*)lds;
  uint8_t* lut = (uint8_t*)lds + kStartsBytes;
  float* bins = (float*)(lds + kStartsBytes + lut_bytes(bk));
  const int sub = threadIdx.x / t.chunk, col = threadIdx.x - sub * t.chunk;
  Unit k;
  request_unit(k, t, qa, ka, blockIdx.x, col);
  for (int i = threadIdx.x; i < bk.side; i += blockDim.x) starts[i] = bk.starts[i];
  for (int i = threadIdx.x; i < waves * n_buckets * 16; i += blockDim.x) ((f32x4*)bins)[i] = f32x4{};
  __syncthreads();
  fill_lut(bk, starts, lut);
  float* own = bins + (threadIdx.x >> 6) * n_buckets * 64 + (threadIdx.x & 63);
  const uint8_t* mid = lut + bk.max_distance;
  const int top = bk.max_distance;
  for (int unit = blockIdx.x; unit < t.units; unit += gridDim.x) {
    if (unit != (int)blockIdx.x) {
      request_unit(k, t, qa, ka, unit, col);
      __syncthreads();      // (the queries of the unit before are done with)
    }
    enter_unit(k, t, qa, ka, queries);
    if (sub >= t.at_once || k.n == 0) continue;
    const T* d = dout + (((int64_t)k.batch * heads + h) * t.q_len + k.i0) * t.k_len;
    auto values = [&](const Raw8<T>& raw) {
      f32x8 v = widened<T>(raw);
      if (k.again)
#pragma unroll
        for (int e = 0; e < 7; ++e) v[e] = e < k.again ? 0.0f : v[e];
      return v;
    };
    auto sum = [](const f32x8& v) { return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7])); };
    auto each = [&](const f32x8& v, const int(&u)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) bin_add(own + u[e] * 64, v[e]);
    };
    if (!k.narrow) {
      for_queries(k, t, sub, [&](int, int i) {
        const f32x8 v = values(load_cols<SHORT, true>(d + (int64_t)i * t.k_len, k.j, t.k_len));
        at_far_query(bk, mid, t, qa, ka, k, i, [&](const int(&u)[8]) { each(v, u); });
      });
      continue;
    }
    // (a step: a block of queries, AHEAD or fewer of them in a lane; those that are not there: the last one once more, not used)
    auto load = [&](Raw8<T>(&raw)[AHEAD], int i, int n) {
#pragma unroll
      for (int r = 0; r < AHEAD; ++r) raw[r] = load_cols<SHORT, true>(d + (int64_t)(i + min(r, n - 1)) * t.k_len, k.j, t.k_len);
    };
    Raw8<T> raw[AHEAD], next[AHEAD];
    int l = sub * t.per_lane, i = l;
    if (l >= k.rows) continue;
    load(raw, i, min(t.per_lane, k.rows - l));
    for (; l < k.rows; l += t.block, i += t.block + k.gap) {
      const int n = min(t.per_lane, k.rows - l);
      if (l + t.block < k.rows) load(next, i + t.block + k.gap, min(t.per_lane, k.rows - l - t.block));
      int2 q[AHEAD];
#pragma unroll
      for (int r = 0; r < AHEAD; ++r) q[r] = queries[l + min(r, n - 1)];
      bool same = k.one_group, row = k.run;      // the queries are of one group; and consecutive, as are the keys
#pragma unroll
      for (int r = 1; r < AHEAD; ++r) {
        same &= q[r].y == q[0].y;
        row &= (q[r].x == q[0].x + r) | (r >= n);
      }
      row &= same;
      const bool apart = same & (k.goff[0] != q[0].y);
      auto bucket_of = [&](int e, int x) { return (int)mid[max(min(k.off[e] - x, top), -top)]; };
      // The step's differences lie between two of them where queries and keys are consecutive: where these share a bucket, the whole
      // step is one sum.  Else it is one per difference, AHEAD + 7 of them.
      int u0 = bucket_of(0, q[0].x + n - 1);
      const bool alike = row & (u0 == bucket_of(7, q[0].x));
      if (alike | apart) {
        float s = 0.0f;
#pragma unroll
        for (int r = 0; r < AHEAD; ++r) s += r < n ? sum(values(raw[r])) : 0.0f;
        bin_add(own + (apart ? bk.count : u0) * 64, s);
      } else if (row) {
        // s[j]: the sum over key - query = j - (AHEAD - 1) of their places in the step
        float s[AHEAD + 7];
#pragma unroll
        for (int j = 0; j < AHEAD + 7; ++j) s[j] = 0.0f;
#pragma unroll
        for (int r = 0; r < AHEAD; ++r) {
          const f32x8 v = values(raw[r]);
#pragma unroll
          for (int e = 0; e < 8; ++e) s[e - r + AHEAD - 1] += r < n ? v[e] : 0.0f;
        }
        int u[AHEAD + 7];
#pragma unroll
        for (int j = 0; j < AHEAD + 7; ++j) u[j] = bucket_of(0, q[0].x + AHEAD - 1 - j);
        float run = 0.0f;
#pragma unroll
        for (int j = 0; j < AHEAD + 7; ++j) {
          run += s[j];
          if (j == AHEAD + 6 || u[j] != u[j + 1]) {
            bin_add(own + u[j] * 64, run);
            run = 0.0f;
          }
        }
      } else {
#pragma unroll
        for (int r = 0; r < AHEAD; ++r) {
          if (r >= n) break;
          int u[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            u[e] = bucket_of(e, q[r].x);
            u[e] = k.goff[e] == q[r].y ? u[e] : bk.count;
          }
          each(values(raw[r]), u);
        }
      }
#pragma unroll
      for (int r = 0; r < AHEAD; ++r) raw[r] = next[r];
    }
  }
  __syncthreads();
  // sixteen lanes to a bucket, four of every wave's bins each
  for (int w = threadIdx.x; w < (n_buckets * 16 + 63) / 64 * 64; w += blockDim.x) {
    const int u = w >> 4;
    float s = 0.0f;
    if (u < n_buckets)
      for (int v = 0; v < waves; ++v) {
        const f32x4 b = ((const f32x4*)bins)[(v * n_buckets + u) * 16 + (w & 15)];
        s += (b[0] + b[1]) + (b[2] + b[3]);
      }
    s = lanes_sum<16>(s);
    if (u < n_buckets && (w & 15) == 0) part[((int64_t)blockIdx.x * n_buckets + u) * heads + h] = s;
  }
}

// most: vectors a unit may have (64 .. 256); threads: of a workgroup at most, at least `most`; groups: workgroups that share
// the units of one of `planes` heads (or head groups); ahead: queries of a step in a lane.
static Tiling tiling(int batch, int q_len, int k_len, int most, int threads, int64_t groups, int planes, int ahead) {
  Tiling t;
  t.q_len = q_len;
  t.k_len = k_len;
  t.n_vec = (k_len + 7) / 8;
  t.chunks = (t.n_vec + most - 1) / most;
  t.chunk = (t.n_vec + t.chunks - 1) / t.chunks;
  // as many waves as leave the fewest lanes without keys
  t.threads = threads;
  for (int n = 64; n <= threads; n += 64)
    if (n >= t.chunk && (int64_t)(n / t.chunk) * t.threads > (int64_t)(t.threads / t.chunk) * n) t.threads = n;
  t.at_once = t.threads / t.chunk;
  // a unit for every workgroup where there are rows for it: whole steps of them, as long as every compute unit has some; the blocks
  // of queries no longer than leaves every unit one
  const int64_t columns = (int64_t)batch * t.chunks, whole = (q_len + t.at_once * ahead - 1) / (t.at_once * ahead);
  t.row_units = (int)std::min<int64_t>({(q_len + t.at_once - 1) / t.at_once, std::max<int64_t>(1, groups / columns),
                                        std::max<int64_t>(whole, std::max<int64_t>(1, 256 / (columns * planes)))});
  const int share = (q_len + t.row_units - 1) / t.row_units;
  t.per_lane = std::max(1, std::min({ahead, kUnitRows / t.at_once, (share + t.at_once - 1) / t.at_once}));
  t.block = t.per_lane * t.at_once;
  const int q_blocks = (q_len + t.block - 1) / t.block;
  t.row_units = std::max(std::min(t.row_units, q_blocks), (q_blocks + kUnitRows / t.block - 1) / (kUnitRows / t.block));
  t.units = (int)(columns * t.row_units);
  t.by_head = false;
  return t;
}

// Fewer vectors than this (a query of a long context): units of 64, and the heads apart until every compute unit has two workgroups
// (16 heads, one query, 4001 keys: 7.9 us with units of up to 256, 5.5 now).
constexpr int64_t kFewVectors = 16384;

// Heads of a workgroup, which share its look-ups.  More write more planes of the bias at one offset at a time, and memory takes writes
// a power of two apart badly: us of [2, 16, 2048, 2048] bf16 into memory that is not in the caches with 16 heads 99, 8 84, 4 61, 2 65, 1 69.
constexpr int kHeadsAtOnce = 4;

template <typename T>
int relative_bias_fwd(const Buckets& bk, const void* table, int table_type, T* out, int batch, int heads, int q_len, int k_len,
                      const int64_t* q_pos, const int64_t* k_pos, int64_t q_first, int64_t k_first, const int64_t* q_group,
                      const int64_t* k_group, hipStream_t stream) {
  const int n_buckets = bk.count + (q_group != nullptr);
  int at_once = std::min(heads, kHeadsAtOnce), head_groups = (heads + at_once - 1) / at_once;
  const bool few = (int64_t)batch * q_len * ((k_len + 7) / 8) < kFewVectors;
  Tiling t = tiling(batch, q_len, k_len, few ? 64 : 256, 256, std::max(1, 2048 / head_groups), 8 * head_groups, 4);
  // (fewer rows than a workgroup holds side by side: heads take their place, as many as keep the threads busy and the table in 16 KB)
  t.by_head = q_len < t.at_once && heads > 1;
  if (t.by_head) {
    at_once = std::min({heads, std::max(t.at_once, kHeadsAtOnce), std::max(kHeadsAtOnce, 16384 / (n_buckets * (int)sizeof(T)))});
    head_groups = (heads + at_once - 1) / at_once;
  }
  while (at_once > (t.by_head ? t.at_once : 1) && (int64_t)t.units * head_groups < 512) {
    at_once = (at_once + 1) / 2;
    head_groups = (heads + at_once - 1) / at_once;
  }
  const int lds = kStartsBytes + lut_bytes(bk) + at_once * n_buckets * (int)sizeof(T);
  relative_bias_fwd_kernel<T><<<dim3(std::min(t.units, 1 << 20), head_groups), dim3(t.threads), lds, stream>>>(
      bk, n_buckets, table, table_type, out, heads, at_once, t, Axis{q_pos, q_group, q_first}, Axis{k_pos, k_group, k_first});
  return 0;
}

// Bins of a workgroup take at most this, so that a compute unit (160 KB) holds two workgroups at least, beside the queries (2 KB) and a
// look-up of two bytes per distance: up to distances of some 2800.  Beyond, one of many bins may be alone.
constexpr int kBinBytes = 72 * 1024;
static int bwd_threads(int n_buckets) { return 64 * std::min(4, std::max(1, kBinBytes / (n_buckets * 256))); }
// Workgroups of one head, a row of partial sums each: as many as the machine's LDS holds at a time (four waves to a SIMD at most) of all
// heads together.  Counted by their bins alone, as the workspace is: behind look-ups of thousands of distances some wait for others to end.
static int bwd_slices(int heads, int n_buckets) {
  const int per_cu = std::max(1, std::min(1024 / bwd_threads(n_buckets), 150 * 1024 / (bwd_threads(n_buckets) * 4 * n_buckets)));
  return std::max(1, 256 * per_cu / heads);
}

int64_t relative_bias_bwd_workspace_elems(int heads, int n_buckets) {
  return heads <= 0 || n_buckets <= 0 ? 0 : (int64_t)bwd_slices(heads, n_buckets) * heads * n_buckets;
}

template <typename T>
int relative_bias_bwd(const Buckets& bk, const T* dout, void* dtable, int table_type, float* workspace, int batch, int heads, int q_len,
                      int k_len, const int64_t* q_pos, const int64_t* k_pos, int64_t q_first, int64_t k_first, const int64_t* q_group,
                      const int64_t* k_group, hipStream_t stream) {
  const int n_buckets = bk.count + (q_group != nullptr);
  int slices = 0;
  if (batch > 0 && q_len > 0 && k_len > 0) {
    const int most = bwd_threads(n_buckets);
    const Tiling t = tiling(batch, q_len, k_len, most, most, bwd_slices(heads, n_buckets), heads, kAhead<T>);
    slices = std::min(t.units, bwd_slices(heads, n_buckets));
    const int lds = kStartsBytes + lut_bytes(bk) + t.threads * 4 * n_buckets;
    const Axis qa{q_pos, q_group, q_first}, ka{k_pos, k_group, k_first};
    if (k_len < 8)
      relative_bias_bwd_kernel<T, true><<<dim3(slices, heads), dim3(t.threads), lds, stream>>>(bk, n_buckets, dout, workspace, heads, t, qa, ka);
    else
      relative_bias_bwd_kernel<T, false><<<dim3(slices, heads), dim3(t.threads), lds, stream>>>(bk, n_buckets, dout, workspace, heads, t, qa, ka);
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
