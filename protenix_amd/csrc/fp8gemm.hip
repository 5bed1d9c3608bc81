// Products of matrices in 8-bit blocks (fp8.h):
//   out[m][n] = sum over blocks of  sa[block][m] sb[..] sum_{k in block} a[m][k] b[n][k]   (+ bias[n])
// a's scales are per row and 128 columns, b's the same (ROWB) or per 128 x 128.
//
// One MFMA of 16 x 16 x 128 covers exactly one block, so its 16 x 16 results, in fp32, are multiplied by the block's scales and added to
// the accumulators by the vector pipe: 4 fused multiply-adds per lane (16 cycles) beside an MFMA's 32, which run at the same time.
// b is the MFMA's first operand, a its second: a lane then holds results of one m, and one product of scales serves all its n of a block.
//
// The 8-bit MFMA does not sum in full fp32: it aligns the products of 8 neighbouring k to the largest of them and cuts what lies below
// 2^-13 of it (measured; over groups it is fp32).  16-bit results take that.  On normal data it is 1.4e-5 of a result, far below their rounding
// (2^-9 and 2^-12 at most); it is bounded by the largest products and not by the result: where two of each 8 stand out ten times and cancel,
// results in fp16 are off by 2.4e-4 of their norm (2.1e-4 of it the rounding), in bf16 as without; a hundred times, by 2.5e-3
// and 3.0e-3 (bf16's rounding alone 1.7e-3).  Results in fp32 do not take it: for those the values, which f16 holds exactly, are widened in registers
// and multiplied by the f16 MFMA, whose sums are fp32 (1e-8 on the same data), at half of the 8-bit rate.
#include <algorithm>
#include <type_traits>

#include "fp8.h"
#include "dropout.h"
#include "kernels.h"

namespace ptx {

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

// A lane's 32 values of 16 rows x 128: pieces of 16 bytes from 16 q and 64 + 16 q on (q = lane / 16), as the MFMA takes them.
template <bool WIDE> struct Fragment {
  i32x8 v;
  Fragment() = default;
  __device__ __forceinline__ Fragment(const i32x4& lo, const i32x4& hi) : v(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)) {}
};
template <> struct Fragment<true> {
  f16x8 v[4];
  Fragment() = default;
  __device__ __forceinline__ Fragment(const i32x4& lo, const i32x4& hi) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const int x = s < 2 ? lo[2 * s + w] : hi[2 * s + w - 4];
        const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, true);
        v[s][4 * w] = a[0];
        v[s][4 * w + 1] = a[1];
        v[s][4 * w + 2] = b[0];
        v[s][4 * w + 3] = b[1];
      }
    }
  }
};
__device__ __forceinline__ f32x4 mma128(const Fragment<false>& a, const Fragment<false>& b) {
  // (scales of 1: the instruction without them, its sum starting from 0)
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, f32x4{}, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma128(const Fragment<true>& a, const Fragment<true>& b) {
  f32x4 d = f32x4{};
#pragma unroll
  for (int s = 0; s < 4; ++s) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v[s], b.v[s], d, 0, 0, 0);
  return d;
}

struct Fp8Args {
  const uint8_t* a;
  const float* sa;
  const uint8_t* b;
  const float* sb;
  const void* bias;
  int bias_type;
  void* out;
  int m, n;
  int blocks;                // of 128 along k
  int tiles_m, tiles_n;
  int splits;                // of the blocks; more than one: out is fp32 [splits][m][n] without bias
};

// A block's result v (0, or 2^-18 to 2^25 in magnitude) times its two scales x and y, whose product may lie beyond fp32 where the result does not:
// v x y = (v 2^half) rest, with half of the exponent of x y on either side.  rest is x y of 24 bits; where x y is a normal number both factors are
// too, and so v x y has the bits that it has with x y formed first; elsewhere they are wherever the result is neither 0 nor infinite.  The tile
// kernels form x y first, one for many v, and take this only for tiles with a scale outside 2^-63 .. 2^63.  Scales of 2^-126 and
// below, those of blocks of zeros, do not count there (zeros in rows or tokens cost nothing more): x y may then be off by 2^-150, and the
// block's result, of values below 448 2^-126, by 2^-125.
struct Fp8Factors {
  int half;
  float rest;
};
__device__ __forceinline__ Fp8Factors factors(float x, float y) {
  const int e = __builtin_amdgcn_frexp_expf(x) + __builtin_amdgcn_frexp_expf(y), half = e >> 1;
  return {half, __builtin_amdgcn_ldexpf(__builtin_amdgcn_frexp_mantf(x) * __builtin_amdgcn_frexp_mantf(y), e - half)};
}
__device__ __forceinline__ float param_at(const void* p, int type, int64_t i) {
  return type == 0 ? ((const float*)p)[i] : type == 1 ? (float)((const bf16_t*)p)[i] : (float)((const f16_t*)p)[i];
}

// The bias at columns col(u, r) (beyond the last one: that one once more), 0 without one.  The type is asked for once: a branch at each value has
// a wait behind each load (1035 x 1000 x 777 with a bias in bf16 7.6 -> 6.0 us).
template <int N, typename T, typename Col> __device__ __forceinline__ void load_bias_as(f32x4 (&out)[N], const T* bias, int cols, Col col) {
  T v[N][4];
#pragma unroll
  for (int u = 0; u < N; ++u)
#pragma unroll
    for (int r = 0; r < 4; ++r) v[u][r] = bias[min(col(u, r), cols - 1)];
#pragma unroll
  for (int u = 0; u < N; ++u) {
#pragma unroll
    for (int r = 0; r < 4; ++r) out[u][r] = (float)v[u][r];
    // (the wait for the loads belongs here: behind the branch it would be one for all loads of what comes next, without a bias too, and what no
    // store uses would be waited for in every block of the next tile)
    asm volatile("" : "+v"(out[u]));
  }
}
template <int N, typename Col> __device__ __forceinline__ void load_bias(f32x4 (&out)[N], const void* bias, int type, int cols, Col col) {
  if (!bias) {
#pragma unroll
    for (int u = 0; u < N; ++u) out[u] = f32x4{};
  } else if (type == 0) {
    load_bias_as(out, (const float*)bias, cols, col);
  } else if (type == 1) {
    load_bias_as(out, (const bf16_t*)bias, cols, col);
  } else {
    load_bias_as(out, (const f16_t*)bias, cols, col);
  }
}

// Four values of one row from column n on (bias and rounding), as many as there are.
template <typename O> __device__ __forceinline__ void store4(O* row, int n, int cols, const f32x4& v) {
  typedef O O4 __attribute__((ext_vector_type(4), aligned(sizeof(O))));
  if (n + 4 <= cols) {
    *reinterpret_cast<O4*>(row + n) = O4{(O)v[0], (O)v[1], (O)v[2], (O)v[3]};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < cols) row[n + e] = (O)v[e];
  }
}

// The tile of a workgroup: ids go round the 8 XCDs; each gets one run of tiles, in columns of 8 tiles of m, so that what its workgroups
// read at a time stays in its L2.
__device__ __forceinline__ void tile_of(uint32_t id, int tiles_m, int tiles_n, int& tm, int& tn) {
  const uint32_t total = (uint32_t)tiles_m * tiles_n, xcd = id & 7, per = total / 8, more = total % 8;
  const uint32_t t = xcd * per + min(xcd, more) + (id >> 3);
  const uint32_t band = 8u * tiles_n, first = t / band, in = t - first * band, high = min(8u, tiles_m - first * 8);
  tm = (int)(first * 8 + in % high);
  tn = (int)(in / high);
}

// Tiles of TM x TN, WM x WN waves of TM / WM x 64 each, and WK such groups of waves that share the blocks of k and add their sums in LDS.
// Both operands' 128 columns of a block go to LDS (direct loads into a ring of NB buffers: NB - 1 blocks are on their way or there
// while one is multiplied), rows of 128 bytes whose 16-byte pieces lie at place piece ^ (row % 8): no bank conflicts.  Rows of b lie in LDS so
// that what a wave stores at a time are runs of 64 bytes: with 16-bit results row 16 u + i of 64 holds
// n = 32 (u / 2) + 8 (i / 4) + 4 (u % 2) + i % 4, and a lane's results of two MFMAs are 8 neighbours; with fp32 ones n = 16 u + i
// (147456 x 128 x 512 in fp32 112 -> 84 us).
//
// 256 x 256, which takes what is large: 256 x 256 is the most that 256 registers a lane hold the sums of (128) with two waves per SIMD, whose
// vector work then hides behind each other's MFMAs, and two buffers of both operands fill the LDS.  8192^3 in 477 us (2.30 PFLOP/s),
// 8192 x 4096 x 8192 in 250 (2.20), with scales per row of both operands (twice the vector work) 546 and 282.  The MFMAs were
// busy 60 % of the time at 1.91 GHz, when it did not look at the range of the scales yet (457 us); a product without scales per block reaches 84 % at 1.67 GHz (375 us), so that what bounds
// both is power.  Without its loads that kernel took 382 us, with loads from the L1 408, from the L2 430; without the scales' vector work 421.
// Of short k: 147456 x 128 x 512 42 us among other passes (39 by itself), in fp32 77 (4.1 TB/s; a fill in the same tiles 5.5): loads 7, products 4 and 4.5 rounds
// of tiles that take 5.
template <int TM, int TN, int WM, int WN, int NB, bool PAIRS> struct Fp8Tile {
  static constexpr int W = WM * WN, MT = TM / WM / 16;
  static constexpr int kSa = 0, kSb = 1024, kB = 2048, kA = kB + TN * 128, kStage = kA + TM * 128;
  static constexpr int PER = (TM + TN) / 8 / W;      // loads of 1 KB per wave and block
  static constexpr int PER_B = TN / 8 / W;
  // The row of b (of 64) that a group s of 8 rows of LDS has for its row e, and how many rows lie between a wave's first load and its load j.
  static __device__ __forceinline__ int b_row(int s, int e) {
    return PAIRS ? 32 * (s >> 2) + 8 * (2 * (s & 1) + (e >> 2)) + 4 * ((s >> 1) & 1) + (e & 3) : 8 * s + e;
  }
  static constexpr int b_rows(int j) { return W == 4 ? 32 * (j & 1) + 64 * (j >> 1) : 8 * W * j; }
  // the first of the 4 columns that lane group q has of MFMA u
  static __device__ __forceinline__ int col(int u, int q) { return PAIRS ? 32 * (u >> 1) + 8 * q + 4 * (u & 1) : 16 * u + 4 * q; }
  static_assert((W == 4 || W % 8 == 0) && TN == 64 * WN && (TN / 8) % W == 0 && (TM / 8) % W == 0 && TM <= 256 && TN <= 256, "whole loads per wave");
};

// (two workgroups of small tiles to a compute unit where their buffers leave the room: 4 waves per SIMD)
template <int TM, int TN, int WM, int WN, int WK, int NB, bool ROWB, typename O>
__global__ __launch_bounds__(64 * WM * WN * WK, TM == 64 && NB == 2 ? 4 : 1) void fp8_tile_product(Fp8Args p) {
  typedef Fp8Tile<TM, TN, WM, WN, NB, sizeof(O) == 2> C;
  __shared__ __align__(16) uint8_t lds_all[WK * NB * C::kStage];
  const int lane = threadIdx.x & 63, wave_of_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = WK > 1 ? wave_of_all / C::W : 0, wave = wave_of_all - group * C::W;
  uint8_t* lds = lds_all + group * NB * C::kStage;
  const int wm = wave / WN, wn = wave % WN, i = lane & 15, q = lane >> 4;
  const int split = blockIdx.y;
  // this group's blocks first .. last - 1; all groups of waves make `steps` steps, those with a block less none in the last one
  const int begin = (int)((int64_t)p.blocks * split / p.splits), count = (int)((int64_t)p.blocks * (split + 1) / p.splits) - begin;
  const int first = begin + count * group / WK, last = begin + count * (group + 1) / WK, steps = (count + WK - 1) / WK;
  const uint32_t pitch = (uint32_t)p.blocks * kFp8Block;
  // What this lane loads: its row of the first load and the last row there is, as offsets (a later load's row lies a number of rows
  // behind; rows beyond the end are the last one once more).
  const int e = lane >> 3;
  const uint32_t piece = (uint32_t)((lane & 7) ^ e) * 16;
  uint32_t first_b = (uint32_t)(64 * (wave >> 3) + C::b_row(wave & 7, e)) * pitch + piece;
  uint32_t first_a = (uint32_t)(8 * wave + e) * pitch + piece;
  const int64_t sp_a = fp8_scale_pitch(p.m), sp_b = fp8_scale_pitch(p.n);
  // where a tile's operands lie
  struct Place {
    int m0, n0;
    uint64_t a, b, sa, sb;
    uint32_t last_a, last_b, off_sa, off_sb;
  };
  auto place = [&](uint32_t tile) {
    Place l;
    int tm, tn;
    tile_of(tile, p.tiles_m, p.tiles_n, tm, tn);
    l.m0 = tm * TM;
    l.n0 = tn * TN;
    l.a = uniform64((uint64_t)(p.a + (int64_t)l.m0 * pitch));
    l.b = uniform64((uint64_t)(p.b + (int64_t)l.n0 * pitch));
    l.last_a = (uint32_t)(min(TM, p.m - l.m0) - 1) * pitch + piece;
    l.last_b = (uint32_t)(min(TN, p.n - l.n0) - 1) * pitch + piece;
    l.sa = uniform64((uint64_t)(p.sa + l.m0));
    l.off_sa = 4u * (uint32_t)min((int64_t)4 * lane, sp_a - 4 - l.m0);
    // b's scales: of this tile's rows, or of the waves' 64 columns each (lane l: wave l of a row of them)
    const int block_n = ROWB ? 0 : l.n0 / kFp8Block;
    l.sb = uniform64((uint64_t)(p.sb + (ROWB ? l.n0 : (int64_t)block_n * p.blocks)));
    l.off_sb = ROWB ? 4u * (uint32_t)min((int64_t)4 * lane, sp_b - 4 - l.n0)
                    : 4u * (uint32_t)(min(l.n0 + 64 * min(lane, WN - 1), p.n - 1) / kFp8Block - block_n) * (uint32_t)p.blocks;
    return l;
  };
  uint32_t tile = blockIdx.x;
  Place from = place(tile);      // what is loaded next belongs to this one
  const uint32_t lds0 = lds_address(lds);
  // one of a wave's PER + 1 loads of a block: a KB of an operand each, and the scales
  auto load = [&](int step, int buf, int j) {
    const uint32_t to = lds0 + buf * C::kStage;
    const int block = WK > 1 ? max(min(first + step, last - 1), first) : first + step;
    const uint64_t k = (uint64_t)block * kFp8Block;
    if (j < C::PER_B) {
      asm volatile("" : "+v"(first_b));      // (the offset is formed here: kept, they would take as many registers as there are loads)
      load_to_lds16_s<0>(from.b + k, min(first_b + C::b_rows(j) * pitch, from.last_b), to + C::kB + 1024 * (wave + C::W * j));
    } else if (j < C::PER) {
      asm volatile("" : "+v"(first_a));
      const int r = j - C::PER_B;
      load_to_lds16_s<0>(from.a + k, min(first_a + 8 * C::W * r * pitch, from.last_a), to + C::kA + 1024 * (wave + C::W * r));
    } else if (wave == 0) {
      load_to_lds16_s<0>(from.sa + 4 * (uint64_t)block * sp_a, from.off_sa, to + C::kSa);
    } else if (wave == C::W - 1) {
      if (ROWB) load_to_lds16_s<0>(from.sb + 4 * (uint64_t)block * sp_b, from.off_sb, to + C::kSb);
      else load_to_lds4_s(from.sb + 4 * (uint64_t)block, from.off_sb, to + C::kSb);
    }
  };
  f32x4 acc[C::MT][4];
#pragma unroll
  for (int t = 0; t < C::MT; ++t)
#pragma unroll
    for (int u = 0; u < 4; ++u) acc[t][u] = f32x4{};
  const int at = i * 128 + ((q ^ (i & 7)) << 4), row0 = wm * (TM / WM);
  typedef Fragment<sizeof(O) == 4> F;
  auto fragment = [&](const uint8_t* tile) {      // 16 rows of 128 bytes
    return F(*reinterpret_cast<const i32x4*>(tile + at), *reinterpret_cast<const i32x4*>(tile + (at ^ 64)));
  };
  struct B {
    F f[4];
  };
  auto read_b = [&](const uint8_t* st) {
    const uint8_t* tb = st + C::kB + 64 * wn * 128;
    return B{{fragment(tb), fragment(tb + 16 * 128), fragment(tb + 32 * 128), fragment(tb + 48 * 128)}};
  };
  auto read_a = [&](const uint8_t* st, int t) { return fragment(st + C::kA + (row0 + 16 * t) * 128); };
  // The smallest (but for 2^-126 and below) and the largest of the scales of this wave's rows and columns in a tile: where they lie within
  // 2^-63 .. 2^63 every product of two is a normal number, else far_apart() looks closer and far_products() forms the tile again.  As whole numbers: 2^-126 and
  // below are the largest of those less 2^-126 and a bit, negative ones the largest of all.  Each block looks at all of them once, a lane at
  // those at at_sa and at_sb of a stage (rows and columns that are not there have any scales: the last one's once more).  8192^3 471 -> 485 us,
  // with scales per row 548 -> 555, tiles of 64 x 64 0 - 3 %; a compare and a branch at each row tile in place of this: 3 and 5 %.
  constexpr int SA = (16 * C::MT + kWave - 1) / kWave;
  constexpr uint32_t LEAST = 0x00800001u;
  int at_sa[SA], at_sb = 0;
  uint32_t low = ~0u, high = 0;
  auto begin_scales = [&]() {
#pragma unroll
    for (int h = 0; h < SA; ++h)
      at_sa[h] = C::kSa + 4 * min(row0 + (C::MT == 1 ? i : min(64 * h + lane, 16 * C::MT - 1)), p.m - from.m0 - 1);
    if (ROWB) at_sb = C::kSb + 4 * min(64 * wn + lane, p.n - from.n0 - 1);
    low = ~0u;
    high = 0;
  };
  begin_scales();
  // (the scale of b by way of LDS too: a load that the compiler knows of would wait for all of these)
  auto read_scale_b = [&](const uint8_t* st) { return ROWB ? 1.0f : *reinterpret_cast<const float*>(st + C::kSb + 4 * wn); };
  auto read_s = [&](const uint8_t* st, int t) { return *reinterpret_cast<const float*>(st + (C::MT == 1 ? at_sa[0] : C::kSa + 4 * (row0 + 16 * t + i))); };
  // A wave's stages overlap: the loads of a later block are spread over this one's first row tiles, a row tile's fragments are read while
  // the one before is multiplied, and its results scaled and added while the next one is.  The waves meet once a block, in front of its
  // last row tile - all reads of its buffer have returned then -, under whose multiplications the next block's first fragments are read.
  // Before the next block is read: this wave's loads of it have landed (all but those of the `after` youngest blocks), and all waves' have.
  auto meet = [&](auto after) {
    if (wave == 0 || wave == C::W - 1)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(after.value * (C::PER + 1)) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(after.value * C::PER) : "memory");
  };
  constexpr std::integral_constant<int, 0> none{};
#pragma unroll
  for (int k = 0; k < NB - 1; ++k)
    if (k == 0 || k < steps)
#pragma unroll
      for (int j = 0; j <= C::PER; ++j) load(k, k, j);
  if (NB - 1 <= steps) meet(std::integral_constant<int, NB - 2>{});
  else meet(none);
  B fb = read_b(lds);
  F fa = read_a(lds, 0);
  float scale_b = read_scale_b(lds), sa = read_s(lds, 0), s_before = 0.0f;
  f32x4 d[4] = {f32x4{}, f32x4{}, f32x4{}, f32x4{}};
  int buf = 0;
  // Whether the smallest or the largest scales of these rows and columns have such a product (of magnitudes, without infinities and NaN): gradients
  // of 1e-22 in a few rows beside ordinary weights do not, and the tile stands (8192 x 4096 x 8192 with one such row in 128: 256 -> 301 us, formed
  // again 943).
  auto far_apart = [&](int m0, int n0) {
    uint32_t low_a = ~0u, high_a = 0, low_b = ~0u, high_b = 0;
    auto look = [&](float v, uint32_t& lo, uint32_t& hi) {
      const uint32_t x = __float_as_uint(v) & 0x7fffffffu;
      if (x >= 0x7f800000u) return;
      lo = min(lo, x - LEAST);
      hi = max(hi, x);
    };
#pragma unroll 4
    for (int block = first; block < last; ++block) {
#pragma unroll
      for (int h = 0; h < SA; ++h) look(p.sa[block * sp_a + min(m0 + row0 + min(64 * h + lane, 16 * C::MT - 1), p.m - 1)], low_a, high_a);
      const int col = min(n0 + 64 * wn + (ROWB ? lane : 0), p.n - 1);
      look(p.sb[ROWB ? block * sp_b + col : (int64_t)(col / kFp8Block) * p.blocks + block], low_b, high_b);
    }
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) {
      low_a = min(low_a, (uint32_t)__shfl_xor((int)low_a, m, 64));
      high_a = max(high_a, (uint32_t)__shfl_xor((int)high_a, m, 64));
      low_b = min(low_b, (uint32_t)__shfl_xor((int)low_b, m, 64));
      high_b = max(high_b, (uint32_t)__shfl_xor((int)high_b, m, 64));
    }
    const float least = __uint_as_float(low_a + LEAST) * __uint_as_float(low_b + LEAST), most = __uint_as_float(high_a) * __uint_as_float(high_b);
    return __builtin_amdgcn_ballot_w64((low_a != ~0u && low_b != ~0u && least < 0x1p-126f) || most > 0x1.fffffep127f) != 0;
  };
  // The wave's part of the tile once more, straight from memory, with each product as Fp8Factors has it: the same bits where the scales' is a
  // normal number.
  auto far_products = [&](int m0, int n0) {
#pragma unroll
    for (int t = 0; t < C::MT; ++t)
#pragma unroll
      for (int u = 0; u < 4; ++u) acc[t][u] = f32x4{};
    for (int block = first; block < last; ++block) {
      int l = lane;
      asm volatile("" : "+v"(l));      // (addresses are formed where they are used: kept over the blocks they take more registers than there are)
      const int li = l & 15, lq = l >> 4;
      auto from_memory = [&](const uint8_t* x, int row) {
        const uint8_t* at = x + (int64_t)row * pitch + block * kFp8Block + 16 * lq;
        return F(*reinterpret_cast<const i32x4*>(at), *reinterpret_cast<const i32x4*>(at + 64));
      };
      B b;
      f32x4 of_b[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        b.f[u] = from_memory(p.b, min(n0 + 64 * wn + C::b_row(2 * u + (li >> 3), li & 7), p.n - 1));
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int col = min(n0 + 64 * wn + (ROWB ? C::col(u, lq) + r : 0), p.n - 1);
          of_b[u][r] = p.sb[ROWB ? block * sp_b + col : (int64_t)(col / kFp8Block) * p.blocks + block];
        }
      }
#pragma unroll
      for (int t = 0; t < C::MT; ++t) {
        __builtin_amdgcn_sched_barrier(0);
        const int row = min(m0 + row0 + 16 * t + li, p.m - 1);
        const F a = from_memory(p.a, row);
        const float of_a = p.sa[block * sp_a + row];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const f32x4 v = mma128(b.f[u], a);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const Fp8Factors f = factors(of_a, of_b[u][r]);
            acc[t][u][r] = __builtin_fmaf(__builtin_amdgcn_ldexpf(v[r], f.half), f.rest, acc[t][u][r]);
          }
        }
      }
    }
  };
  // One block; loads: of step `to_load`, into the buffer of the block before, where `loading`; next: there is a block behind this one in
  // its tile.
  auto multiply = [&](int to_load, bool loading, auto loads, auto next) {
    const uint8_t* st = lds + buf * C::kStage;
    const int buf_next = buf + 1 == NB ? 0 : buf + 1, buf_loaded = buf == 0 ? NB - 1 : buf - 1;
    f32x4 rb[4];
    if constexpr (ROWB) {
#pragma unroll
      for (int u = 0; u < 4; ++u) rb[u] = *reinterpret_cast<const f32x4*>(st + C::kSb + 4 * (64 * wn + C::col(u, q)));
    }
    uint32_t scales[SA + 1];
#pragma unroll
    for (int t = 0; t < C::MT; ++t) {
      __builtin_amdgcn_sched_barrier(0);      // (else all reads move to the front, and registers run out)
      const float s = sa * scale_b;
      const bool ahead = next.value && t + 1 == C::MT;      // (known where the loop is unrolled)
      const uint8_t* sn = lds + buf_next * C::kStage;
      if (t == 0) {
#pragma unroll
        for (int h = 0; h < SA; ++h) scales[h] = C::MT == 1 ? __float_as_uint(sa) : *reinterpret_cast<const uint32_t*>(st + at_sa[h]);
        scales[SA] = ROWB ? *reinterpret_cast<const uint32_t*>(st + at_sb) : __float_as_uint(scale_b);
      }
      F fa_next;
      if (t + 1 < C::MT) {
        fa_next = read_a(st, t + 1);
        sa = read_s(st, t + 1);
      }
      if constexpr (loads.value) {
        // (as many at a time as end by half of the row tiles; two or three of nine make no difference, all at once 2 to 5 % more)
        constexpr int HALF = (C::MT + 1) / 2, EACH = (C::PER + HALF) / HALF;
        if (loading)
#pragma unroll
          for (int j = EACH * t; j < EACH * (t + 1); ++j)
            if (j <= C::PER) load(to_load, buf_loaded, j);
      }
      if (ahead) meet(std::integral_constant<int, loads.value ? NB - 2 : 0>{});
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int before = t == 0 ? C::MT - 1 : t - 1;
        if (!ROWB || t > 0) {
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[before][u][r] = __builtin_fmaf(d[u][r], ROWB ? s_before * rb[u][r] : s_before, acc[before][u][r]);
          asm volatile("" : "+v"(acc[before][u]));      // (here and not at the block's end, where the compiler would gather them all)
        }
        d[u] = mma128(fb.f[u], fa);
        if (ahead) fb.f[u] = fragment(sn + C::kB + (64 * wn + 16 * u) * 128);
      }
      if (t == 0) {
#pragma unroll
        for (int h = 0; h <= SA; ++h) {
          low = min(low, scales[h] - LEAST);
          high = max(high, scales[h]);
        }
      }
      s_before = s;
      if (ahead) {
        fa = read_a(sn, 0);
        sa = read_s(sn, 0);
        scale_b = read_scale_b(sn);
        buf = buf_next;
      } else if (t + 1 < C::MT) {
        fa = fa_next;
      }
    }
    if constexpr (ROWB) {      // (the scales of b's rows are the block's own)
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[C::MT - 1][u][r] = __builtin_fmaf(d[u][r], s_before * rb[u][r], acc[C::MT - 1][u][r]);
    }
  };
  // A workgroup walks over tiles (where it has one buffer to fill ahead and no sums of groups to add): the last block of one is multiplied
  // while the next one's first is loaded, and its results are stored while that is on its way.
  constexpr bool WALKS = WK == 1 && NB == 2;
  for (;;) {
    const int m0 = from.m0, n0 = from.n0;
    int step = 0;
    for (; step + NB - 1 < steps; ++step) multiply(step + NB - 1, true, std::true_type{}, std::true_type{});
    if constexpr (NB > 2)
      for (; step + 1 < steps; ++step) multiply(0, false, std::false_type{}, std::true_type{});
    tile += gridDim.x;
    const bool more = WALKS && tile < (uint32_t)p.tiles_m * p.tiles_n;
    if (more) from = place(tile);
    if (WK == 1 || first + step < last) multiply(0, more, std::integral_constant<bool, WALKS>{}, std::false_type{});
    if constexpr (!ROWB) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[C::MT - 1][u][r] = __builtin_fmaf(d[u][r], s_before, acc[C::MT - 1][u][r]);
    }
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(low < 0x20000000u - LEAST || high > 0x5f000000u) != 0, 0))
      if (far_apart(m0, n0)) far_products(m0, n0);
    if constexpr (WK > 1) {
      // the groups' sums, added in their order
      f32x4* sums = reinterpret_cast<f32x4*>(lds_all) + wave * C::MT * 4 * kWave + lane;
      __syncthreads();
      if (group > 0)
#pragma unroll
        for (int t = 0; t < C::MT; ++t)
#pragma unroll
          for (int u = 0; u < 4; ++u) sums[((group - 1) * C::W * C::MT * 4 + 4 * t + u) * kWave] = acc[t][u];
      __syncthreads();
      if (group > 0) return;
#pragma unroll
      for (int g = 0; g < WK - 1; ++g)
#pragma unroll
        for (int t = 0; t < C::MT; ++t)
#pragma unroll
          for (int u = 0; u < 4; ++u) acc[t][u] += sums[(g * C::W * C::MT * 4 + 4 * t + u) * kWave];
    }
    const int n = n0 + 64 * wn;
    f32x4 bias[4];
    // (here and not where a row is stored: what it reads would be waited for in every block of the next tile, since a row may not be)
#pragma unroll
    for (int u = 0; u < 4; ++u) asm volatile("" : "+v"(acc[C::MT - 1][u]));
    // (the next tile's first block has landed before the first store: stores in front of these loads cost 1 to 3 % where k is short)
    if (more) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    load_bias(bias, p.bias, p.bias_type, p.n, [&](int u, int r) { return n + C::col(u, q) + r; });
#pragma unroll
    for (int t = 0; t < C::MT; ++t) {
      const int m = m0 + row0 + 16 * t + i;
      if (m >= p.m) continue;
      if (p.splits > 1) {
        float* row = (float*)p.out + ((int64_t)split * p.m + m) * p.n;
#pragma unroll
        for (int u = 0; u < 4; ++u) store4(row, n + C::col(u, q), p.n, acc[t][u]);
      } else {
        O* row = (O*)p.out + (int64_t)m * p.n;
        if (sizeof(O) == 2 && n + 64 <= p.n) {
#pragma unroll
          for (int u = 0; u < 4; u += 2) {
            f32x8 v;
#pragma unroll
            for (int r = 0; r < 8; ++r) v[r] = acc[t][u + r / 4][r % 4] + bias[u + r / 4][r % 4];
            store_cols(row + n + C::col(u, q), v, 8);
          }
        } else {
#pragma unroll
          for (int u = 0; u < 4; ++u) store4(row, n + C::col(u, q), p.n, acc[t][u] + bias[u]);
        }
      }
    }
    if (!more) break;
    // (what this wave loaded of the next tile has landed)
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    buf ^= 1;
    const uint8_t* st = lds + buf * C::kStage;
    fb = read_b(st);
    fa = read_a(st, 0);
    sa = read_s(st, 0);
    scale_b = read_scale_b(st);
    begin_scales();
    s_before = 0.0f;
#pragma unroll
    for (int u = 0; u < 4; ++u) d[u] = f32x4{};
#pragma unroll
    for (int t = 0; t < C::MT; ++t)
#pragma unroll
      for (int u = 0; u < 4; ++u) acc[t][u] = f32x4{};
  }
}

// Partial results of splits of k, added in their order.
template <typename O>
__global__ __launch_bounds__(256) void fp8_join_kernel(const float* __restrict__ part, int splits, int64_t count, int n, const void* bias,
                                                       int bias_type, O* __restrict__ out) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= count) return;
  typedef float F4 __attribute__((ext_vector_type(4), aligned(4)));
  if (at + 4 <= count) {
    F4 s = *reinterpret_cast<const F4*>(part + at);
    for (int k = 1; k < splits; ++k) s += *reinterpret_cast<const F4*>(part + k * count + at);
    const int first = (int)(at % n);
    f32x4 add[1];
    load_bias(add, bias, bias_type, n, [&](int, int e) { return n < 4 ? (first + e) % n : first + e < n ? first + e : first + e - n; });
    store4(out + at, 0, 4, f32x4{s[0], s[1], s[2], s[3]} + add[0]);
  } else {
    for (int64_t c = at; c < count; ++c) {
      float s = part[c];
      for (int k = 1; k < splits; ++k) s += part[k * count + c];
      out[c] = (O)(s + (bias ? param_at(bias, bias_type, c % n) : 0.0f));
    }
  }
}

// Up to 16 rows of a: bound by reading b once, and by the time a read takes.  A workgroup has 16 rows of b; its waves share the blocks of k,
// read b straight into registers (16 rows of whole 128-byte lines) and a from the caches, four blocks before the first is multiplied,
// and add their sums in LDS, in their order.  1 x 2048 x 8192 5.3 us, 1 x 4096 x 4096 5.5 (3.0 TB/s, 2.5 us of it the launch's).  With more
// rows the caches are asked for a too often (37 x 4096 x 4096 12 us in three groups of 16, as tiles with a split of k 8).
template <typename O>
__global__ __launch_bounds__(512) void fp8_few_rows_product(Fp8Args p) {
  constexpr int W = 8;
  __shared__ f32x4 sums[W][kWave];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16, row = min(i, p.m - 1);
  const int64_t pitch = fp8_pitch((int64_t)p.blocks * kFp8Block), sp = fp8_scale_pitch(p.m);
  typedef Fragment<sizeof(O) == 4> F;
  const float *sb = p.sb + (int64_t)(n0 / kFp8Block) * p.blocks, *sa = p.sa + row;
  const uint8_t *rb = p.b + min(n0 + i, p.n - 1) * pitch + 16 * q, *ra = p.a + row * pitch + 16 * q;
  f32x4 acc = f32x4{};
  // (in front of everything, by the wave that stores)
  f32x4 bias[1] = {f32x4{}};
  if (wave == 0) load_bias(bias, p.bias, p.bias_type, p.n, [&](int, int r) { return n0 + 4 * q + r; });
  auto multiply = [&](int first, auto count) {
    constexpr int N = count.value;
    i32x4 b[N][2], a[N][2];
    float s[N], t[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int64_t at = (int64_t)(first + W * j) * kFp8Block;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        b[j][h] = *reinterpret_cast<const i32x4*>(rb + at + 64 * h);
        a[j][h] = *reinterpret_cast<const i32x4*>(ra + at + 64 * h);
      }
      s[j] = sb[first + W * j];
      t[j] = sa[(first + W * j) * sp];
    }
    __builtin_amdgcn_sched_barrier(0);      // (else the loads move to where they are used, one after the other)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const f32x4 d = mma128(F(b[j][0], b[j][1]), F(a[j][0], a[j][1]));
      const Fp8Factors f = factors(s[j], t[j]);
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[r] = __builtin_fmaf(__builtin_amdgcn_ldexpf(d[r], f.half), f.rest, acc[r]);
    }
  };
  int block = wave;
  for (; block + 3 * W < p.blocks; block += 4 * W) multiply(block, std::integral_constant<int, 4>{});
  for (; block + W < p.blocks; block += 2 * W) multiply(block, std::integral_constant<int, 2>{});
  if (block < p.blocks) multiply(block, std::integral_constant<int, 1>{});
  sums[wave][lane] = acc;
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int w = 1; w < W; ++w) acc += sums[w][lane];
  const int n = n0 + 4 * q;
  if (i >= p.m) return;
  store4((O*)p.out + (int64_t)i * p.n, n, p.n, acc + bias[0]);
}

// ---- which kernel ---------------------------------------------------------------------------------------
namespace {
// The tile kernels, as (tile; workgroups that the 256 compute units hold at once; what a round of these takes per block of k, in units of 10 ns,
// with 16-bit and with fp32 results; 0: not built).  The one whose rounds take least is chosen.  us at k = 4096 when the costs were set, in the order below (the fifth without
// fp32): 1024 x 1024 12.0 / 16.6 / 22.9 / 41.6, 1280^2 22.0 / 19.0 / 22.9, 1536^2 32.6 / 32.3 / 23.4 / 41.8, 2048^2 - / - / 26.4 / 44.7 / 38.1 /
// 50.4, 2560^2 - / - / 46.6 / 48.9 / 38.5 / 50.5, 3328^2 68.5 / 83.1 / 72.3 / 51.3 for the last four, 4608^2 135 / 136 / 114 / 106;
// 192 x 256 and 256 x 256 3328^2 52 / 56, 4608^2 92 / 106, 6144 x 4096 105 / 106, 8192 x 8192 270 / 230 (whole rounds are bound by power); fp32 1024^2 16.6 /
// 20.6 / 31.7, 1536^2 46.8 / 44.3 / 33.3 / 44.8, 2560^2 66 / 68, 4096^2 141 / 138 for the two of 128 x 128.
enum Fp8Kernel { kFewRows, k64Deep, k64Pair, k128Split, k128Pair, k256x128, k192, k256 };
struct Fp8Shape {
  Fp8Kernel kernel;
  int tm, tn, at_once, cost16, cost32;
};
constexpr Fp8Shape kFp8Shapes[] = {{k64Deep, 64, 64, 256, 36, 50},     {k64Pair, 64, 64, 512, 55, 75},      {k128Split, 128, 128, 256, 72, 100},
                                   {k128Pair, 128, 128, 512, 138, 145}, {k256x128, 256, 128, 256, 119, 0}, {k192, 192, 256, 256, 146, 0},
                                   {k256, 256, 256, 256, 175, 0}};
struct Fp8Plan {
  Fp8Kernel kernel;
  int splits;
};
Fp8Plan fp8_plan(int64_t m, int64_t n, int64_t blocks, bool square, bool wide) {
  // (16 x 4096 x 4096 6.6 us, as tiles 9.9; 16 x 8192 x 1024 9.5 and 9.3)
  // (and a launch has fewer than 2^32 threads: 512 per 16 columns)
  if (m <= 16 && square && n <= 1 << 26) return {kFewRows, 1};
  auto tiles = [&](int tm, int tn) { return ((m + tm - 1) / tm) * ((n + tn - 1) / tn); };
  Fp8Plan best{k64Deep, 1};
  int64_t least = INT64_MAX;
  for (const Fp8Shape& s : kFp8Shapes) {
    // (its fp32 results with scales per row take 150 registers, and so one workgroup to a compute unit: 1300 x 1024 x 1300 14.5 us, two rounds of k64Deep
    // 13.6, 1024 x 4096 x 1100 40.0 and 32.5)
    if (s.kernel == k64Pair && wide && !square) continue;
    const int64_t cost = (tiles(s.tm, s.tn) + s.at_once - 1) / s.at_once * (wide ? s.cost32 : s.cost16);
    if (cost > 0 && cost < least) {
      least = cost;
      best.kernel = s.kernel;
    }
  }
  // Few small tiles share the sum over k with one another, as many as fill the machine and leave each 8 blocks (64 x 4096 x 2048 with 1, 2, 4, 8
  // parts 11.4, 10.0, 9.0, 10.7 us; 512 x 147456 x 128 with 1, 8, 16, 32 306, 49, 41, 48).
  if (best.kernel == k64Deep)
    while (best.splits < 64 && tiles(64, 64) * 2 * best.splits <= 256 && blocks / (2 * best.splits) >= 8) best.splits *= 2;
  return best;
}
}  // namespace

int64_t fp8_matmul_workspace_elems(int64_t m, int64_t n, int64_t blocks, bool square, bool wide) {
  const Fp8Plan plan = fp8_plan(m, n, blocks, square, wide);
  return plan.splits > 1 ? plan.splits * m * n : 0;
}

template <int TM, int TN, int WM, int WN, int WK, int NB, typename O> static void tile_product(Fp8Args p, bool square, hipStream_t stream) {
  p.tiles_m = (p.m + TM - 1) / TM;
  p.tiles_n = (p.n + TN - 1) / TN;
  auto* kernel = fp8_tile_product<TM, TN, WM, WN, WK, NB, false, O>;
  if constexpr (TM > 64 || NB > 2 || sizeof(O) == 2)      // (the one that fp8_plan leaves out)
    if (!square) kernel = fp8_tile_product<TM, TN, WM, WN, WK, NB, true, O>;
  // (walking over tiles: as many workgroups as the compute units hold)
  const unsigned tiles = (unsigned)p.tiles_m * p.tiles_n;
  const unsigned groups = WK == 1 && NB == 2 ? std::min(tiles, 256u * (TM * TN > 128 * 128 ? 1 : 2)) : tiles;
  kernel<<<dim3(groups, p.splits), dim3(64 * WM * WN * WK), 0, stream>>>(p);
}

template <typename O>
int fp8_matmul(const void* a, const float* sa, const void* b, const float* sb, bool square, const void* bias, int bias_type, O* out,
               float* workspace, int m, int n, int blocks, hipStream_t stream) {
  const Fp8Plan plan = fp8_plan(m, n, blocks, square, sizeof(O) == 4);
  Fp8Args p{(const uint8_t*)a, sa, (const uint8_t*)b, sb, bias, bias_type, out, m, n, blocks, 0, 0, plan.splits};
  if (plan.splits > 1) {
    p.out = workspace;
    p.bias = nullptr;
  }
  switch (plan.kernel) {
    case kFewRows: fp8_few_rows_product<O><<<dim3((n + 15) / 16), dim3(512), 0, stream>>>(p); break;
    case k64Deep: tile_product<64, 64, 4, 1, 2, 4, O>(p, square, stream); break;
    case k64Pair: tile_product<64, 64, 4, 1, 2, 2, O>(p, square, stream); break;
    case k128Split: tile_product<128, 128, 2, 2, 2, 2, O>(p, square, stream); break;
    case k128Pair: tile_product<128, 128, 2, 2, 1, 2, O>(p, square, stream); break;
    case k256x128:      // (with fp32 results two workgroups of 128 x 128 to a compute unit take fewer or as many rounds, of 145 against 210)
      if constexpr (sizeof(O) == 2) tile_product<256, 128, 4, 2, 1, 2, O>(p, square, stream);
      break;
    case k192:
      if constexpr (sizeof(O) == 2) tile_product<192, 256, 2, 4, 1, 2, O>(p, square, stream);
      break;
    case k256:      // (fp32 results have widened fragments, twice the registers)
      if constexpr (sizeof(O) == 2) tile_product<256, 256, 2, 4, 1, 2, O>(p, square, stream);
  }
  if (plan.splits > 1) {
    const int64_t count = (int64_t)m * n;
    fp8_join_kernel<O><<<dim3((unsigned)((count + 1023) / 1024)), dim3(256), 0, stream>>>(workspace, plan.splits, count, n, bias, bias_type, out);
  }
  return 0;
}

#define PTX_FP8_TYPES(O)                                                                                                          \
  template int fp8_matmul(const void*, const float*, const void*, const float*, bool, const void*, int, O*, float*, int, int, int, \
                          hipStream_t);
PTX_FP8_TYPES(float)
PTX_FP8_TYPES(bf16_t)
PTX_FP8_TYPES(f16_t)

}  // namespace ptx
