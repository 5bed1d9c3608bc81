// Products of matrices in 8-bit blocks (fp8.h):
//   out[m][n] = sum over blocks of  sa[block][m] sb[..] sum_{k in block} a[m][k] b[n][k]   (+ bias[n])
// a's scales are per row and 128 columns, b's the same (ROWB) or per 128 x 128.
//
// One MFMA of 16 x 16 x 128 covers exactly one block, so its 16 x 16 results, in fp32, are multiplied by the block's scales and added to
// the accumulators by the vector pipe: 4 fused multiply-adds per lane (16 cycles) beside an MFMA's 32, which run at the same time.
// b is the MFMA's first operand, a its second: a lane then holds results of one m, and one product of scales serves all its n of a block.
//
// The 8-bit MFMA does not sum in full fp32: it aligns the products of 8 neighbouring k to the largest of them and cuts what lies below
// 2^-13 of it (measured; over groups it is fp32).  On normal data that is 1.4e-5 of a result, far below the rounding of 16-bit results
// (2^-9 and 2^-12 at most), which take it.  Results in fp32 do not: for those the values, which f16 holds exactly, are widened in registers
// and multiplied by the f16 MFMA, whose sums are fp32 (1e-8 on the same data), at half of the 8-bit rate.
#include <algorithm>

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
  __device__ __forceinline__ Fragment(const i32x4& lo, const i32x4& hi) : v(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)) {}
};
template <> struct Fragment<true> {
  f16x8 v[4];
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

__device__ __forceinline__ float param_at(const void* p, int type, int64_t i) {
  return type == 0 ? ((const float*)p)[i] : type == 1 ? (float)((const bf16_t*)p)[i] : (float)((const f16_t*)p)[i];
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

// Tiles of TM x TN, WM x WN waves of TM / WM x 64 each.  Both operands' 128 columns of a block go to LDS (direct loads, two buffers: one
// block is loaded while the other is multiplied), rows of 128 bytes whose 16-byte pieces lie at place piece ^ (row % 8).  Rows of b
// lie in LDS so that a lane's results of four MFMAs are 16 neighbouring n: row 16 t + i of 64 holds n = 16 (i / 4) + 4 t + i % 4.
template <int TM, int TN, int WM, int WN> struct Fp8Tile {
  static constexpr int W = WM * WN, MT = TM / WM / 16;
  static constexpr int kB = 0, kA = TN * 128, kSa = kA + TM * 128, kSb = kSa + 1024, kStage = kSb + 1024;
  static constexpr int PER = (TM + TN) / 8 / W;      // loads of 1 KB per wave and block
  static constexpr int PER_B = TN / 8 / W;
  static_assert(TN == 64 * WN && (TN / 8) % W == 0 && (TM / 8) % W == 0 && TM <= 256 && TN <= 256, "whole loads per wave");
};

template <int TM, int TN, int WM, int WN, bool ROWB, typename O>
__global__ __launch_bounds__(64 * WM * WN) void fp8_tile_product(Fp8Args p) {
  typedef Fp8Tile<TM, TN, WM, WN> C;
  __shared__ __align__(16) uint8_t lds[2 * C::kStage];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN, i = lane & 15, q = lane >> 4;
  const int split = blockIdx.y;
  int tm, tn;
  tile_of(blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
  const int m0 = tm * TM, n0 = tn * TN;
  const int first = (int)((int64_t)p.blocks * split / p.splits), last = (int)((int64_t)p.blocks * (split + 1) / p.splits);
  const uint32_t pitch = (uint32_t)p.blocks * kFp8Block;
  // what this lane loads: rows beyond the end are the last one once more
  const int e = lane >> 3;
  const uint32_t piece = (uint32_t)((lane & 7) ^ e) * 16;
  uint32_t off[C::PER];
#pragma unroll
  for (int j = 0; j < C::PER; ++j) {
    if (j < C::PER_B) {
      const int g = wave + C::W * j, s = g & 7;
      const int row = 64 * (g >> 3) + 16 * (2 * (s & 1) + (e >> 2)) + 4 * (s >> 1) + (e & 3);
      off[j] = (uint32_t)min(row, p.n - 1 - n0) * pitch + piece;
    } else {
      const int row = 8 * (wave + C::W * (j - C::PER_B)) + e;
      off[j] = (uint32_t)min(row, p.m - 1 - m0) * pitch + piece;
    }
  }
  const uint64_t base_a = uniform64((uint64_t)(p.a + (int64_t)m0 * pitch)), base_b = uniform64((uint64_t)(p.b + (int64_t)n0 * pitch));
  const int64_t sp_a = fp8_scale_pitch(p.m), sp_b = fp8_scale_pitch(p.n);
  const uint64_t base_sa = uniform64((uint64_t)(p.sa + m0));
  const uint32_t off_sa = 4u * (uint32_t)min((int64_t)4 * lane, sp_a - 4 - m0);
  const uint64_t base_sb = uniform64((uint64_t)(p.sb + (ROWB ? n0 : 0)));
  const uint32_t off_sb = ROWB ? 4u * (uint32_t)min((int64_t)4 * lane, sp_b - 4 - n0) : 0u;
  const uint32_t lds0 = lds_address(lds);
  auto load = [&](int block, int buf) {
    const uint32_t to = lds0 + buf * C::kStage;
    const uint64_t k = (uint64_t)block * kFp8Block;
#pragma unroll
    for (int j = 0; j < C::PER; ++j) {
      if (j < C::PER_B) load_to_lds16_s<0>(base_b + k, off[j], to + C::kB + 1024 * (wave + C::W * j));
      else load_to_lds16_s<0>(base_a + k, off[j], to + C::kA + 1024 * (wave + C::W * (j - C::PER_B)));
    }
    if (wave == 0) load_to_lds16_s<0>(base_sa + 4 * (uint64_t)block * sp_a, off_sa, to + C::kSa);
    if (ROWB && wave == C::W - 1) load_to_lds16_s<0>(base_sb + 4 * (uint64_t)block * sp_b, off_sb, to + C::kSb);
  };
  // this wave's scale of b per block
  const float* sb = p.sb + (ROWB ? 0 : (int64_t)__builtin_amdgcn_readfirstlane(min(n0 + 64 * wn, p.n - 1) / kFp8Block) * p.blocks);
  f32x4 acc[C::MT][4];
#pragma unroll
  for (int t = 0; t < C::MT; ++t)
#pragma unroll
    for (int u = 0; u < 4; ++u) acc[t][u] = f32x4{};
  const int at = i * 128 + ((q ^ (i & 7)) << 4);
  typedef Fragment<sizeof(O) == 4> F;
  auto fragment = [&](const uint8_t* tile) {      // 16 rows of 128 bytes
    return F(*reinterpret_cast<const i32x4*>(tile + at), *reinterpret_cast<const i32x4*>(tile + (at ^ 64)));
  };
  load(first, 0);
  float next_sb = ROWB ? 1.0f : sb[first];
  for (int block = first; block < last; ++block) {
    const int buf = (block - first) & 1;
    ring_barrier<0>();
    if (block + 1 < last) load(block + 1, buf ^ 1);
    const float scale_b = next_sb;
    if (!ROWB && block + 1 < last) next_sb = sb[block + 1];
    const uint8_t* st = lds + buf * C::kStage;
    const uint8_t* tb = st + C::kB + 64 * wn * 128;
    const F fb[4] = {fragment(tb), fragment(tb + 16 * 128), fragment(tb + 32 * 128), fragment(tb + 48 * 128)};
    f32x4 rb[4];
    if constexpr (ROWB) {
#pragma unroll
      for (int u = 0; u < 4; ++u) rb[u] = *reinterpret_cast<const f32x4*>(st + C::kSb + 4 * (64 * wn + 16 * q + 4 * u));
    }
#pragma unroll
    for (int t = 0; t < C::MT; ++t) {
      const int row = wm * (TM / WM) + 16 * t;
      const F fa = fragment(st + C::kA + row * 128);
      const float s = *reinterpret_cast<const float*>(st + C::kSa + 4 * (row + i)) * scale_b;
      f32x4 d[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) d[u] = mma128(fb[u], fa);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[t][u][r] = __builtin_fmaf(d[u][r], ROWB ? s * rb[u][r] : s, acc[t][u][r]);
    }
  }
  const int n = n0 + 64 * wn + 16 * q;
  f32x4 bias[4];
#pragma unroll
  for (int u = 0; u < 4; ++u)
#pragma unroll
    for (int r = 0; r < 4; ++r) bias[u][r] = p.bias && n + 4 * u + r < p.n ? param_at(p.bias, p.bias_type, n + 4 * u + r) : 0.0f;
#pragma unroll
  for (int t = 0; t < C::MT; ++t) {
    const int m = m0 + wm * (TM / WM) + 16 * t + i;
    if (m >= p.m) continue;
    if (p.splits > 1) {
      float* row = (float*)p.out + ((int64_t)split * p.m + m) * p.n;
#pragma unroll
      for (int u = 0; u < 4; ++u) store4(row, n + 4 * u, p.n, acc[t][u]);
    } else {
      O* row = (O*)p.out + (int64_t)m * p.n;
      if (n + 16 <= p.n && sizeof(O) == 2) {
#pragma unroll
        for (int u = 0; u < 4; u += 2) {
          f32x8 v;
#pragma unroll
          for (int r = 0; r < 8; ++r) v[r] = acc[t][u + r / 4][r % 4] + bias[u + r / 4][r % 4];
          store_cols(row + n + 4 * u, v, 8);
        }
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u) store4(row, n + 4 * u, p.n, acc[t][u] + bias[u]);
      }
    }
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
    if (bias)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += param_at(bias, bias_type, (at + e) % n);
    store4(out + at, 0, 4, f32x4{s[0], s[1], s[2], s[3]});
  } else {
    for (int64_t c = at; c < count; ++c) {
      float s = part[c];
      for (int k = 1; k < splits; ++k) s += part[k * count + c];
      out[c] = (O)(s + (bias ? param_at(bias, bias_type, c % n) : 0.0f));
    }
  }
}

// Few rows of a (16 MT of them): bound by reading b once.  A workgroup has 16 rows of b; its waves share the blocks of k (one each in
// turn), read b straight into registers (16 rows of whole 128-byte lines) and a from the caches, and add their sums in LDS, in their order.
template <int MT, typename O>
__global__ __launch_bounds__(512) void fp8_few_rows_product(Fp8Args p) {
  constexpr int W = 8;
  __shared__ f32x4 sums[W][MT][kWave];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int64_t pitch = (int64_t)p.blocks * kFp8Block, sp = fp8_scale_pitch(p.m);
  typedef Fragment<sizeof(O) == 4> F;
  auto fragment = [&](const uint8_t* row) {
    return F(*reinterpret_cast<const i32x4*>(row + 16 * q), *reinterpret_cast<const i32x4*>(row + 64 + 16 * q));
  };
  const uint8_t* rb = p.b + min(n0 + i, p.n - 1) * pitch;
  const float* sb = p.sb + (int64_t)(n0 / kFp8Block) * p.blocks;
  f32x4 acc[MT];
  const uint8_t* ra[MT];
  int row[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    acc[t] = f32x4{};
    row[t] = min(16 * t + i, p.m - 1);
    ra[t] = p.a + row[t] * pitch;
  }
#pragma unroll 2
  for (int block = wave; block < p.blocks; block += W) {
    const F fb = fragment(rb + (int64_t)block * kFp8Block);
    const float s = sb[block];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const f32x4 d = mma128(fb, fragment(ra[t] + (int64_t)block * kFp8Block));
      const float f = s * p.sa[block * sp + row[t]];
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[t][r] = __builtin_fmaf(d[r], f, acc[t][r]);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) sums[wave][t][lane] = acc[t];
  __syncthreads();
  for (int t = wave; t < MT; t += W) {
    f32x4 v = sums[0][t][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) v += sums[w][t][lane];
    const int m = 16 * t + i, n = n0 + 4 * q;
    if (m >= p.m) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] += p.bias && n + r < p.n ? param_at(p.bias, p.bias_type, n + r) : 0.0f;
    store4((O*)p.out + (int64_t)m * p.n, n, p.n, v);
  }
}

// ---- which kernel ---------------------------------------------------------------------------------------
namespace {
struct Fp8Plan {
  int tile;      // 0: few rows, else 64, 128 or 256
  int splits;
};
Fp8Plan fp8_plan(int64_t m, int64_t n, int64_t blocks, bool square) {
  if (m <= 64 && square) return {0, 1};
  auto tiles = [&](int t) { return ((m + t - 1) / t) * ((n + t - 1) / t); };
  if (tiles(256) >= 192) return {256, 1};
  if (tiles(128) >= 192) return {128, 1};
  const int tile = 64;
  const int64_t count = tiles(tile);
  int splits = 1;
  while (splits < 16 && count * splits < 256 && blocks / (2 * splits) >= 4) splits *= 2;
  return {tile, splits};
}
}  // namespace

int64_t fp8_matmul_workspace_elems(int64_t m, int64_t n, int64_t blocks, bool square) {
  const Fp8Plan plan = fp8_plan(m, n, blocks, square);
  return plan.splits > 1 ? plan.splits * m * n : 0;
}

template <int TM, int TN, int WM, int WN, typename O> static void tile_product(Fp8Args p, bool square, hipStream_t stream) {
  p.tiles_m = (p.m + TM - 1) / TM;
  p.tiles_n = (p.n + TN - 1) / TN;
  auto* kernel = square ? fp8_tile_product<TM, TN, WM, WN, false, O> : fp8_tile_product<TM, TN, WM, WN, true, O>;
  kernel<<<dim3((unsigned)p.tiles_m * p.tiles_n, p.splits), dim3(64 * WM * WN), 0, stream>>>(p);
}

template <typename O>
int fp8_matmul(const void* a, const float* sa, const void* b, const float* sb, bool square, const void* bias, int bias_type, O* out,
               float* workspace, int m, int n, int blocks, hipStream_t stream) {
  const Fp8Plan plan = fp8_plan(m, n, blocks, square);
  Fp8Args p{(const uint8_t*)a, sa, (const uint8_t*)b, sb, bias, bias_type, out, m, n, blocks, 0, 0, plan.splits};
  if (plan.tile == 0) {
    const dim3 grid((n + 15) / 16), block(512);
    switch ((m + 15) / 16) {
      case 1: fp8_few_rows_product<1, O><<<grid, block, 0, stream>>>(p); break;
      case 2: fp8_few_rows_product<2, O><<<grid, block, 0, stream>>>(p); break;
      case 3: fp8_few_rows_product<3, O><<<grid, block, 0, stream>>>(p); break;
      default: fp8_few_rows_product<4, O><<<grid, block, 0, stream>>>(p);
    }
    return 0;
  }
  if (plan.splits > 1) {
    p.out = workspace;
    p.bias = nullptr;
  }
  if (plan.tile == 256) tile_product<256, 256, 2, 4, O>(p, square, stream);
  else if (plan.tile == 128) tile_product<128, 128, 2, 2, O>(p, square, stream);
  else tile_product<64, 64, 4, 1, O>(p, square, stream);
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
