// The dropout mask of the residual updates (dropout.hip, dropnorm.hip), 8-column vectors at any alignment and sums over lanes (those
// and relbias.hip).
//
// The mask is never stored: forward and backward kernels draw it from Philox4x32-10, the counter-based generator of
// Salmon, Moraes, Dror and Shaw (Parallel random numbers: as easy as 1, 2, 3, 2011).  A mask row's columns lie in
// blocks of 8; block k of mask row r has the counter (k, r, 0, draw) and the seed as its key.  Draw 0 gives the block's
// 8 numbers of 16 bits (word i / 2, low half first), draw 1 the 16 bits below them: an element is kept where the 32-bit
// number is at least round(p 2^32).  The second draw is made only where a first number equals the threshold's upper half
// (8 in 65536 blocks; never where the lower half is 0, as for p = 1/4), so that p has a resolution of 2^-32 for the
// price of 16 bits.  What a number depends on is its mask row and column alone: neither the types, the
// alignment nor the launch.
#pragma once
#include "common.h"

namespace ptx {

struct Dropout {
  uint32_t key[2];
  const int64_t* seed;   // read from device memory where given: the key then
  uint32_t hi, lo;       // the threshold round(p 2^32): hi 2^16 + lo; 0 = no dropout, 2^16 and 0 = nothing stays
  float scale;           // 1 / (1 - p), 1 for p = 0, 0 for p = 1
  // Rows are [outer][shared][inner]; the rows of one (outer, inner) have the same mask row, outer * inner + inner.
  uint32_t shared, inner;
};

__device__ __forceinline__ Dropout with_key(Dropout d) {
  if (d.seed && (d.hi | d.lo)) {
    const uint64_t s = (uint64_t)*d.seed;
    d.key[0] = (uint32_t)s;
    d.key[1] = (uint32_t)(s >> 32);
  }
  return d;
}

__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) { return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96); }

__device__ __forceinline__ void philox(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c[0] * 0xD2511F53u, b = (uint64_t)c[2] * 0xCD9E8D57u;
    c[0] = xor3((uint32_t)(b >> 32), c[1], k0);
    c[1] = (uint32_t)b;
    c[2] = xor3((uint32_t)(a >> 32), c[3], k1);
    c[3] = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

// Which elements of block k of the mask row stay: bit e / 2 + 16 (e % 2) for element e (as the words hold them; the other bits
// are of no use).
__device__ __forceinline__ uint32_t dropout_keeps(const Dropout& d, uint32_t row, uint32_t k) {
  if (!(d.hi | d.lo)) return ~0u;
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  uint32_t w[4] = {k, row, 0u, 0u};
  philox(w, d.key[0], d.key[1]);
  // (a number equal to hi is kept where lo is 0; where it is not, the second draw decides)
  const unsigned short least = (unsigned short)(d.hi + (d.lo != 0) - 1);      // what is above it is kept
  const u16x2 above = {least, least}, one = {1, 1}, same = {(unsigned short)d.hi, (unsigned short)d.hi};
  uint32_t keeps = 0;
  u16x2 off = {0xFFFF, 0xFFFF};
#pragma unroll
  for (int i = 3; i >= 0; --i) {
    const u16x2 u = __builtin_bit_cast(u16x2, w[i]);
    keeps = keeps << 1 | __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_elementwise_sub_sat(u, above), one));
    off = __builtin_elementwise_min(off, u ^ same);
  }
  if (d.lo != 0 && (off[0] == 0 || off[1] == 0)) {
    uint32_t v[4] = {k, row, 0u, 1u};
    philox(v, d.key[0], d.key[1]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t u = e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xFFFFu;
      const uint32_t below = e & 1 ? v[e >> 1] >> 16 : v[e >> 1] & 0xFFFFu;
      if (u == d.hi && below >= d.lo) keeps |= 1u << (e / 2 + 16 * (e % 2));
    }
  }
  asm volatile("" : "+v"(keeps));      // (formed here: where it is used, the compiler would wait for loads in between first)
  return keeps;
}

// x where element e stays, else exactly 0 whatever x holds; `scale` is left to the caller's multiplication
__device__ __forceinline__ float kept(float x, uint32_t keeps, int e) {
  return __uint_as_float(__float_as_uint(x) & (uint32_t)((int32_t)(keeps << (31 - (e / 2 + 16 * (e % 2)))) >> 31));
}

// The sum over G neighbouring lanes, in all of them, on the vector pipe: moves within rows of 16 lanes, then exchanges of rows and
// halves (a shuffle through LDS takes some hundred cycles a step, and a norm's row has up to eighteen of them).
template <int CTRL> __device__ __forceinline__ float lane_move(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
template <int G> __device__ __forceinline__ float lanes_sum(float v) {
  static_assert(G >= 1 && G <= 64 && (G & (G - 1)) == 0, "a power of two of lanes");
  if constexpr (G >= 2) v += lane_move<0xB1>(v);       // lane ^ 1 (within four: 1 0 3 2)
  if constexpr (G >= 4) v += lane_move<0x4E>(v);       // lane ^ 2 (2 3 0 1)
  if constexpr (G >= 8) v += lane_move<0x141>(v);      // 7 - lane within 8: the other four
  if constexpr (G >= 16) v += lane_move<0x140>(v);      // 15 - lane within 16: the other eight
  // (the results by way of variables: a cast of a vector's element takes the first one)
  if constexpr (G >= 32) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto w = __builtin_amdgcn_permlane16_swap(u, u, false, false);      // rows 0 0 2 2 and 1 1 3 3
    const uint32_t a = w[0], b = w[1];
    v = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
  }
  if constexpr (G >= 64) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto w = __builtin_amdgcn_permlane32_swap(u, u, false, false);      // the halves
    const uint32_t a = w[0], b = w[1];
    v = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
  }
  return v;
}

// Eight elements at an element's alignment (rows of odd lengths): gfx950 takes vector accesses at any address, so an
// odd row costs the lines it straddles and nothing else.
template <typename T> struct Unaligned8 { typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T)))); };
template <typename T> using Raw8 = typename Unaligned8<T>::type;

template <typename T> __device__ __forceinline__ f32x8 widened(const Raw8<T>& v) {
  f32x8 o;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = (float)v[e];
  return o;
}
template <typename T> __device__ __forceinline__ Raw8<T> rounded(const f32x8& v) {
  Raw8<T> o;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = (T)v[e];
  return o;
}

// Columns col .. col + n - 1 of a row (n <= 8).  The load of a row's last, shorter block is moved back to where it ends with the
// row, so that a load is one instruction without a branch (behind a branch the next load would wait for this one), and what it
// brings is moved to its place when it is used.  Rows of fewer than 8 columns (SHORT) are read one by one.
template <bool SHORT, bool NT = false, typename T> __device__ __forceinline__ Raw8<T> load_cols(const T* row, int col, int cols) {
  if constexpr (SHORT) {
    Raw8<T> v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < cols ? row[e] : (T)0.0f;
    return v;
  } else {
    const Raw8<T>* p = reinterpret_cast<const Raw8<T>*>(row + min(col, cols - 8));
    return NT ? __builtin_nontemporal_load(p) : *p;
  }
}
template <bool SHORT, typename T> __device__ __forceinline__ f32x8 used_cols(const Raw8<T>& raw, int n) {
  f32x8 v = widened<T>(raw);
  if (!SHORT && n < 8) {
    asm volatile("");      // (kept behind its branch: made into selects for every lane, this is a fifth of a kernel's arithmetic)
    const int s = 8 - n;
#pragma unroll
    for (int step = 4; step >= 1; step >>= 1)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = s & step ? (e + step < 8 ? v[e + step] : 0.0f) : v[e];
  }
  return v;
}
template <bool NT = false, typename T> __device__ __forceinline__ void store_cols(T* p, const f32x8& v, int n) {
  if (n >= 8) {
    Raw8<T>* to = reinterpret_cast<Raw8<T>*>(p);
    const Raw8<T> o = rounded<T>(v);
    if (NT) __builtin_nontemporal_store(o, to); else *to = o;
  } else {
    // four, two and one of them, as n has them (a wave that stores its last lane's up to 7 one by one waits for 7 stores)
    typedef T T4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    typedef T T2 __attribute__((ext_vector_type(2), aligned(sizeof(T))));
    const bool behind4 = n & 4, behind2 = n & 2;
    if (n & 4) *reinterpret_cast<T4*>(p) = T4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    if (n & 2) *reinterpret_cast<T2*>(p + (n & 4)) = T2{(T)(behind4 ? v[4] : v[0]), (T)(behind4 ? v[5] : v[1])};
    const float last = behind4 ? (behind2 ? v[6] : v[4]) : behind2 ? v[2] : v[0];
    if (n & 1) p[n & 6] = (T)last;
  }
}

}  // namespace ptx
