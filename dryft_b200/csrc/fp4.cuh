// Microscaled 4-bit floating point: a number is one of 0, 1/2, 1, 3/2, 2, 3, 4, 6 or minus that (code: sign, two bits of exponent, one of fraction), times the scale of
// its group of consecutive numbers of a row.  Every step is a 32-bit one, |.| are magnitudes of finite numbers, roundings to the nearest, ties to even:
//
//   MX: groups of 32, s = 2^max(floor(log2 max|group|) - 2, -127) (the shared exponents of the OCP microscaling formats), c = fp4(x / s), value c s
//   NV: groups of 16, g = max(max|row| / 2688, 2^-112), u = 1 / (6 g), s = e4m3(max|group| u), r = 1 / (s g) (0 where s = 0), c = fp4(x r), value (c s) g
//
// (2688 = 6 x 448, the largest number and the largest scale; 2^-112 keeps 1 / (s g) finite.)  Magnitudes above 6 become 6.  A group with an infinity or a NaN has the
// scale NaN and codes of 1.  A row's form depends on that row alone.
//
// Layout: blocks of 128 rows by 256 inputs, block (row / 128, input / 256) behind one another along the inputs.  A block is its scales, then its codes, as the tensor cores take
// them, so that a copy of consecutive bytes fills a stage of shared memory (no tensor maps): codes in rows of 128 bytes, two a byte, the lower input in the lower half, 16-byte
// pieces exchanged as the 128-byte swizzle has them; scales in words of four (64 inputs of NV, 128 of MX), 512 bytes for 128 rows: row r's word at 16 (r % 32) + 4 (r / 32).
// Inputs behind the last are zeros with scales of zero (MX: 2^-127); rows behind the last are whatever was there: what the tensor cores make of them is nobody's result.
#pragma once

#include "common.cuh"

namespace fp4 {
enum Kind { MX = 0, NV = 1 };
constexpr int ROWS = 128, INPUTS = 256, CODE_BYTES = ROWS * INPUTS / 2;
template <int KIND> struct Format {
  static constexpr int GROUP = KIND == NV ? 16 : 32;
  static constexpr int WORD_INPUTS = 4 * GROUP, WORDS = INPUTS / WORD_INPUTS;   // inputs that share a word of scales; words of a block's row
  static constexpr int SCALE_BYTES = 512 * WORDS, BLOCK_BYTES = SCALE_BYTES + CODE_BYTES;
};
__host__ __device__ __forceinline__ int blocks_of(int k) { return (k + INPUTS - 1) / INPUTS; }
// of 16 inputs `unit` (0..15 in a block) of row r (0..127): eight bytes
__host__ __device__ __forceinline__ int code_at(int r, int unit) { return r * 128 + (((unit >> 1) ^ (r & 7)) << 4) + (unit & 1) * 8; }
__host__ __device__ __forceinline__ int scale_word_at(int r, int word) { return word * 512 + (r & 31) * 16 + (r >> 5) * 4; }

constexpr unsigned char NV_NAN = 0x7f, MX_NAN = 0xff;
__device__ __forceinline__ float scale_value(unsigned byte, bool nv) {
  if (nv) {
    unsigned h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((unsigned short)byte));
    float f;
    asm("{ .reg .b16 lo, hi; mov.b32 {lo, hi}, %1; cvt.f32.f16 %0, lo; }" : "=f"(f) : "r"(h2));
    return f;
  }
  return byte == MX_NAN ? __uint_as_float(0x7fffffffu) : byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);   // (2^-127 has no exponent bits)
}
constexpr int UNIT = 16, BLOCK_UNITS = INPUTS / UNIT;   // numbers that a lane has at a time; units of a block's row
// Sixteen numbers as they lie in memory.
template <typename T> struct Raw { unsigned w[UNIT * sizeof(T) / 4]; };
__device__ __forceinline__ float number(const Raw<__nv_bfloat16>& r, int i) { return __uint_as_float(i & 1 ? r.w[i / 2] & 0xffff0000u : r.w[i / 2] << 16); }
__device__ __forceinline__ float number(const Raw<float>& r, int i) { return __uint_as_float(r.w[i]); }

// From column c on; zeros behind column k.  Through L2 (`ld_prev`): the launch before this one may have written them.
template <typename T> __device__ __forceinline__ Raw<T> load(const T* row, int c, int k, bool words) {
  Raw<T> r;
  constexpr int N = UNIT * sizeof(T) / 16;
  if (words && c + UNIT <= k) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint4 a = ld_prev(reinterpret_cast<const uint4*>(row + c) + i);
      r.w[4 * i] = a.x;
      r.w[4 * i + 1] = a.y;
      r.w[4 * i + 2] = a.z;
      r.w[4 * i + 3] = a.w;
    }
    return r;
  }
#pragma unroll
  for (int i = 0; i < 4 * N; ++i) r.w[i] = 0;
#pragma unroll
  for (int i = 0; i < UNIT; ++i)
    if (c + i < k) {
      if (sizeof(T) == 4) r.w[i] = __ldcg(reinterpret_cast<const unsigned*>(row) + c + i);
      else r.w[i / 2] |= (unsigned)__ldcg(reinterpret_cast<const unsigned short*>(row) + c + i) << (i & 1) * 16;
    }
  return r;
}
// The same where rows begin anywhere: the 16-byte words that hold the numbers, shifted.  (A word that holds one byte of a row can be read; a number a load would cross memory 8 times.)
template <typename T> __device__ __forceinline__ Raw<T> load_shifted(const T* row, int c, int k) {
  constexpr int N = UNIT * sizeof(T) / 4;
  Raw<T> r;
  unsigned w[N + 4];
  const uintptr_t at = reinterpret_cast<uintptr_t>(row + c), end = reinterpret_cast<uintptr_t>(row + min(c + UNIT, k));
  const uint4* const p = reinterpret_cast<const uint4*>(at & ~(uintptr_t)15);
#pragma unroll
  for (int i = 0; i < (N + 4) / 4; ++i) {
    const uint4 a = c < k && reinterpret_cast<uintptr_t>(p + i) < end ? ld_prev(p + i) : make_uint4(0u, 0u, 0u, 0u);
    w[4 * i] = a.x;
    w[4 * i + 1] = a.y;
    w[4 * i + 2] = a.z;
    w[4 * i + 3] = a.w;
  }
#pragma unroll
  for (int i = 0; i < N + 2; ++i) w[i] = at & 8 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < N + 1; ++i) w[i] = at & 4 ? w[i + 1] : w[i];
#pragma unroll
  for (int i = 0; i < N; ++i) r.w[i] = __funnelshift_r(w[i], w[i + 1], at & 2 ? 16 : 0);
  const int left = k - c;   // numbers of the row; zeros behind them
  if (left < UNIT) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      constexpr int PER = 4 / sizeof(T);
      if (PER * i >= left) r.w[i] = 0;
      else if (PER == 2 && 2 * i + 1 >= left) r.w[i] &= 0xffffu;
    }
  }
  return r;
}
// SILU: the row holds gate numbers, then as many others: silu(gate) rounded, times the other, rounded (the points of `silu_mul`).
template <typename T, bool SILU, bool SHIFTED = false> __device__ __forceinline__ Raw<T> load_unit(const T* row, int c, int k, bool words) {
  Raw<T> r = SHIFTED ? load_shifted(row, c, k) : load(row, c, k, words);
  if constexpr (SILU) {
    const Raw<T> up = SHIFTED ? load_shifted(row + k, c, k) : load(row + k, c, k, words);
#pragma unroll
    for (int i = 0; i < UNIT / 2; ++i) {
      float v[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) v[e] = rnd<__nv_bfloat16>(silu_fast(number(r, 2 * i + e))) * number(up, 2 * i + e);
      const __nv_bfloat162 two = __floats2bfloat162_rn(v[0], v[1]);
      r.w[i] = *reinterpret_cast<const unsigned*>(&two);
    }
  }
  return r;
}

struct Size { unsigned most; bool bad; };   // the bits of the largest finite magnitude as a 32-bit number (bits of magnitudes are in their order); whether one is not finite
template <typename T> __device__ __forceinline__ Size size_of(const Raw<T>& r) {
  unsigned most = 0;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < UNIT / 2; ++i)   // (a NaN stays one; an integer maximum of the masked bits: 1 to 4% of a rounding longer)
      asm("{ .reg .b32 a; abs.bf16x2 a, %1; max.NaN.bf16x2 %0, %0, a; }" : "+r"(most) : "r"(r.w[i]));
    most = max(most & 0xffff0000u, most << 16);
  } else {
#pragma unroll
    for (int i = 0; i < UNIT; ++i) most = max(most, r.w[i] & 0x7fffffffu);
  }
  if (most < 0x7f800000u) return {most, false};
  most = 0;
#pragma unroll
  for (int i = 0; i < UNIT; ++i) {
    const unsigned a = __float_as_uint(number(r, i)) & 0x7fffffffu;
    if (a < 0x7f800000u) most = max(most, a);
  }
  return {most, true};
}
__device__ __forceinline__ float row_factor(unsigned most) { return fmaxf(__fdiv_rn(__uint_as_float(most), 2688.f), __uint_as_float((127u - 112u) << 23)); }
// codes of eight numbers times r, the first in the lowest four bits
template <typename T> __device__ __forceinline__ unsigned codes8(const Raw<T>& x, int first, float r) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = number(x, first + i) * r;
  unsigned w;
  asm("{ .reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3}; }"
      : "=r"(w) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return w;
}

// A unit's codes, and the word of scales that it begins (where it begins one: NV every fourth unit, MX every eighth).  Neighbouring lanes have neighbouring units; all 32 take part.
// factor, u: of the row (NV).
template <int KIND, typename T> __device__ __forceinline__ uint2 round_unit(const Raw<T>& r, float factor, float u, unsigned& word) {
  Size s = size_of(r);
  unsigned byte;
  float by;
  if (KIND == NV) {
    unsigned short two;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(0.f), "f"(__uint_as_float(s.most) * u));
    byte = two & 0xff;
    by = byte == 0 ? 0.f : __frcp_rn(scale_value(byte, true) * factor);
    if (s.bad) byte = NV_NAN;
    word = byte | __shfl_down_sync(0xffffffffu, byte, 1) << 8;
    word |= __shfl_down_sync(0xffffffffu, word, 2) << 16;
  } else {
    s.most = max(s.most, __shfl_xor_sync(0xffffffffu, s.most, 1));
    s.bad |= __shfl_xor_sync(0xffffffffu, (int)s.bad, 1) != 0;
    byte = max((int)(s.most >> 23) - 2, 0);
    by = __uint_as_float((254u - byte) << 23);   // 1 / s: 2^127 at the most
    if (s.bad) byte = MX_NAN;
    word = byte | __shfl_down_sync(0xffffffffu, byte, 2) << 8;
    word |= __shfl_down_sync(0xffffffffu, word, 4) << 16;
  }
  return s.bad ? make_uint2(0x22222222u, 0x22222222u) : make_uint2(codes8(r, 0, by), codes8(r, 8, by));
}

// 32 bytes: a whole sector a lane
__device__ __forceinline__ void st_words8(void* to, const unsigned* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
}  // namespace fp4
