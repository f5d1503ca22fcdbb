// Microscaled 4-bit floating point: a number is one of 0, 1/2, 1, 3/2, 2, 3, 4, 6 or minus that (code: sign, two bits of exponent, one of fraction), times the scale of
// its group of consecutive numbers of a row.  Every step is a 32-bit one, |.| are magnitudes of finite numbers, roundings to the nearest, ties to even:
//
//   MX: groups of 32, s = 2^max(floor(log2 max|group|) - 2, -127) (the shared exponents of the OCP microscaling formats), c = fp4(x / s), value c s
//   NV: groups of 16, g = max(max|row| / 2688, 2^-112), u = 1 / (6 g), s = e4m3(max|group| u), r = 1 / (s g) (0 where s = 0), c = fp4(x r), value (c s) g
//
// (2688 = 6 x 448, the largest number and the largest scale; 2^-112 keeps 1 / (s g) finite.)  Magnitudes above 6 become 6.  A group with an infinity or a NaN has the
// scale NaN and codes of 1.  A row's form depends on that row alone, so a result does not depend on which rows a step has.
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
// 32 bytes: a whole sector a lane
__device__ __forceinline__ void st_words8(void* to, const unsigned* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
}  // namespace fp4
