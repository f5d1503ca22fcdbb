// Numbers held in 4 bits: a group of consecutive numbers shares a scale s and a middle z (both bfloat16), and code c, 0..15,
// stands for  z + (c - 7.5) s.  With c - 7.5 instead of c the stored z is the middle of the group's range, which is smaller than its
// ends and so rounded to bfloat16 with the smaller error.
#pragma once

#include "common.cuh"
#include <math.h>

struct GroupCode { float s, z; };   // the values of the two stored bfloat16 numbers

// s = bf16((hi - lo) / 15), z = bf16((hi + lo) / 2): 32-bit operations rounded one by one, so that every implementation of these lines gets the
// same bits.  A group with an infinity or NaN in it has no scale: it stands for NaN as a whole.
__device__ __forceinline__ GroupCode group_code(float lo, float hi) {
  const float s = __fdiv_rn(__fadd_rn(hi, -lo), 15.f), z = __fmul_rn(__fadd_rn(hi, lo), 0.5f);
  GroupCode g = {rnd<__nv_bfloat16>(s), rnd<__nv_bfloat16>(z)};
  if (!(fabsf(g.s) < INFINITY) || !(fabsf(g.z) < INFINITY)) g.s = g.z = __int_as_float(0x7fc00000);
  return g;
}
// nearest code (ties to the even one); 8 where every number of the group is the same
__device__ __forceinline__ unsigned code_of(float x, GroupCode g) {
  if (!(g.s > 0.f)) return 8u;
  const float c = rintf(__fadd_rn(__fdiv_rn(__fadd_rn(x, -g.z), g.s), 7.5f));
  return (unsigned)fminf(fmaxf(c, 0.f), 15.f);
}
__device__ __forceinline__ float value_of(unsigned c, GroupCode g) { return fmaf((float)c - 7.5f, g.s, g.z); }   // the product is exact: one rounding

__device__ __forceinline__ unsigned pack_code(GroupCode g) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(g.s, g.z);
  return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ GroupCode unpack_code(unsigned w) { return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)}; }

// Four pairs of codes as bfloat16 pairs 16 + c: the codes in bits 4i..4i+3 of the word's two halves, put into the upper mantissa bits of 16.0.
// Products over them are corrected by the group's sum of the other operand: sum (c - 7.5) x = sum (16 + c) x - 23.5 sum x.  (128 + c, with the code in
// the lowest bits, would save one shift, but its sums are six times larger than what is left of them, and so are their rounding errors.)
constexpr float CODE_BIAS = 23.5f;
__device__ __forceinline__ unsigned code_pair(unsigned w, int i) {
  const unsigned at = i == 0 ? w << 3 : w >> (4 * i - 3);
  return (at & 0x00780078u) | 0x41804180u;
}

__device__ __forceinline__ void mma_16816(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
constexpr unsigned ONES_BF16 = 0x3f803f80u;   // two ones: a product with them sums the other operand, in the places where its products are

// One output of a product, straight from its definition: sum over the inputs, in their order, of (z + (c - 7.5) s) x, for row `row` of the weights (linear4.cu has their
// layout), x(i) being the activations.  By one thread and slow: for results that are not finite.  Where one of the sums that the fast forms are made of is an infinity,
// what they add to it may be its opposite, and the NaN that they end in need not be the product's.
template <typename X> __device__ __forceinline__ float defined_product(const uint4* codes, const uint2* scales, int row, int k, int group_bits, X x) {
  const int wide = (k + 127) / 128 * 128, r = row & 7, h = row >> 3 & 1;   // inputs as laid out
  const size_t tile = row >> 4;
  codes += tile * (wide / 64) * 32 + r * 4;
  scales += tile * (wide >> group_bits) * 8 + r;
  float sum = 0.f;
#pragma unroll 1
  for (int at = 0; at < k && sum == sum; at += 16) {   // a step: word s of the four lanes of a row of its block (what is NaN stays NaN)
    const uint2 sz = scales[(at >> group_bits) * 8];
    const GroupCode g = unpack_code(h ? sz.y : sz.x);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const unsigned word = reinterpret_cast<const unsigned*>(codes + (at >> 6) * 32 + c)[at >> 4 & 3];
#pragma unroll
      for (int e = 0; e < 4; ++e) sum = fmaf(value_of(word >> (4 * (2 * (e >> 1) + h) + 16 * (e & 1)) & 15u, g), x(at + 4 * c + e), sum);
    }
  }
  return sum;
}

// ---------------------------------------------------------------------------------------------- the cache's pages
// A page of one key head is one tile of bytes: its tokens' codes, then [token][group] of (s, z).  A token's codes take ROW = 16 ceil(d / 32) bytes.
//
// Keys are the 16-row operand of S^T = K Q^T.  Token t's row: for each quarter c of a warp's lanes U = ceil(d / 32) words, word u with the eight codes that the
// lane multiplies in the steps 2u and 2u + 1 of 16 dims: dims 16 (2u + step) + 4c + e.  Nibbles of the low half: (step 0, e 0), (0, 2), (1, 0), (1, 2); of the
// high half the same with e + 1.
// Values are the transposed operand of O^T = V^T P^T.  16 tokens are a tile of 32 lanes x U x 8 bytes: lane (r, c) holds, for the dims
// 16 (2u + step) + 2r + h, the tokens 2c, 2c + 1, 2c + 8, 2c + 9, 16 bits each: nibble 2 step + h.  A token writes whole 16-bit words.
__host__ __device__ constexpr int kv4_units(int d) { return (d + 31) / 32; }
__host__ __device__ constexpr int kv4_row_bytes(int d) { return 16 * kv4_units(d); }
__host__ __device__ constexpr size_t kv4_tile_bytes(int page, int d, int group) { return (size_t)page * (kv4_row_bytes(d) + 4 * (d / group)); }
__device__ __forceinline__ int kv4_value_at(int t, int r, int u, int units) {   // where token t of a page has its 16 bits for lane row r and unit u
  const int k = t & 15, c = (k & 7) >> 1, i = (k & 1) + 2 * (k >> 3);
  return (t >> 4) * 256 * units + ((r * 4 + c) * units + u) * 8 + 2 * i;
}
