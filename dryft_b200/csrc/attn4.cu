// Attention of query rows over the paged cache held in 4 bits (four_bit.cuh).  Compiled per model with -DDRYFT_HEAD_DIM, -DDRYFT_GROUP (query heads per key
// head), -DDRYFT_PAGE and -DDRYFT_BITS_GROUP (numbers that share a scale).
//
// Row n at position p of slot s sees the keys j with  max(0, p + 1 - window) <= j <= p  (window <= 0: all of them); a row of slot -1 is padding, its output zeros.
// A block takes up to eight query heads of a (row, key head) and one split of its keys.  Splits are whole tiles of 16 keys.  Up to 16 splits are the blocks of
// a thread-block cluster and meet in its shared memory; more leave (acc, m, l) in memory and a second launch joins them.  Either way in the splits' order.
#include "four_bit.cuh"

#include <cuda_fp16.h>

#if !defined(DRYFT_HEAD_DIM) || !defined(DRYFT_GROUP) || !defined(DRYFT_PAGE) || !defined(DRYFT_BITS_GROUP)
#error "compile with -DDRYFT_HEAD_DIM=.. -DDRYFT_GROUP=.. -DDRYFT_PAGE=.. -DDRYFT_BITS_GROUP=.."
#endif

namespace {
constexpr int D = DRYFT_HEAD_DIM, G = DRYFT_GROUP, PAGE = DRYFT_PAGE, BG = DRYFT_BITS_GROUP;
constexpr int UNITS = kv4_units(D), ROW = kv4_row_bytes(D), GROUPS = D / BG;
constexpr size_t TILE = kv4_tile_bytes(PAGE, D, BG);
static_assert(D % 16 == 0 && D <= 256 && D % BG == 0 && BG % 16 == 0 && BG <= 128, "head size in steps of 16, whole groups");
static_assert(G >= 1 && G <= 16 && PAGE % 16 == 0, "1..16 query heads per key head, pages of whole tiles of 16 tokens");

__device__ __forceinline__ void wait_before_reading() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

struct Span { int first, end; };   // keys of a split: whole tiles of 16, `least` of them at least, cut at the row's first and last key
__device__ __forceinline__ Span span_of(int pos, int window, int split, int splits, int least) {
  const int lo = window > 0 && pos + 1 > window ? pos + 1 - window : 0;
  const int t0 = lo / 16, tiles = pos / 16 + 1 - t0, per = max(least, (tiles + splits - 1) / splits);
  const int a = t0 + min(tiles, split * per), b = t0 + min(tiles, (split + 1) * per);
  return {max(lo, a * 16), min(pos + 1, b * 16)};
}

// What a block knows of its work: head tile `ht` (of eight query heads) of a key head of a row, and its split.
constexpr int HEAD_TILES = (G + 7) / 8, HEADS = G < 8 ? G : 8;   // (query heads of a block; the last tile may have fewer)
struct Work { int n, head, ht, split, n_kv, splits; };
__device__ __forceinline__ Work work_of_block() {   // grid (splits, key heads x head tiles, rows)
  return {(int)blockIdx.z, (int)blockIdx.y / HEAD_TILES, (int)blockIdx.y % HEAD_TILES, (int)blockIdx.x, (int)gridDim.y / HEAD_TILES, (int)gridDim.x};
}

// ---------------------------------------------------------------------------------------------- bfloat16: tensor cores
// S^T = K Q^T and O^T = V^T P^T on mma.sync.m16n8k16, the codes straight out of the cache's words: keys' as bfloat16 16 + c (`code_pair`), values' as float16 c - 8:
//   score  = s_k (sum (16 + c) q - 23.5 sum q) + z_k sum q          group by group, in 32 bits; sum q is the query's own
//   output = sum p' (c - 8) / unit + sum p (z_v + s_v / 2)          p' = fp16(p s_v unit): the weight rounded with its scale, by up to 2^-11
// `unit` is a power of two that keeps p' between float16's ends: set when a tile's scales are larger than all before it (the first tile's are), so a weight with a
// scale is off by up to 2^-29 of the largest scale, where that is more than 2^-11 of its own (scales 2^18 apart).  Scores, running maximum and sums are 32-bit.  (Weights in bfloat16 and values as 16 + c, corrected by
// -23.5 sum p': off by 0.0023 of the whole, not 0.0017, which the result's own rounding is; and the tensor cores cut sums off, not round them, which took another
// 0.0013 of sums three times as large over 128 tiles.)
// A warp walks tiles of 16 keys of its own, copied STAGES - 1 tiles ahead into its own ring.  The maximum
// of a column follows the scores only when one exceeds it by more than 2^8: what is summed stays below 2^8 times the number of keys.
// What bounds it: issue.  A tile is some 410 instructions of its warp, 212 of them on the pipe for logic, which takes one every other cycle (taking 128 codes a lane
// apart is half of those): with four warps on a scheduler that pipe is 67% busy and a tile takes 0.39 us of the scheduler.  64 rows of up to 8,192
// keys, 32 / 8 heads of 128: 96 us, 3,250 GB/s; one row of 16,383 keys, 64 / 8 heads: 17 us (16 us by way of memory, and a second launch on the host); eight rows of
// 650 keys 8 us; one, 7.  Sixteen warps a block: 10.1 us for the eight rows; two tiles unrolled: as before.
typedef __nv_bfloat16 bf16;
constexpr int STEPS = D / 16, UNIT = PAGE % 32 ? 1 : 2, STAGES = D <= 128 ? 4 / UNIT : 2, MOST_SPLITS = 16;   // UNIT: tiles that are copied together
constexpr int CODES = 256 * UNITS, SCALES = 64 * GROUPS, STAGE = UNIT * 2 * (CODES + SCALES);   // bytes of a tile's keys (or values), of their scales; of a stage
constexpr int PART = STEPS * 128;                                                          // floats of a warp's O^T: [step][lane][4]
template <int WARPS> struct Block {
  static constexpr size_t RING = (size_t)WARPS * STAGES * STAGE, JOIN = (size_t)WARPS * PART * 4, TOP_AT = RING > JOIN ? RING : JOIN;
  static constexpr size_t SMEM = TOP_AT + (WARPS * 16 + 16) * 4;                           // ... then the warps' maxima and sums, and the block's
  static constexpr int AT_ONCE = D <= 128 ? 16 / WARPS : 8 / WARPS;                        // blocks a multiprocessor that the registers leave room for
};

__device__ __forceinline__ unsigned transposed(unsigned v) {   // an 8 x 8 fragment of 16-bit values
  unsigned r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// The codes of a word of values, less 8, as four pairs of float16: two of the four places of a half word lie in the mantissa as they are, above 1024 (c in its lowest
// bits) and above 64 (c in bits 4..7), the other two a byte further up.  (A difference of float16 numbers that is exact.)
__device__ __forceinline__ unsigned half_sub(unsigned x, unsigned y) {
  unsigned r;
  asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
  return r;
}
__device__ __forceinline__ void codes_less_8(unsigned (&v)[4], unsigned w) {
  constexpr unsigned BY_1 = 0x64006400u, BY_16 = 0x54005400u, LESS_1 = 0x64086408u, LESS_16 = 0x54805480u;   // 1024 and 64, 1032 and 72
  const unsigned u = w >> 8;
  v[0] = half_sub((w & 0x000f000fu) | BY_1, LESS_1);
  v[1] = half_sub((w & 0x00f000f0u) | BY_16, LESS_16);
  v[2] = half_sub((u & 0x000f000fu) | BY_1, LESS_1);
  v[3] = half_sub((u & 0x00f000f0u) | BY_16, LESS_16);
}
__device__ __forceinline__ void mma_16816_half(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned half_two(float x, float y) {
  const __half2 v = __floats2half2_rn(x, y);
  return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ float reciprocal(float power_of_two) { return __uint_as_float(0x7f000000u - __float_as_uint(power_of_two)); }   // 2^-126 to 2^126
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void copy16(unsigned to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from)); }
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ unsigned in_block(unsigned at, int block) {   // the same place of another block of the cluster
  unsigned r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(block));
  return r;
}
__device__ __forceinline__ float4 cluster_load4(unsigned at) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}
// N words from shared memory, in as few loads as their alignment (that of N words) allows
template <int N> __device__ __forceinline__ void load_words(unsigned (&w)[N], const unsigned char* from) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(from)[i];
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const uint2 v = reinterpret_cast<const uint2*>(from)[i];
      w[2 * i] = v.x; w[2 * i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const unsigned*>(from)[i];
  }
}

// Where a column's maximum starts: below every score but -inf, and what -inf is above it is -inf, not NaN.
constexpr float LOWEST = -3.402823466e38f;

// What a warp keeps of its eight columns (query heads); a lane has the columns 2c and 2c + 1, and in `acc` the dims 16 j + 2r and + 1 of both.
struct Columns {
  float acc[STEPS][4], off[GROUPS][2], top[2], sum[2];
  float unit;   // what `acc` is in, beside the scales: the warp's, 2^120 at most
};
constexpr float UNIT_MOST = 1.329227995784916e36f;   // 2^120
// A lane's scales times the unit come to 255 at most (2^8 times that is a float16); where they come to more, the unit is set so that the largest becomes 2^WIDE to twice that:
// all 2 GROUPS of a lane come to 128 at most then, and follow up to twice that size without another look.
constexpr float SCALES_MOST = 255.f;
constexpr unsigned WIDE = GROUPS <= 1 ? 5 : GROUPS <= 2 ? 4 : GROUPS <= 4 ? 3 : GROUPS <= 8 ? 2 : 1;

// A tile of 16 keys.  EDGE: keys may be out of the row's sight; such a key may hold anything, so its scales are taken for zeros.
template <bool EDGE>
__device__ __forceinline__ void tile_of_keys(Columns& o, const unsigned char* k, const unsigned char* k_scales, const unsigned char* v, const unsigned char* v_scales,
                                             const uint2 (&qf)[STEPS], const float (&qs)[GROUPS][2], float scale2, int key0, Span keys) {
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const bool seen0 = !EDGE || (key0 + r >= keys.first && key0 + r < keys.end), seen1 = !EDGE || (key0 + r + 8 >= keys.first && key0 + r + 8 < keys.end);
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  {
    unsigned lo[UNITS], hi[UNITS], lo_s[GROUPS], hi_s[GROUPS];
    load_words<UNITS>(lo, k + r * ROW + c * UNITS * 4);
    load_words<UNITS>(hi, k + (r + 8) * ROW + c * UNITS * 4);
    load_words<GROUPS>(lo_s, k_scales + r * GROUPS * 4);
    load_words<GROUPS>(hi_s, k_scales + (r + 8) * GROUPS * 4);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      float part[4] = {-CODE_BIAS * qs[g][0], -CODE_BIAS * qs[g][1], -CODE_BIAS * qs[g][0], -CODE_BIAS * qs[g][1]};
#pragma unroll
      for (int j = g * BG / 16; j < (g + 1) * BG / 16; ++j) {
        const int h = 2 * (j & 1);
        mma_16816(part, code_pair(lo[j / 2], h), code_pair(hi[j / 2], h), code_pair(lo[j / 2], h + 1), code_pair(hi[j / 2], h + 1), qf[j].x, qf[j].y);
      }
      const GroupCode a = unpack_code(lo_s[g]), b = unpack_code(hi_s[g]);
      s[0] = fmaf(a.s, part[0], fmaf(a.z, qs[g][0], s[0]));
      s[1] = fmaf(a.s, part[1], fmaf(a.z, qs[g][1], s[1]));
      s[2] = fmaf(b.s, part[2], fmaf(b.z, qs[g][0], s[2]));
      s[3] = fmaf(b.s, part[3], fmaf(b.z, qs[g][1], s[3]));
    }
  }
  if (EDGE) {
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = (i < 2 ? seen0 : seen1) ? s[i] * scale2 : -INFINITY;
    scale2 = 1.f;
  }
  // the values' (s, z), in registers or, where they are many, read where they are used
  constexpr bool HELD = GROUPS <= 4;
  unsigned lo_s[HELD ? GROUPS : 1], hi_s[HELD ? GROUPS : 1];
  if constexpr (HELD) {
    load_words(lo_s, v_scales + r * GROUPS * 4);
    load_words(hi_s, v_scales + (r + 8) * GROUPS * 4);
  }
  const auto value_scale = [&](int g, int half) {
    if constexpr (HELD)
      return unpack_code((half ? seen1 : seen0) ? (half ? hi_s[g] : lo_s[g]) : 0u);
    else
      return unpack_code((half ? seen1 : seen0) ? reinterpret_cast<const unsigned*>(v_scales)[(r + 8 * half) * GROUPS + g] : 0u);
  };
  float all = 0.f;   // of the lane's scales, in units
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) all = fmaf(value_scale(g, 0).s, o.unit, fmaf(value_scale(g, 1).s, o.unit, all));
  float d[4];   // powers of two above the maximum
#pragma unroll
  for (int i = 0; i < 4; ++i) d[i] = fmaf(s[i], scale2, -o.top[i & 1]);
  if (__any_sync(0xffffffffu, (fmaxf(fmaxf(d[0], d[1]), fmaxf(d[2], d[3])) > 8.f) | !(all <= SCALES_MOST))) {
    float most = 0.f;   // of the tile's scales (NaN is passed over)
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) most = fmaxf(most, fmaxf(value_scale(g, 0).s, value_scale(g, 1).s));
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, x));
    const float per_unit = reciprocal(o.unit);
    if (most * o.unit >= (float)(2 << WIDE)) o.unit = __uint_as_float((254u + WIDE - (__float_as_uint(most) >> 23)) << 23);
    const float less = o.unit * per_unit;   // the new unit in old ones, exact
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float m = fmaxf(o.top[i], fmaxf(s[i] * scale2, s[i + 2] * scale2));
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
      const float lower = exp2_fast(o.top[i] - m);
      o.top[i] = m;
      o.sum[i] *= lower;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) o.off[g][i] *= lower;
#pragma unroll
      for (int j = 0; j < STEPS; ++j) {
        o.acc[j][i] *= lower * less;
        o.acc[j][i + 2] *= lower * less;
      }
      d[i] = fmaf(s[i], scale2, -m);
      d[i + 2] = fmaf(s[i + 2], scale2, -m);
    }
  }
  float p[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    p[i] = exp2_fast(d[i]);
    o.sum[i & 1] += p[i];
  }
  unsigned vw[2 * UNITS];
  load_words<2 * UNITS>(vw, v + lane * UNITS * 8);
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const GroupCode a = value_scale(g, 0), b = value_scale(g, 1);
    const float as = a.s * o.unit, bs = b.s * o.unit;
    unsigned x[4], y[4];
    const unsigned b0 = transposed(half_two(p[0] * as, p[1] * as)), b1 = transposed(half_two(p[2] * bs, p[3] * bs));
    const float az = fmaf(0.5f, a.s, a.z), bz = fmaf(0.5f, b.s, b.z);   // what code 8 stands for
    o.off[g][0] = fmaf(p[0], az, fmaf(p[2], bz, o.off[g][0]));
    o.off[g][1] = fmaf(p[1], az, fmaf(p[3], bz, o.off[g][1]));
#pragma unroll
    for (int j = g * BG / 16; j < (g + 1) * BG / 16; ++j) {
      const int h = 2 * (j & 1);
      if (h == 0 || j == g * BG / 16) {
        codes_less_8(x, vw[j / 2 * 2]);
        codes_less_8(y, vw[j / 2 * 2 + 1]);
      }
      mma_16816_half(o.acc[j], x[h], x[h + 1], y[h], y[h + 1], b0, b1);
    }
  }
}

template <int WARPS>
__global__ void __launch_bounds__(WARPS * 32, Block<WARPS>::AT_ONCE) attn4_mma_kernel(const bf16* q, const unsigned char* k_pages, const unsigned char* v_pages,
                                                                                      const int* __restrict__ page_table, int max_pages,
                                                                                      const int* __restrict__ tok_slot, const int* __restrict__ tok_pos, bf16* out,
                                                                                      float* part_o, float* part_ml, int cluster, int least, float scale, int window) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
  const Work w = work_of_block();
  const int n_kv = w.n_kv, splits = w.splits;
  const int slot = tok_slot[w.n], pos = tok_pos[w.n], heads = min(8, G - 8 * w.ht);
  const size_t head0 = ((size_t)w.n * n_kv + w.head) * G + 8 * w.ht;   // the block's first query head
  let_next_launch_in();
  if (slot < 0) {                                                      // (the whole cluster)
    wait_before_reading();
    if (w.split == 0)
      for (int i = threadIdx.x; i < heads * D; i += WARPS * 32) out[head0 * D + i] = from_f32<bf16>(0.f);
    return;
  }
  const Span keys = span_of(pos, window, w.split, splits, least);
  // the warp's units of UNIT tiles: its share of the split's, one behind the other
  constexpr int KEYS = UNIT * 16;
  const int u0 = keys.first / KEYS, units = keys.end > keys.first ? (keys.end + KEYS - 1) / KEYS - u0 : 0;
  const int a = u0 + units * warp / WARPS, b = u0 + units * (warp + 1) / WARPS;

  Columns o;
  o.unit = UNIT_MOST;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    o.top[i] = LOWEST;
    o.sum[i] = 0.f;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) o.off[g][i] = 0.f;
#pragma unroll
    for (int j = 0; j < STEPS; ++j) o.acc[j][i] = o.acc[j][i + 2] = 0.f;
  }
  if (units == 0 && splits > 1 && !cluster) {   // a split without keys: sums of zero, which the join does not look behind
    wait_before_reading();
    if (threadIdx.x < heads) *reinterpret_cast<float2*>(part_ml + ((head0 + threadIdx.x) * splits + w.split) * 2) = make_float2(LOWEST, 0.f);
    return;
  }
  constexpr int PER_PAGE = PAGE / KEYS;
  const int* const pages = page_table + (size_t)slot * max_pages;
  int page0 = a / PER_PAGE, held = 0;   // page numbers of 32 pages, one a lane
  auto fetch = [&] { held = a < b && page0 + lane <= (b - 1) / PER_PAGE ? pages[page0 + lane] : 0; };
  fetch();
  wait_before_reading();
  if (a < b) {
    unsigned char* const ring = smem + warp * STAGES * STAGE;
    const unsigned ring_at = (unsigned)__cvta_generic_to_shared(ring) + lane * 16;
    constexpr int C = UNIT * CODES, S = UNIT * SCALES;   // a stage: keys' codes, values' codes, keys' scales, values' scales
    const unsigned char *kp = nullptr, *vp = nullptr;    // the next unit's codes, less what a unit has, and its scales in the same way
    const unsigned char *ksp = nullptr, *vsp = nullptr;
    int ask = a, put = 0;
    auto request = [&] {
      if (ask < b) {
        if (ask % PER_PAGE == 0 || ask == a) {
          if (ask / PER_PAGE - page0 >= 32) {
            page0 = ask / PER_PAGE;
            fetch();
          }
          const size_t at = ((size_t)__shfl_sync(0xffffffffu, held, ask / PER_PAGE - page0) * n_kv + w.head) * TILE + lane * 16;
          kp = k_pages + at + ask % PER_PAGE * C;
          vp = v_pages + at + ask % PER_PAGE * C;
          ksp = k_pages + at + ROW * PAGE + ask % PER_PAGE * S;
          vsp = v_pages + at + ROW * PAGE + ask % PER_PAGE * S;
        }
        const unsigned to = ring_at + put * STAGE;
#pragma unroll
        for (int i = 0; i < C; i += 512)
          if (C - i >= 512 || i + lane * 16 < C) {
            copy16(to + i, kp + i);
            copy16(to + C + i, vp + i);
          }
#pragma unroll
        for (int i = 0; i < S; i += 512)
          if (S - i >= 512 || i + lane * 16 < S) {
            copy16(to + 2 * C + i, ksp + i);
            copy16(to + 2 * C + S + i, vsp + i);
          }
        kp += C;
        vp += C;
        ksp += S;
        vsp += S;
        put = put + 1 == STAGES ? 0 : put + 1;
        ++ask;
      }
      asm volatile("cp.async.commit_group;");
    };
#pragma unroll 1
    for (int i = 0; i < STAGES - 1; ++i) request();

    // the queries as column operand: head r's dims 16 j + 4c + e; their sums over the groups, of heads 2c and 2c + 1
    uint2 qf[STEPS];
    float qs[GROUPS][2];
#pragma unroll
    for (int j = 0; j < STEPS; ++j)
      qf[j] = r < heads ? __ldcg(reinterpret_cast<const uint2*>(q + (head0 + r) * D + 16 * j + 4 * c)) : make_uint2(0, 0);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = g * BG / 16; j < (g + 1) * BG / 16; ++j) mma_16816(s, ONES_BF16, ONES_BF16, ONES_BF16, ONES_BF16, qf[j].x, qf[j].y);
      qs[g][0] = s[0];
      qs[g][1] = s[1];
    }
    const float scale2 = scale * 1.4426950408889634f;   // scores in powers of two

    const unsigned char* st = ring;
#pragma unroll 1
    for (int u = a; u < b; ++u) {
      __syncwarp();   // every lane has read the stage that the next request writes
      request();
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1));
      __syncwarp();
      if (u * KEYS >= keys.first && u * KEYS + KEYS <= keys.end) {
#pragma unroll 1
        for (int i = 0; i < UNIT; ++i)
          tile_of_keys<false>(o, st + i * CODES, st + 2 * C + i * SCALES, st + C + i * CODES, st + 2 * C + S + i * SCALES, qf, qs, scale2, 0, keys);
      } else {
#pragma unroll 1
        for (int i = 0; i < UNIT; ++i)
          if (u * KEYS + i * 16 < keys.end && u * KEYS + i * 16 + 16 > keys.first)
            tile_of_keys<true>(o, st + i * CODES, st + 2 * C + i * SCALES, st + C + i * CODES, st + 2 * C + S + i * SCALES, qf, qs, scale2, u * KEYS + i * 16, keys);
      }
      st = st == ring + (STAGES - 1) * STAGE ? ring : st + STAGE;
    }
    asm volatile("cp.async.wait_group 0;");
    // what the lanes of a column have of its sums
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        o.sum[i] += __shfl_xor_sync(0xffffffffu, o.sum[i], x);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) o.off[g][i] += __shfl_xor_sync(0xffffffffu, o.off[g][i], x);
      }
  }

  // The block's part.  The warps' maxima first; then each puts its sums on the block's maximum, and they are added in the warps' order.
  float* const tops = reinterpret_cast<float*>(smem + Block<WARPS>::TOP_AT);   // [warp][8] maxima, [warp][8] sums, then the block's [8][2]
  float* const sums = tops + WARPS * 8;
  float2* const whole = reinterpret_cast<float2*>(sums + WARPS * 8);
  float4* const parts = reinterpret_cast<float4*>(smem);         // [warp][step][lane]
  if (r == 0) *reinterpret_cast<float2*>(tops + warp * 8 + 2 * c) = make_float2(o.top[0], o.top[1]);
  __syncthreads();
  float top[2] = {LOWEST, LOWEST}, by[2];
#pragma unroll
  for (int x = 0; x < WARPS; ++x) {
    const float2 m = *reinterpret_cast<const float2*>(tops + x * 8 + 2 * c);
    top[0] = fmaxf(top[0], m.x);
    top[1] = fmaxf(top[1], m.y);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) by[i] = exp2_fast(o.top[i] - top[i]);   // (1 where nothing has been seen: zeros, or the NaN of scores that are NaN)
  if (r == 0) *reinterpret_cast<float2*>(sums + warp * 8 + 2 * c) = make_float2(o.sum[0] * by[0], o.sum[1] * by[1]);
  const float per_unit = reciprocal(o.unit);
#pragma unroll
  for (int j = 0; j < STEPS; ++j) {
    const int g = 16 * j / BG;
    const float e0 = o.off[g][0], e1 = o.off[g][1];
    parts[(warp * STEPS + j) * 32 + lane] = make_float4(fmaf(o.acc[j][0], per_unit, e0) * by[0], fmaf(o.acc[j][1], per_unit, e1) * by[1],
                                                        fmaf(o.acc[j][2], per_unit, e0) * by[0], fmaf(o.acc[j][3], per_unit, e1) * by[1]);
  }
  __syncthreads();
  float l[2] = {0.f, 0.f};
#pragma unroll
  for (int x = 0; x < WARPS; ++x) {
    const float2 v = *reinterpret_cast<const float2*>(sums + x * 8 + 2 * c);
    l[0] += v.x;
    l[1] += v.y;
  }
  auto write = [&](int j, int from, float4 v, float l0, float l1) {   // dims 16 j + 2 (row of lane `from`) and the next of heads 2c, 2c + 1
    bf16* const to = out + (head0 + 2 * c) * D + 16 * j + 2 * (from >> 2);
    const float i0 = 1.f / l0, i1 = 1.f / l1;
    if (2 * c < heads) *reinterpret_cast<__nv_bfloat162*>(to) = __floats2bfloat162_rn(v.x * i0, v.z * i0);
    if (2 * c + 1 < heads) *reinterpret_cast<__nv_bfloat162*>(to + D) = __floats2bfloat162_rn(v.y * i1, v.w * i1);
  };
  for (int j = warp; j < STEPS; j += WARPS) {
    float4 v = parts[j * 32 + lane];
#pragma unroll
    for (int x = 1; x < WARPS; ++x) {
      const float4 y = parts[(x * STEPS + j) * 32 + lane];
      v = make_float4(v.x + y.x, v.y + y.y, v.z + y.z, v.w + y.w);
    }
    if (splits == 1)
      write(j, lane, v, l[0], l[1]);
    else if (cluster)
      parts[j * 32 + lane] = v;
    else {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (2 * c + i < heads)
          *reinterpret_cast<float2*>(part_o + ((head0 + 2 * c + i) * splits + w.split) * D + 16 * j + 2 * r) = i ? make_float2(v.y, v.w) : make_float2(v.x, v.z);
    }
  }
  if (splits == 1) return;
  if (warp == 0 && r == 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (cluster)
        whole[2 * c + i] = make_float2(top[i], l[i]);
      else if (2 * c + i < heads)
        *reinterpret_cast<float2*>(part_ml + ((head0 + 2 * c + i) * splits + w.split) * 2) = make_float2(top[i], l[i]);
    }
  }
  if (!cluster) return;
  // every block of the cluster joins its share of the steps' lanes, over the splits in their order
  cluster_barrier();
  {
    const unsigned whole_at = (unsigned)__cvta_generic_to_shared(whole), parts_at = (unsigned)__cvta_generic_to_shared(parts);
    for (int i = threadIdx.x * splits + w.split; i < STEPS * 32; i += WARPS * 32 * splits) {
      const int col = 2 * (i & 3);
      float m0 = LOWEST, m1 = LOWEST, l0 = 0.f, l1 = 0.f;
      float2 w0[MOST_SPLITS], w1[MOST_SPLITS];
#pragma unroll
      for (int x = 0; x < MOST_SPLITS; ++x) {
        w0[x] = w1[x] = make_float2(LOWEST, 0.f);
        if (x < splits) {
          const float4 v = cluster_load4(in_block(whole_at + col * 8, x));
          w0[x] = make_float2(v.x, v.y);
          w1[x] = make_float2(v.z, v.w);
        }
        m0 = fmaxf(m0, w0[x].x);
        m1 = fmaxf(m1, w1[x].x);
      }
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int x = 0; x < MOST_SPLITS; ++x)
        if (x < splits) {
          const float b0 = exp2_fast(w0[x].x - m0), b1 = exp2_fast(w1[x].x - m1);
          l0 = fmaf(b0, w0[x].y, l0);
          l1 = fmaf(b1, w1[x].y, l1);
          const float4 y = cluster_load4(in_block(parts_at + i * 16, x));
          v = make_float4(fmaf(b0, y.x, v.x), fmaf(b1, y.y, v.y), fmaf(b0, y.z, v.z), fmaf(b1, y.w, v.w));
        }
      bf16* const to = out + (head0 + col) * D + 16 * (i >> 5) + 2 * ((i & 31) >> 2);
      const float i0 = 1.f / l0, i1 = 1.f / l1;
      if (col < heads) *reinterpret_cast<__nv_bfloat162*>(to) = __floats2bfloat162_rn(v.x * i0, v.z * i0);
      if (col + 1 < heads) *reinterpret_cast<__nv_bfloat162*>(to + D) = __floats2bfloat162_rn(v.y * i1, v.w * i1);
    }
  }
  cluster_barrier();   // a block's shared memory stays until the others have read it
}

// ---------------------------------------------------------------------------------------------- 32-bit
// Every product is a 32-bit multiply-add (no tensor core keeps 24 bits).  A warp takes every eighth tile of 16 keys of the split, with a running maximum and sums of
// its own, joined in the warps' order behind the last one.  Scores: two lanes a key, half of the dims each.  Values: a lane keeps four dims (times QUADS) of every
// head and walks the tile's tokens, whose codes are four 8-byte words of the layout; where a head has fewer than 32 such quads, lanes share the tokens.
// A tile's codes, keys' and values', are requested before its scores are formed: what bounds the kernel is that chain (page number, codes, scores, weights, sums),
// about 2 us a tile and warp.  13 rows, windows of 100 keys, three key heads of 48: 6.4 us (13.7 with a thread a key and a thread a dim, the values' 128 loads one
// behind the other); eight rows of 500 keys, eight key heads of 128: 10 us (29.2).
constexpr int THREADS = 128, F32_WARPS = 8, QUADS = (8 * UNITS + 31) / 32, SHARE = 8 * UNITS <= 8 ? 4 : 8 * UNITS <= 16 ? 2 : 1;

__global__ void __launch_bounds__(F32_WARPS * 32) attn4_f32_kernel(const float* __restrict__ q, const unsigned char* __restrict__ k_pages,
                                                                   const unsigned char* __restrict__ v_pages, const int* __restrict__ page_table, int max_pages,
                                                                   const int* __restrict__ tok_slot, const int* __restrict__ tok_pos, float* out, float* part_o,
                                                                   float* part_ml, float scale, int window) {
  __shared__ __align__(16) float qs[HEADS][D];   // the queries, later the block's sums
  __shared__ float ps[F32_WARPS][16][HEADS], tops[F32_WARPS][HEADS], sums[F32_WARPS][HEADS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Work w = work_of_block();
  const int n_kv = w.n_kv, splits = w.splits;
  const int slot = tok_slot[w.n], pos = tok_pos[w.n], heads = min(8, G - 8 * w.ht);
  const size_t head0 = ((size_t)w.n * n_kv + w.head) * G + 8 * w.ht;
  if (slot < 0) {
    if (w.split == 0)
      for (int i = tid; i < heads * D; i += F32_WARPS * 32) out[head0 * D + i] = 0.f;
    return;
  }
  const Span keys = span_of(pos, window, w.split, splits, 1);
  for (int i = tid; i < HEADS * D; i += F32_WARPS * 32) qs[i / D][i % D] = i / D < heads ? q[head0 * D + i] : 0.f;
  __syncthreads();
  float acc[QUADS][4][HEADS], top[HEADS], sum[HEADS];
#pragma unroll
  for (int g = 0; g < HEADS; ++g) {
    top[g] = LOWEST;
    sum[g] = 0.f;
#pragma unroll
    for (int i = 0; i < QUADS; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e][g] = 0.f;
  }
  const int key = lane & 15, half = lane >> 4, part = SHARE > 1 ? lane / (8 * UNITS) : 0;
  const int* const pages = page_table + (size_t)slot * max_pages;
  for (int t = keys.first / 16 + warp; t * 16 < keys.end; t += F32_WARPS) {
    const size_t page_at = ((size_t)pages[t * 16 / PAGE] * n_kv + w.head) * TILE;
    const int in_page = t * 16 % PAGE;
    const unsigned char* const kt = k_pages + page_at;
    const unsigned char* const vt = v_pages + page_at;
    const bool seen = t * 16 + key >= keys.first && t * 16 + key < keys.end;
    // a key's codes: quarters 2 half and 2 half + 1 of its row, UNITS words each; a quad's: the tokens' words, four tokens each
    unsigned kw[2 * UNITS], ks[GROUPS];
    load_words<2 * UNITS>(kw, kt + (size_t)(in_page + key) * ROW + half * UNITS * 8);
    load_words<GROUPS>(ks, kt + (size_t)ROW * PAGE + (size_t)(in_page + key) * GROUPS * 4);
    uint2 vw[QUADS][4 / SHARE];
#pragma unroll
    for (int i = 0; i < QUADS; ++i) {
      const int at = SHARE > 1 ? lane % (8 * UNITS) : lane + 32 * i, r = at & 7, u = at >> 3;
#pragma unroll
      for (int c = 0; c < 4 / SHARE; ++c)
        vw[i][c] = u < UNITS && part < SHARE
                       ? *reinterpret_cast<const uint2*>(vt + kv4_value_at(in_page + 2 * (c + part * (4 / SHARE)), r, u, UNITS)) : make_uint2(0, 0);
    }
    float s[HEADS];
#pragma unroll
    for (int g = 0; g < HEADS; ++g) s[g] = 0.f;
#pragma unroll
    for (int step = 0; step < D / 16; ++step) {
      const GroupCode gc = unpack_code(ks[step * 16 / BG]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {   // four numbers of one step and quarter
        const unsigned word = kw[c * UNITS + step / 2] >> (8 * (step & 1));
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = value_of(word >> (4 * (e >> 1) + 16 * (e & 1)) & 15u, gc);
#pragma unroll
        for (int g = 0; g < HEADS; ++g) {
          const float4 x = *reinterpret_cast<const float4*>(&qs[g][step * 16 + 4 * (2 * half + c)]);
          s[g] = fmaf(v[0], x.x, fmaf(v[1], x.y, fmaf(v[2], x.z, fmaf(v[3], x.w, s[g]))));
        }
      }
    }
    float lower[HEADS];
#pragma unroll
    for (int g = 0; g < HEADS; ++g) {
      s[g] += __shfl_xor_sync(0xffffffffu, s[g], 16);
      s[g] = seen ? s[g] * scale : -INFINITY;
      const float m = fmaxf(top[g], warp_max(s[g]));
      lower[g] = m == top[g] ? 1.f : expf(top[g] - m);
      top[g] = m;
      const float p = s[g] == -INFINITY ? 0.f : expf(s[g] - m);
      sum[g] = fmaf(sum[g], lower[g], p);   // (of the lane's keys; either half has them)
      if (half == 0) ps[warp][key][g] = p;
#pragma unroll
      for (int i = 0; i < QUADS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e][g] *= lower[g];
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < QUADS; ++i) {
      const int u = SHARE > 1 ? lane % (8 * UNITS) >> 3 : (lane + 32 * i) >> 3;
      if (u >= UNITS || part >= SHARE) continue;
#pragma unroll
      for (int x = 0; x < 16 / SHARE; ++x) {   // word x / 4's token x % 4
        const int c = x >> 2, tok = 2 * (c + part * (4 / SHARE)) + (x & 1) + 8 * ((x >> 1) & 1), j = t * 16 + tok;
        const unsigned word = (x & 2 ? vw[i][c].y : vw[i][c].x) >> (16 * (x & 1));
        const unsigned* const sz = reinterpret_cast<const unsigned*>(vt + (size_t)ROW * PAGE) + (in_page + tok) * GROUPS;
        const bool there = j >= keys.first && j < keys.end;   // (what is out of sight may be anything)
        const int g0 = 32 * u / BG, g1 = min(GROUPS - 1, (32 * u + 16) / BG);
        const GroupCode a = unpack_code(there ? sz[g0] : 0u), b = BG >= 32 ? a : unpack_code(there ? sz[g1] : 0u);
        const float v[4] = {value_of(word & 15u, a), value_of(word >> 4 & 15u, a), value_of(word >> 8 & 15u, b), value_of(word >> 12 & 15u, b)};
#pragma unroll
        for (int g = 0; g < HEADS; ++g) {
          const float p = ps[warp][tok][g];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][e][g] = fmaf(p, v[e], acc[i][e][g]);
        }
      }
    }
    __syncwarp();
  }
  // the warps' sums on the block's maximum, in their order
#pragma unroll
  for (int g = 0; g < HEADS; ++g) {
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], x);
    if (lane == 0) {
      tops[warp][g] = top[g];
      sums[warp][g] = sum[g];
    }
    if constexpr (SHARE > 1) {
#pragma unroll
      for (int x = 16; x >= 8 * UNITS; x >>= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[0][e][g] += __shfl_xor_sync(0xffffffffu, acc[0][e][g], x);
    }
  }
  __syncthreads();
  float total[HEADS];
#pragma unroll
  for (int g = 0; g < HEADS; ++g) {
    float m = LOWEST, l = 0.f;
#pragma unroll
    for (int x = 0; x < F32_WARPS; ++x) m = fmaxf(m, tops[x][g]);
#pragma unroll
    for (int x = 0; x < F32_WARPS; ++x) l = fmaf(sums[x][g], tops[x][g] == m ? 1.f : expf(tops[x][g] - m), l);
    const float by = top[g] == m ? 1.f : expf(top[g] - m);
#pragma unroll
    for (int i = 0; i < QUADS; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e][g] *= by;
    top[g] = m;
    total[g] = l;
  }
#pragma unroll 1
  for (int x = 0; x < F32_WARPS; ++x) {
    if (warp == x)
#pragma unroll
      for (int i = 0; i < QUADS; ++i) {
        const int at = SHARE > 1 ? lane % (8 * UNITS) : lane + 32 * i, r = at & 7, u = at >> 3;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int dim = 16 * (2 * u + (e >> 1)) + 2 * r + (e & 1);
          if (dim >= D || part > 0) continue;
#pragma unroll
          for (int g = 0; g < HEADS; ++g) qs[g][dim] = x == 0 ? acc[i][e][g] : qs[g][dim] + acc[i][e][g];
        }
      }
    __syncthreads();
  }
#pragma unroll
  for (int g = 0; g < HEADS; ++g) {
    if (g >= heads) break;
    for (int x = tid; x < D; x += F32_WARPS * 32) {
      if (splits == 1)
        out[(head0 + g) * D + x] = qs[g][x] / total[g];
      else
        part_o[((head0 + g) * splits + w.split) * D + x] = qs[g][x];
    }
    if (splits > 1 && tid == 0) {
      part_ml[((head0 + g) * splits + w.split) * 2] = top[g] * 1.4426950408889634f;   // in powers of two, as the join takes them
      part_ml[((head0 + g) * splits + w.split) * 2 + 1] = total[g];
    }
  }
}

// A warp per (row, query head): the splits' sums joined in their order.  Maxima are powers of two; a split without keys has sums of zero.
template <typename T>
__global__ void __launch_bounds__(THREADS) attn4_join_kernel(const float* part_o, const float* part_ml, const int* __restrict__ tok_slot, T* out, int n_heads, int total,
                                                             int splits) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int h = blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (h >= total || tok_slot[h / n_heads] < 0) return;   // (padding: the first launch wrote its zeros)
  constexpr int MINE = (D + 31) / 32;
  float m = -INFINITY, l = 0.f, a[MINE];
#pragma unroll
  for (int i = 0; i < MINE; ++i) a[i] = 0.f;
  const float2* const ml = reinterpret_cast<const float2*>(part_ml) + (size_t)h * splits;
  for (int s0 = 0; s0 < splits; s0 += 32) m = fmaxf(m, s0 + lane < splits ? __ldcg(ml + s0 + lane).x : -INFINITY);
  m = warp_max(m);
  const float* const o = part_o + (size_t)h * splits * D;
  for (int s0 = 0; s0 < splits; s0 += 32) {
    const float2 v = s0 + lane < splits ? __ldcg(ml + s0 + lane) : make_float2(-INFINITY, 0.f);
    const float mine = v.x == -INFINITY ? 0.f : exp2f(v.x - m);
#pragma unroll 4
    for (int s = 0; s < min(32, splits - s0); ++s) {
      const float by = __shfl_sync(0xffffffffu, mine, s), sum = __shfl_sync(0xffffffffu, v.y, s);
      if (sum == 0.f) continue;   // no keys: its partial sums may not have been written
      l = fmaf(sum, by, l);       // (the sum of a split whose scores are all NaN is NaN, whatever it is multiplied with)
#pragma unroll
      for (int i = 0; i < MINE; ++i)
        if (D % 32 == 0 || lane + 32 * i < D) a[i] = fmaf(__ldcg(o + (size_t)(s0 + s) * D + lane + 32 * i), by, a[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < MINE; ++i)
    if (D % 32 == 0 || lane + 32 * i < D) out[(size_t)h * D + lane + 32 * i] = from_f32<T>(a[i] / l);
}

struct Args {
  const void *q, *k_pages, *v_pages;
  const int* page_table;
  int max_pages;
  const int *tok_slot, *tok_pos;
  void* out;
  float *part_o, *part_ml;
  int n, n_kv, splits, least;
  float scale;
  int window, pdl;
  cudaStream_t st;
};

template <typename... P, typename... A>
int launch(void (*kern)(P...), dim3 grid, int threads, size_t bytes, int cluster, bool dependent, cudaStream_t st, A... a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int count = 0;
  if (cluster > 1) {
    attr[count].id = cudaLaunchAttributeClusterDimension;
    attr[count].val.clusterDim.x = cluster;
    attr[count].val.clusterDim.y = attr[count].val.clusterDim.z = 1;
    ++count;
  }
  if (dependent) {
    attr[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[count].val.programmaticStreamSerializationAllowed = 1;
    ++count;
  }
  cfg.attrs = attr;
  cfg.numAttrs = count;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, (P)a...);
  return e != cudaSuccess ? (int)e : launch_status();
}

dim3 grid_of(const Args& a) { return dim3(a.splits, a.n_kv * HEAD_TILES, a.n); }

template <typename T> int join(const Args& a) {
  const int total = a.n * a.n_kv * G;
  return launch(attn4_join_kernel<T>, dim3((total + THREADS / 32 - 1) / (THREADS / 32)), THREADS, 0, 1, a.pdl & 2, a.st, a.part_o, a.part_ml, a.tok_slot, (T*)a.out, a.n_kv * G,
                total, a.splits);
}

int rows_f32(const Args& a) {
  const int rc = launch(attn4_f32_kernel, grid_of(a), F32_WARPS * 32, 0, 1, false, a.st, (const float*)a.q, (const unsigned char*)a.k_pages, (const unsigned char*)a.v_pages,
                        a.page_table, a.max_pages, a.tok_slot, a.tok_pos, (float*)a.out, a.part_o, a.part_ml, a.scale, a.window);
  return rc || a.splits == 1 ? rc : join<float>(a);
}

template <int WARPS> int rows_bf16(const Args& a) {
  static bool asked[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return DRYFT_ERR_UNSUPPORTED;
  if (!asked[dev]) {   // (asking twice does no harm)
    cudaError_t e = cudaFuncSetAttribute(attn4_mma_kernel<WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Block<WARPS>::SMEM);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(attn4_mma_kernel<WARPS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return (int)e;
    asked[dev] = true;
  }
  const int cluster = a.splits > 1 && a.part_o == nullptr;
  if (cluster && a.splits > MOST_SPLITS) return DRYFT_ERR_UNSUPPORTED;
  const int rc = launch(attn4_mma_kernel<WARPS>, grid_of(a), WARPS * 32, Block<WARPS>::SMEM, cluster ? a.splits : 1, a.pdl & 1, a.st, (const bf16*)a.q,
                        (const unsigned char*)a.k_pages, (const unsigned char*)a.v_pages, a.page_table, a.max_pages, a.tok_slot, a.tok_pos, (bf16*)a.out, a.part_o,
                        a.part_ml, cluster, a.least, a.scale, a.window);
  return rc || a.splits == 1 || cluster ? rc : join<bf16>(a);
}
}  // namespace

// pdl: 1, the first launch is a programmatic dependent of the one before it (not in 32 bits); 2, the joining launch is one of the first; both or neither.
DRYFT_API int dryft_attn4_rows(int is_bf16, const void* q, const void* k_pages, const void* v_pages, const int* page_table, int max_pages, const int* tok_slot,
                               const int* tok_pos, void* out, float* part_o, float* part_ml, int n, int n_kv, int splits, int least, int warps, float scale, int window,
                               int pdl, void* stream) {
  if (n <= 0) return 0;
  if (n > 65535 || n_kv * HEAD_TILES > 65535) return DRYFT_ERR_UNSUPPORTED;
  return (!is_bf16 ? rows_f32 : warps == 4 ? rows_bf16<4> : rows_bf16<8>)({q, k_pages, v_pages, page_table, max_pages, tok_slot, tok_pos, out, part_o, part_ml, n, n_kv, splits, least, scale, window, pdl,
                                           (cudaStream_t)stream});
}
DRYFT_API int dryft_attn4_sizes(int which) { return which == 0 ? D : which == 1 ? G : which == 2 ? PAGE : BG; }
