// Products with weights held in 4 bits (four_bit.cuh): y[m, n] = sum_k w[n, k] x[m, k].
//
// The weights' layout.  16 rows of W by 64 inputs are 32 lanes x 16 bytes: lane (r, c) holds word s = 0..3 for the inputs 16 s + 4c + e, nibble i of the low
// half being row r (i even) or r + 8 (i odd), e = 2 (i / 2), and of the high half the same with e + 1 -- the order in which the lane's registers of a
// 16 x 16 operand come out of the word (`code_pair`).  Blocks of 64 inputs of a tile of 16 rows follow one another, an even number of them, then the next tile.  Beside
// them [tile][group][r][row r, row r + 8] of (s, z).  Behind the last input and the last row s and z are zeros.
#include "four_bit.cuh"

namespace {
constexpr int WARPS = 8;
__host__ __device__ constexpr int blocks_of(int k) { return (k + 127) / 128 * 2; }                              // of 64 inputs, as laid out
__host__ __device__ constexpr int groups_of(int k, int group) { return (k + 127) / 128 * 128 / group; }

// 32-bit: a block per 16 rows of W and ROWS rows of x, the inputs dealt out to the warps in blocks of 64.  A lane has four inputs of rows r and r + 8 of W at a time: four
// numbers of each row of x (the eight lanes of a quarter read the same ones), 8 ROWS multiply-adds.  The sums of a row do not depend on how many there are.
// Bound by those multiply-adds and x's loads, not by the weights: 5 rows, 389 outputs of 80 inputs 3.3 us, a launch; 8 rows, 6,144 of 2,560 24 us, 10 TFLOP/s; 64 rows,
// 19,456 of 2,560 487 us, 13 TFLOP/s.
template <int ROWS>
__global__ void __launch_bounds__(WARPS * 32, 2) linear4_f32_kernel(const float* x, long long x_stride, const uint4* __restrict__ codes,
                                                                 const uint2* __restrict__ scales, float* y, int m, int n, int k, int group_bits) {
  __shared__ float part[WARPS][2][ROWS][8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
  const int tile = blockIdx.x, m0 = blockIdx.y * ROWS, rows = min(ROWS, m - m0), blocks = blocks_of(k), groups = groups_of(k, 1 << group_bits);
  const float* const x0 = x + m0 * x_stride + 4 * c;
  float acc[2][ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) acc[0][i] = acc[1][i] = 0.f;
  for (int b = warp; b * 64 < k; b += WARPS) {
    const uint4 raw = codes[((size_t)tile * blocks + b) * 32 + lane];
    const unsigned words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int at = 64 * b + 16 * s;
      if (at >= k) break;
      float4 xv[ROWS];
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
        if (i < rows) xv[i] = *reinterpret_cast<const float4*>(x0 + i * x_stride + at);
      const uint2 sz = scales[((size_t)tile * groups + (at >> group_bits)) * 8 + r];
      const GroupCode g[2] = {unpack_code(sz.x), unpack_code(sz.y)};
      float w[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const unsigned pair = code_pair(words[s], e + h);
          w[h][e] = fmaf(__uint_as_float(pair << 16) - CODE_BIAS, g[h].s, g[h].z);
          w[h][e + 1] = fmaf(__uint_as_float(pair & 0xffff0000u) - CODE_BIAS, g[h].s, g[h].z);
        }
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
        if (i < rows)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            acc[h][i] = fmaf(w[h][0], xv[i].x, acc[h][i]);
            acc[h][i] = fmaf(w[h][1], xv[i].y, acc[h][i]);
            acc[h][i] = fmaf(w[h][2], xv[i].z, acc[h][i]);
            acc[h][i] = fmaf(w[h][3], xv[i].w, acc[h][i]);
          }
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v = acc[h][i];
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      if (c == 0) part[warp][h][i][r] = v;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * rows; i += WARPS * 32) {
    const int row = i & 15, mm = i >> 4;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) v += part[w][row >> 3][mm][row & 7];
    if (tile * 16 + row < n) y[(size_t)(m0 + mm) * n + tile * 16 + row] = v;
  }
}

// A warp per block of 64 inputs of a tile: what its codes stand for.  PART 0: in float32, 1: rounded to bfloat16, 2: what that rounding left, rounded to bfloat16.
// A lane writes four numbers of a row at a time; four neighbours fill a sector.  Bound by what it writes: 24,576 x 4,096 in bfloat16 47 us, 5,470 GB/s.
template <int PART>
__global__ void __launch_bounds__(256) weight4_expand_kernel(const uint4* __restrict__ codes, const uint2* __restrict__ scales, void* w, int n, int k, int group_bits) {
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3, blocks = blocks_of(k), groups = groups_of(k, 1 << group_bits);
  const long long at = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), total = (long long)((n + 15) / 16) * blocks;
  if (at >= total) return;
  const long long tile = at / blocks;
  const int b = (int)(at % blocks);
  const uint4 raw = __ldcs(codes + at * 32 + lane);
  const unsigned words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int col = 64 * b + 16 * s;
    if (col >= k) break;
    const uint2 sz = scales[(tile * groups + (col >> group_bits)) * 8 + r];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long long row = tile * 16 + r + 8 * h;
      if (row >= n) continue;
      const GroupCode g = unpack_code(h ? sz.y : sz.x);
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = value_of(words[s] >> (4 * (2 * (e >> 1) + h) + 16 * (e & 1)) & 15u, g);
      if (PART == 0) {
        *reinterpret_cast<float4*>((float*)w + row * k + col + 4 * c) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
        if (PART == 2)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] -= rnd<__nv_bfloat16>(v[e]);   // exact
        const __nv_bfloat162 x = __floats2bfloat162_rn(v[0], v[1]), y = __floats2bfloat162_rn(v[2], v[3]);
        *reinterpret_cast<uint2*>((__nv_bfloat16*)w + row * k + col + 4 * c) = make_uint2(*reinterpret_cast<const unsigned*>(&x), *reinterpret_cast<const unsigned*>(&y));
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------- bfloat16: tensor cores
// y^T = W x^T on mma.sync.m16n8k16: 16 rows of W are the 16-row operand, straight from the codes (16 + c, `code_pair`), eight rows of x the columns.  A group's
// products are summed over 16 + c from zero (a constant that no instruction has to put there), then  y += s acc + (z - 23.5 s) sum_k x  in 32 bits, so nothing is rounded below
// 32 bits before the result.  The warps of a block share a tile's inputs: each walks its own blocks of 64, their sums meet in shared memory.
typedef __nv_bfloat16 bf16;

__device__ __forceinline__ float2 two_of(unsigned w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }

__device__ __forceinline__ void copy16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from));
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N)); }
__device__ __forceinline__ unsigned word_of(uint4 v, int s) { return s == 0 ? v.x : s == 1 ? v.y : s == 2 ? v.z : v.w; }

// Few rows of x (up to 16), all of whose numbers fit in shared memory.  Bound by issue: a slot of 128 inputs is 200 instructions of a warp, half of them on the
// pipe for logic (which takes one every other cycle, 64% busy); the 64 that take the codes apart are a third of all.  One row, 151,936 outputs of 2,560 inputs: 56 us,
// 3,900 GB/s, 60% of a copy's rate; 6,144 outputs 4.7 us, 19,456 9.9 us, of which some 3 us are the launch and the first bytes' way.  A block of 16 warps is 16 / TEAM teams; a team takes
// a tile of 16 rows of W at a time, its warps the tile's inputs in turn shares.  Each warp copies its own share of the codes into its own ring, SLOTS - 1 slots of
// PB blocks of 64 inputs ahead, across the ends of tiles, so that the requests never drain; a lane reads what it copied itself, and nothing waits for another warp
// but a tile's end.
constexpr int FEW_WARPS = 16;

template <int NT, int GS, int TEAM, int PB, int SLOTS> struct Few {
  static constexpr int SCALES = GS == 8 ? 1 : PB * 4 / GS;    // groups that begin in a slot
  static constexpr int SLOT = PB * 512 + SCALES * 256;
  static constexpr int REDS = TEAM == FEW_WARPS ? 1 : 2;       // buffers for a tile's sums
  static constexpr size_t RED_BYTES = (size_t)REDS * FEW_WARPS * NT * 512, RING_BYTES = (size_t)FEW_WARPS * SLOTS * SLOT;
  __host__ __device__ static int slots_of(int k) { return blocks_of(k) / PB; }   // of a tile
  // rows of x lie 32 bytes further apart than a multiple of 128, which keeps a warp's reads of eight rows apart
  __host__ __device__ static int row_bytes(int k) { return blocks_of(k) * 128 + 32; }
  static size_t bytes(int m, int k) { return RED_BYTES + RING_BYTES + (size_t)slots_of(k) * SCALES * NT * 32 + (size_t)m * row_bytes(k); }
};

// What stands around the product in a decoder's layer is done on its way (rounding points as in gemm_decode.cu):
//   norm_w: x is RMS-normed first, every block for itself: T(T(x rsqrt(mean x^2 + eps)) w);
//   RESIDUAL: y += the result, in place;  SILU: W holds N / 2 gate rows, then as many rows to multiply with; a team takes a tile of either in turn, y = T(silu(gate)) up.
enum Mode { STORE_BF16 = 0, STORE_F32 = 1, RESIDUAL = 2, SILU = 3 };
__device__ __forceinline__ float bfr(float v) { return rnd<bf16>(v); }

// A result that is not finite, worked out again from the definition (x: a row in shared memory)
__device__ __noinline__ float defined_result(const uint4* codes, const uint2* scales, int row, int k, int group_bits, const unsigned char* x) {
  return defined_product(codes, scales, row, k, group_bits, [x](int i) { return __bfloat162float(reinterpret_cast<const bf16*>(x)[i]); });
}

// ALONE: no norm, and the result is stored (one row, 151,936 outputs of 2,560 inputs: 56.2 us so, 57.9 where the kernel asks what to do)
template <int NT, int GS, int TEAM, int PB, int SLOTS, bool ALONE>
__global__ void __launch_bounds__(FEW_WARPS * 32, 1) linear4_few_kernel(const bf16* x, long long x_stride, const uint4* __restrict__ codes,
                                                                        const uint2* __restrict__ scales, void* y, int m, int n, int k, int group_bits, int how,
                                                                        const float* __restrict__ norm_w, float eps) {
  const int mode = ALONE && how != STORE_F32 ? STORE_BF16 : how;
  const bool fused_silu = !ALONE && mode == SILU;
  typedef Few<NT, GS, TEAM, PB, SLOTS> F;
  constexpr int SCALES = F::SCALES, SLOT = F::SLOT, TEAMS = FEW_WARPS / TEAM, STEPS = PB * 4 / SCALES;
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3, team = warp / TEAM;
  const int tiles = (n + 15) / 16, slots = F::slots_of(k), row_bytes = F::row_bytes(k);
  float* const red = reinterpret_cast<float*>(smem);
  float2* const xs = reinterpret_cast<float2*>(smem + F::RED_BYTES);   // [slot][SCALES][NT][c]: sums of columns 2c, 2c + 1 over the group
  unsigned char* const rings = reinterpret_cast<unsigned char*>(xs + slots * SCALES * NT * 4);
  unsigned char* const rows = rings + F::RING_BYTES;
  const int per = (slots + TEAM - 1) / TEAM, s0 = min(slots, warp % TEAM * per), ns = min(slots, s0 + per) - s0;
  // the team's tiles: block and team together count through them, the block's number first
  const int half = fused_silu ? tiles / 2 : 0, turns = fused_silu ? half : tiles;   // a turn: a tile, or a gate tile and the one `half` tiles behind it
  const int first = blockIdx.x + team * gridDim.x, step = gridDim.x * TEAMS, mine = (first < turns ? (turns - 1 - first) / step + 1 : 0) * (fused_silu ? 2 : 1);
  const int total = mine * ns;   // the warp's slots

  // Slot i of the warp goes into place i mod SLOTS of its ring.  Codes and scales lie slot behind slot, tile behind tile.  (A group of 128 has two slots of one
  // block: the scale is then the same for both.)
  int sent = 0, until = ns;
  unsigned at = first * slots + s0;
  unsigned jump = fused_silu ? half * slots - ns : step * slots - ns;   // from a tile's last slot to the next tile's first one
  const unsigned jumps = step * slots - 2 * ns;                           // SILU: of the two jumps of a turn
  const unsigned ring = (unsigned)__cvta_generic_to_shared(rings + warp * F::RING_BYTES / FEW_WARPS) + lane * 16;
  const unsigned ring_scales = ring - lane * 8 + PB * 512;
  const uint4* const my_codes = codes + lane;
  const uint2* const my_scales = scales + r;
  const int half_scale = GS < 8 && PB == 1 && group_bits == 7;
  auto request = [&](int place) {
    if (sent < total) {
      const uint4* const from = my_codes + (size_t)at * (PB * 32);
      const uint2* const from_scale = my_scales + (size_t)(PB == 1 && GS == 4 ? at >> half_scale : at) * (SCALES * 8);
#pragma unroll
      for (int i = 0; i < PB; ++i) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ring + place * SLOT + i * 512), "l"(from + i * 32));
#pragma unroll
      for (int g = 0; g < SCALES; ++g)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(ring_scales + place * SLOT + g * 256), "l"(from_scale + g * 8));
      ++at;
      if (--until == 0) {
        until = ns;
        at += jump;
        if (fused_silu) jump = jumps - jump;
      }
    }
    ++sent;
    copies_end();
  };
  let_next_launch_in();
#pragma unroll
  for (int i = 0; i < SLOTS - 1; ++i) request(i);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int pieces = blocks_of(k) * 8;   // of 16 bytes in a row of x
  for (int row = 0; row < m; ++row)
    for (int i = threadIdx.x; i < pieces; i += FEW_WARPS * 32) {
      unsigned char* const to = rows + (size_t)row * row_bytes + i * 16;
      if (8 * i < k)
        copy16(to, x + row * x_stride + 8 * i);
      else
        *reinterpret_cast<uint4*>(to) = make_uint4(0, 0, 0, 0);
    }
  copies_end();
  copies_wait<0>();
  __syncthreads();
  if (!ALONE && norm_w != nullptr) {   // the warps share the rows, or a row
    const int wr = m == 1 ? 16 : m == 2 ? 8 : m <= 4 ? 4 : m <= 8 ? 2 : 1, row = warp / wr, part = warp % wr;
    unsigned char* const at_x = rows + (size_t)row * row_bytes;
    float ss = 0.f;
    if (row < m)
      for (int i = part * 32 + lane; 8 * i < k; i += wr * 32) {
        const uint4 v = *reinterpret_cast<const uint4*>(at_x + i * 16);
        const unsigned e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 p = two_of(e[j]);
          ss = fmaf(p.x, p.x, fmaf(p.y, p.y, ss));
        }
      }
    ss = warp_sum(ss);
    if (lane == 0) red[warp] = ss;
    __syncthreads();
    if (row < m) {
      ss = 0.f;
      for (int i = 0; i < wr; ++i) ss += red[row * wr + i];
      const float inv = rsqrtf(ss / (float)k + eps);
      for (int i = part * 32 + lane; 8 * i < k; i += wr * 32) {
        uint4* const cell = reinterpret_cast<uint4*>(at_x + i * 16);
        const uint4 v = *cell;
        unsigned e[4] = {v.x, v.y, v.z, v.w};
        const float4 w0 = reinterpret_cast<const float4*>(norm_w)[2 * i], w1 = reinterpret_cast<const float4*>(norm_w)[2 * i + 1];
        const float w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 p = two_of(e[j]);
          const __nv_bfloat162 q = __floats2bfloat162_rn(bfr(p.x * inv) * w[2 * j], bfr(p.y * inv) * w[2 * j + 1]);
          e[j] = *reinterpret_cast<const unsigned*>(&q);
        }
        *cell = make_uint4(e[0], e[1], e[2], e[3]);
      }
    }
    __syncthreads();
  }
  const unsigned char* at_row[NT];   // the lane's share of the first step of its column; columns behind the last one repeat it
#pragma unroll
  for (int j = 0; j < NT; ++j) at_row[j] = rows + (size_t)min(8 * j + r, m - 1) * row_bytes + 8 * c;
  for (int i = warp; i < slots * SCALES; i += FEW_WARPS)
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float sum = 0.f;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const uint2 v = *reinterpret_cast<const uint2*>(at_row[j] + (i * STEPS + s) * 32);
        const float2 p = two_of(v.x), q = two_of(v.y);
        sum += (p.x + p.y) + (q.x + q.y);
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      const float a = __shfl_sync(0xffffffffu, sum, 8 * c), b = __shfl_sync(0xffffffffu, sum, 8 * c + 4);
      if (r == 0) xs[(i * NT + j) * 4 + c] = make_float2(a, b);
    }
  __syncthreads();

  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
  int tile = 0;
  float none = 0.f;   // of infinities and NaN among the thread's results
  constexpr int OUTS = (NT * 128 + TEAM * 32 - 1) / (TEAM * 32);   // results of a thread
  float gate[OUTS];
  // A team's sums of a tile, in the warps' order; with two buffers the last tile's are read while this one's are written.
  const int out_row = threadIdx.x & 15, out_col = threadIdx.x % (TEAM * 32) >> 4;   // lane (row & 7) * 4 + (col & 7) / 2, element 2 (row >= 8) + (col & 1)
  const float* const out_from = red + team * TEAM * NT * 128 + (out_row & 7) * 16 + ((out_col & 7) >> 1) * 4 + 2 * (out_row >> 3) + (out_col & 1);
  auto tile_done = [&] {
    const int buffer = F::REDS == 2 ? (tile & 1) * FEW_WARPS * NT * 128 : 0;
    if (F::REDS == 1 && tile > 0) __syncthreads();
    float* const to = red + buffer + warp * NT * 128 + lane * 4;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      *reinterpret_cast<float4*>(to + j * 128) = make_float4(acc[j][0], acc[j][1], acc[j][2], acc[j][3]);
      acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    }
    asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(TEAM * 32) : "memory");
    const int turn = fused_silu ? tile >> 1 : tile, row = (first + turn * step) * 16 + out_row;
#pragma unroll
    for (int i = 0; i < OUTS; ++i) {
      const int col = out_col + i * (TEAM * 2);
      if (col >= NT * 8) continue;
      const float* const place = out_from + buffer + (col >> 3) * 128;
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < TEAM; ++w) v += place[w * NT * 128];
      if (row >= n || col >= m) continue;
      if (ALONE)
        none = fmaf(v, 0.f, none);
      else if (!(fabsf(v) < INFINITY))
        v = defined_result(codes, scales, row + (tile & 1) * half * 16, k, group_bits, rows + (size_t)col * row_bytes);
      bf16* const to = reinterpret_cast<bf16*>(y) + (size_t)col * n + row;
      if (mode == STORE_BF16) {
        *to = __float2bfloat16_rn(v);
      } else if (ALONE || mode == STORE_F32) {
        reinterpret_cast<float*>(y)[(size_t)col * n + row] = v;
      } else if (mode == RESIDUAL) {
        *to = __float2bfloat16_rn(ld_prev_bf16(to) + bfr(v));
      } else if ((tile & 1) == 0) {
        gate[i] = bfr(v);
      } else {
        reinterpret_cast<bf16*>(y)[(size_t)col * (n / 2) + row] = __float2bfloat16_rn(bfr(gate[i] / (1.f + expf(-gate[i]))) * bfr(v));
      }
    }
    ++tile;
  };
  if (ns == 0)
    for (int t = 0; t < mine; ++t) tile_done();
  const unsigned char* const my_ring = rings + warp * F::RING_BYTES / FEW_WARPS;
  int here = s0;
  for (int i = 0; i < total; i += SLOTS) {
#pragma unroll
    for (int u = 0; u < SLOTS; ++u) {
      if (i + u >= total) break;
      request((u + SLOTS - 1) % SLOTS);   // into the place that was read last
      copies_wait<SLOTS - 1>();
      const unsigned char* const from = my_ring + u * SLOT;
      uint4 w[PB];
#pragma unroll
      for (int b = 0; b < PB; ++b) w[b] = *reinterpret_cast<const uint4*>(from + b * 512 + lane * 16);
      const float2* const my_xs = xs + here * (SCALES * NT * 4) + c;
#pragma unroll
      for (int g = 0; g < SCALES; ++g) {
        const uint2 sz = *reinterpret_cast<const uint2*>(from + PB * 512 + g * 256 + lane * 8);
        const GroupCode lo = unpack_code(sz.x), hi = unpack_code(sz.y);
        float2 sum[NT];
        float part[NT][4];
        const float lo_z = fmaf(-CODE_BIAS, lo.s, lo.z), hi_z = fmaf(-CODE_BIAS, hi.s, hi.z);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          sum[j] = my_xs[(g * NT + j) * 4];
          part[j][0] = part[j][1] = part[j][2] = part[j][3] = 0.f;
        }
#pragma unroll
        for (int q = g * STEPS; q < (g + 1) * STEPS; ++q) {
          const unsigned v = word_of(w[q / 4], q % 4), a0 = code_pair(v, 0), a1 = code_pair(v, 1), a2 = code_pair(v, 2), a3 = code_pair(v, 3);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const uint2 bx = *reinterpret_cast<const uint2*>(at_row[j] + here * (PB * 128) + q * 32);
            mma_16816(part[j], a0, a1, a2, a3, bx.x, bx.y);
          }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          acc[j][0] = fmaf(lo.s, part[j][0], fmaf(lo_z, sum[j].x, acc[j][0]));
          acc[j][1] = fmaf(lo.s, part[j][1], fmaf(lo_z, sum[j].y, acc[j][1]));
          acc[j][2] = fmaf(hi.s, part[j][2], fmaf(hi_z, sum[j].x, acc[j][2]));
          acc[j][3] = fmaf(hi.s, part[j][3], fmaf(hi_z, sum[j].y, acc[j][3]));
        }
      }
      if (++here == s0 + ns) {
        here = s0;
        tile_done();
      }
    }
  }
  copies_wait<0>();
  if (ALONE && !(none == 0.f))   // behind all tiles: the code that every tile runs stays short (one row, 6,144 outputs: 4.7 us, 4.9 with the call in it)
#pragma unroll 1
    for (int i = 0; i < mine * OUTS; ++i) {
      const int row = (first + i / OUTS * step) * 16 + out_row, col = out_col + i % OUTS * (TEAM * 2);
      if (col >= m || row >= n) continue;
      bf16* const to = reinterpret_cast<bf16*>(y) + (size_t)col * n + row;
      float* const wide = reinterpret_cast<float*>(y) + (size_t)col * n + row;
      if (fabsf(mode == STORE_F32 ? *wide : __bfloat162float(*to)) < INFINITY) continue;
      const float v = defined_result(codes, scales, row, k, group_bits, rows + (size_t)col * row_bytes);
      if (mode == STORE_F32)
        *wide = v;
      else
        *to = __float2bfloat16_rn(v);
    }
}

constexpr size_t SMEM_MOST = 227 * 1024;

template <typename... P, typename... A> int launch(void (*kern)(P...), bool (&asked)[64], int grid, int threads, size_t bytes, int pdl, cudaStream_t st, A... a) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return DRYFT_ERR_UNSUPPORTED;
  if (!asked[dev]) {   // (asking twice does no harm)
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_MOST);
    if (e != cudaSuccess) return (int)e;
    asked[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl & 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, (P)a...);
  return e != cudaSuccess ? (int)e : launch_status();
}

struct Args {
  const void* x;
  long long x_stride;
  const void *codes, *scales;
  void* y;
  int m, n, k, group, mode;
  const float* norm_w;
  float eps;
  int pdl;
  cudaStream_t st;
};

template <int NT, int GS, int TEAM, int PB, int SLOTS, bool ALONE> int few(const Args& a) {
  static bool asked[64] = {false};
  const int tiles = (a.n + 15) / 16, turns = a.mode == SILU ? tiles / 2 : tiles;
  return launch(linear4_few_kernel<NT, GS, TEAM, PB, SLOTS, ALONE>, asked, turns < 148 ? turns : 148, FEW_WARPS * 32, Few<NT, GS, TEAM, PB, SLOTS>::bytes(a.m, a.k), a.pdl, a.st,
                (const bf16*)a.x, a.x_stride, (const uint4*)a.codes, (const uint2*)a.scales, a.y, a.m, a.n, a.k, __builtin_ctz(a.group), a.mode, a.norm_w, a.eps);
}
// Four warps a tile where shared memory has room for their rings beside x (eight rows: up to about 7,000 inputs), else all sixteen with shorter rings, which only
// 32-bit results use.  2,560 inputs, one row, four / eight / sixteen warps a tile: 151,936 outputs 55.6 / 63.6 / 81.9 us, 6,144 outputs 4.8 / 5.4 / 5.7 us (a tile's
// end costs each warp as much as half a slot).  Where only the sixteen fit, the tensor memory kernel is as fast or faster (16 rows of 4,096 inputs, 24,576 outputs:
// 21.3 us and 29.1; 8 rows of 9,728 inputs, 2,560 outputs: 11.4 and 12.1), but not where it has two products to make for 32 bits.
constexpr int slots_of_group(int gs) { return gs == 1 ? 2 : gs == 2 ? 3 : 4; }   // as many as 98 KB hold: the scales of small groups are longer than the codes
template <int NT, int GS> bool four_fit(int m, int k) { return Few<NT, GS, 4, 2, slots_of_group(GS)>::bytes(m, k) <= SMEM_MOST; }
template <int NT, int GS> bool sixteen_fit(int m, int k) { return Few<NT, GS == 8 ? 4 : GS, 16, 1, 4>::bytes(m, k) <= SMEM_MOST; }
template <int NT> int fits(int m, int k, int group) {
  if (group == 128 ? four_fit<NT, 8>(m, k) : group == 64 ? four_fit<NT, 4>(m, k) : group == 32 ? four_fit<NT, 2>(m, k) : four_fit<NT, 1>(m, k)) return 1;
  return (group >= 64 ? sixteen_fit<NT, 4>(m, k) : group == 32 ? sixteen_fit<NT, 2>(m, k) : sixteen_fit<NT, 1>(m, k)) ? 2 : 0;
}
int takes(int m, int k, int group) { return m <= 8 ? fits<1>(m, k, group) : m <= 16 ? fits<2>(m, k, group) : 0; }

template <int NT, int GS, bool ALONE> int few_rows(const Args& a) {
  constexpr int GM = GS == 8 ? 4 : GS;
  if (four_fit<NT, GS>(a.m, a.k)) return few<NT, GS, 4, 2, slots_of_group(GS), ALONE>(a);
  if constexpr (ALONE) return few<NT, GM, 16, 1, 4, true>(a);
  return DRYFT_ERR_UNSUPPORTED;
}
template <int GS, bool ALONE> int by_mode(const Args& a) { return a.m <= 8 ? few_rows<1, GS, ALONE>(a) : few_rows<2, GS, ALONE>(a); }
template <int GS> int by_rows(const Args& a) { return a.mode <= STORE_F32 && a.norm_w == nullptr ? by_mode<GS, true>(a) : by_mode<GS, false>(a); }
}  // namespace

// Whether the kernel for few rows of bfloat16 takes so many rows of so many inputs (they have to fit in shared memory): 1, with four warps a tile and whatever stands
// around the product; 2, with sixteen, and the product alone; 0, not.
DRYFT_API int dryft_linear4_takes(int m, int k, int group) { return takes(m, k, group); }

// mode: Mode.  Modes beyond storing, and norm_w (which has k numbers on a 16-byte boundary; null: no norm), are the bfloat16 kernel's; SILU wants n to be a multiple of 32.
DRYFT_API int dryft_linear4(int is_bf16, int mode, const void* x, long long x_stride, const void* codes, const void* scales, void* y, int m, int n, int k, int group,
                            const float* norm_w, float eps, int pdl, void* stream) {
  if (m <= 0 || n <= 0) return 0;
  const cudaStream_t st = (cudaStream_t)stream;
  if (is_bf16) {
    if (!takes(m, k, group) || (mode == SILU && n % 32) || ((uintptr_t)norm_w & 15)) return DRYFT_ERR_UNSUPPORTED;
    const Args a = {x, x_stride, codes, scales, y, m, n, k, group, mode, norm_w, eps, pdl, st};
    return (group == 128 ? by_rows<8> : group == 64 ? by_rows<4> : group == 32 ? by_rows<2> : by_rows<1>)(a);
  }
  if (mode != STORE_F32 || norm_w) return DRYFT_ERR_UNSUPPORTED;
  const int rows = m == 1 ? 1 : m <= 4 ? 4 : m <= 8 ? 8 : 16;
  auto kern = rows == 1 ? linear4_f32_kernel<1> : rows == 4 ? linear4_f32_kernel<4> : rows == 8 ? linear4_f32_kernel<8> : linear4_f32_kernel<16>;
  kern<<<dim3((n + 15) / 16, (m + rows - 1) / rows), WARPS * 32, 0, st>>>((const float*)x, x_stride, (const uint4*)codes, (const uint2*)scales, (float*)y, m, n, k,
                                                                         __builtin_ctz(group));
  return launch_status();
}

// part 0: float32; 1: bfloat16; 2: the rest of that rounding in bfloat16
DRYFT_API int dryft_weight4_expand(int part, const void* codes, const void* scales, void* w, int n, int k, int group, void* stream) {
  if (n <= 0) return 0;
  const long long total = (long long)((n + 15) / 16) * blocks_of(k);
  auto kern = part == 0 ? weight4_expand_kernel<0> : part == 1 ? weight4_expand_kernel<1> : weight4_expand_kernel<2>;
  kern<<<(unsigned)((total + 7) / 8), 256, 0, (cudaStream_t)stream>>>((const uint4*)codes, (const uint2*)scales, w, n, k, __builtin_ctz(group));
  return launch_status();
}
