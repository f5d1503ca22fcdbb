// Products with weights held in 4 bits (four_bit.cuh): y[m, n] = sum_k w[n, k] x[m, k].
//
// The weights' layout.  16 rows of W by 64 inputs are 32 lanes x 16 bytes: lane (r, c) holds word s = 0..3 for the inputs 16 s + 4c + e, nibble i of the low
// half being row r (i even) or r + 8 (i odd), e = 2 (i / 2), and of the high half the same with e + 1 -- the order in which the lane's registers of a
// 16 x 16 operand come out of the word (`code_pair`).  Blocks of 64 inputs of a tile of 16 rows follow one another, then the next tile; the last block and the last tile
// are filled up with codes that nothing reads as numbers.  Beside them [tile][group][r][row r, row r + 8] of (s, z).
#include "four_bit.cuh"

namespace {
constexpr int WARPS = 4, ROWS = 8;

// A block per 16 rows of W and ROWS rows of x, the inputs dealt out to the warps in blocks of 64.
template <typename T, typename O>
__global__ void __launch_bounds__(WARPS * 32) linear4_rows_kernel(const T* x, long long x_stride, const uint4* __restrict__ codes, const uint2* __restrict__ scales,
                                                                  O* y, int m, int n, int k, int group) {
  __shared__ float part[WARPS][2][ROWS][8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
  const int tile = blockIdx.x, m0 = blockIdx.y * ROWS, rows = min(ROWS, m - m0), blocks = (k + 63) / 64, groups = k / group;
  float acc[2][ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) acc[0][i] = acc[1][i] = 0.f;
  for (int b = warp; b < blocks; b += WARPS) {
    const uint4 raw = codes[((size_t)tile * blocks + b) * 32 + lane];
    const unsigned words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int at = 64 * b + 16 * s;
      if (at >= k) break;
      const uint2 sz = scales[((size_t)tile * groups + at / group) * 8 + r];
      const GroupCode g[2] = {unpack_code(sz.x), unpack_code(sz.y)};
      float w[2][4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int h = 0; h < 2; ++h) w[h][e] = value_of(words[s] >> (4 * (2 * (e >> 1) + h) + 16 * (e & 1)) & 15u, g[h]);
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        if (i >= rows) break;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float xv = to_f32<T>(x[(m0 + i) * x_stride + at + 4 * c + e]);
          acc[0][i] = fmaf(w[0][e], xv, acc[0][i]);
          acc[1][i] = fmaf(w[1][e], xv, acc[1][i]);
        }
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
    if (tile * 16 + row < n) y[(size_t)(m0 + mm) * n + tile * 16 + row] = from_f32<O>(v);
  }
}

// A warp per block of 64 inputs of a tile: what its codes stand for, in T.
template <typename T>
__global__ void __launch_bounds__(256) weight4_expand_kernel(const uint4* __restrict__ codes, const uint2* __restrict__ scales, T* w, int n, int k, int group) {
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3, blocks = (k + 63) / 64, groups = k / group;
  const long long at = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), total = (long long)((n + 15) / 16) * blocks;
  if (at >= total) return;
  const long long tile = at / blocks;
  const int b = (int)(at % blocks);
  const uint4 raw = codes[at * 32 + lane];
  const unsigned words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int col = 64 * b + 16 * s;
    if (col >= k) break;
    const uint2 sz = scales[(tile * groups + col / group) * 8 + r];
    const GroupCode g[2] = {unpack_code(sz.x), unpack_code(sz.y)};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long long row = tile * 16 + r + 8 * h;
      if (row >= n) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[row * k + col + 4 * c + e] = from_f32<T>(value_of(words[s] >> (4 * (2 * (e >> 1) + h) + 16 * (e & 1)) & 15u, g[h]));
    }
  }
}

template <typename T, typename O>
int rows(const void* x, long long x_stride, const void* codes, const void* scales, void* y, int m, int n, int k, int group, cudaStream_t st) {
  linear4_rows_kernel<T, O><<<dim3((n + 15) / 16, (m + ROWS - 1) / ROWS), WARPS * 32, 0, st>>>((const T*)x, x_stride, (const uint4*)codes, (const uint2*)scales,
                                                                                             (O*)y, m, n, k, group);
  return launch_status();
}
}  // namespace

DRYFT_API int dryft_linear4(int is_bf16, int out_bf16, const void* x, long long x_stride, const void* codes, const void* scales, void* y, int m, int n, int k,
                            int group, void* stream) {
  if (m <= 0 || n <= 0) return 0;
  typedef __nv_bfloat16 bf16;
  auto f = is_bf16 ? (out_bf16 ? rows<bf16, bf16> : rows<bf16, float>) : rows<float, float>;
  return f(x, x_stride, codes, scales, y, m, n, k, group, (cudaStream_t)stream);
}

DRYFT_API int dryft_weight4_expand(int is_bf16, const void* codes, const void* scales, void* w, int n, int k, int group, void* stream) {
  if (n <= 0) return 0;
  const long long total = (long long)((n + 15) / 16) * ((k + 63) / 64);
  const unsigned grid = (unsigned)((total + 7) / 8);
  if (is_bf16)
    weight4_expand_kernel<__nv_bfloat16><<<grid, 256, 0, (cudaStream_t)stream>>>((const uint4*)codes, (const uint2*)scales, (__nv_bfloat16*)w, n, k, group);
  else
    weight4_expand_kernel<float><<<grid, 256, 0, (cudaStream_t)stream>>>((const uint4*)codes, (const uint2*)scales, (float*)w, n, k, group);
  return launch_status();
}
