// Rounding rows to microscaled 4-bit floating point (fp4.cuh has the format and the layout) and taking them out again.
#include "fp4.cuh"

namespace {
using namespace fp4;
typedef __nv_bfloat16 bf16;
constexpr int UNIT = 16;        // numbers that a lane has at a time
constexpr int THREADS = 256, WARPS = THREADS / 32;

// 16 numbers from column c on; zeros behind column k.  Through L2 (`ld_prev`): the launch before this one may have written them.
__device__ __forceinline__ void load16(const bf16* row, int c, int k, bool words, float (&v)[UNIT]) {
  if (words && c + UNIT <= k) {
    const uint4* const p = reinterpret_cast<const uint4*>(row + c);
    const uint4 a = ld_prev(p), b = ld_prev(p + 1);
    const unsigned w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < UNIT; ++i) v[i] = c + i < k ? ld_prev_bf16(row + c + i) : 0.f;
}
__device__ __forceinline__ void load16(const float* row, int c, int k, bool words, float (&v)[UNIT]) {
  if (words && c + UNIT <= k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 a = ld_prev(reinterpret_cast<const float4*>(row + c) + i);
      v[4 * i] = a.x;
      v[4 * i + 1] = a.y;
      v[4 * i + 2] = a.z;
      v[4 * i + 3] = a.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < UNIT; ++i) v[i] = c + i < k ? ld_prev(row + c + i) : 0.f;
}

struct Size { unsigned most; bool bad; };   // the bits of the largest finite magnitude (magnitudes' bits are in their order); whether one is not finite
__device__ __forceinline__ Size size_of(const float (&v)[UNIT]) {
  Size s = {0u, false};
#pragma unroll
  for (int i = 0; i < UNIT; ++i) {
    const unsigned a = __float_as_uint(v[i]) & 0x7fffffffu;
    if (a < 0x7f800000u) s.most = max(s.most, a);
    else s.bad = true;
  }
  return s;
}
// codes of eight numbers, the first in the lowest four bits
__device__ __forceinline__ unsigned codes8(const float* v, float r) {
  unsigned w;
  asm("{ .reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3}; }"
      : "=r"(w)
      : "f"(v[0] * r), "f"(v[1] * r), "f"(v[2] * r), "f"(v[3] * r), "f"(v[4] * r), "f"(v[5] * r), "f"(v[6] * r), "f"(v[7] * r));
  return w;
}

// A row is 1, 2, 4 or 8 warps' (`span` lanes), 16 numbers a lane at a time.
template <typename T, int KIND> __global__ void __launch_bounds__(THREADS) fp4_quantise_kernel(const T* x, long long stride, unsigned char* held, float* factors, int rows,
                                                                                               int k, int span, bool words) {
  typedef Format<KIND> F;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  let_next_launch_in();   // (behind the wait: what comes in may rely on all that was written before this launch)
  __shared__ unsigned most_s[WARPS];
  const int at = threadIdx.x & (span - 1), row = blockIdx.x * (THREADS / span) + threadIdx.x / span, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int units = blocks_of(k) * (INPUTS / UNIT);
  const bool live = row < rows;
  const T* const from = x + (live ? row : 0) * stride;
  float factor = 0.f, u = 0.f;
  if (KIND == NV) {
    unsigned most = 0;
    if (live)
      for (int i = at; i * UNIT < k; i += span) {
        float v[UNIT];
        load16(from, i * UNIT, k, words, v);
        most = max(most, size_of(v).most);
      }
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) most_s[warp] = most;
    __syncthreads();
    const int first = warp & ~(span / 32 - 1);
    for (int w = 0; w < span / 32; ++w) most = max(most, most_s[first + w]);
    factor = fmaxf(__fdiv_rn(__uint_as_float(most), 2688.f), __uint_as_float((127u - 112u) << 23));
    u = __frcp_rn(6.f * factor);
    if (live && at == 0) factors[row] = factor;
  }
  unsigned char* const block_row = held + (size_t)((live ? row : 0) / ROWS) * blocks_of(k) * F::BLOCK_BYTES;
  const int r128 = row % ROWS;
  for (int i0 = 0; i0 < units; i0 += span) {   // (whole warps, for the exchanges)
    const int i = i0 + at;
    float v[UNIT];
    if (live && i < units) load16(from, i * UNIT, k, words, v);
    else
#pragma unroll
      for (int j = 0; j < UNIT; ++j) v[j] = 0.f;
    Size s = size_of(v);
    unsigned byte, word;
    float r;
    if (KIND == NV) {
      unsigned short two;
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(0.f), "f"(__uint_as_float(s.most) * u));
      byte = two & 0xff;
      r = byte == 0 ? 0.f : __frcp_rn(scale_value(byte, true) * factor);
      if (s.bad) byte = NV_NAN;
      word = byte | __shfl_down_sync(0xffffffffu, byte, 1) << 8;
      word |= __shfl_down_sync(0xffffffffu, word, 2) << 16;
    } else {
      s.most = max(s.most, __shfl_xor_sync(0xffffffffu, s.most, 1));
      s.bad |= __shfl_xor_sync(0xffffffffu, (int)s.bad, 1) != 0;
      byte = max((int)(s.most >> 23) - 2, 0);
      r = __uint_as_float((254u - byte) << 23);   // 1 / s: 2^127 at the most
      if (s.bad) byte = MX_NAN;
      word = byte | __shfl_down_sync(0xffffffffu, byte, 2) << 8;
      word |= __shfl_down_sync(0xffffffffu, word, 4) << 16;
    }
    uint2 c = make_uint2(codes8(v, r), codes8(v + 8, r));
    if (s.bad) c = make_uint2(0x22222222u, 0x22222222u);
    if (live && i < units) {
      unsigned char* const block = block_row + (size_t)(i / (INPUTS / UNIT)) * F::BLOCK_BYTES;
      const int unit = i % (INPUTS / UNIT);
      *reinterpret_cast<uint2*>(block + F::SCALE_BYTES + code_at(r128, unit)) = c;
      constexpr int PER_WORD = F::WORD_INPUTS / UNIT;
      if (unit % PER_WORD == 0) *reinterpret_cast<unsigned*>(block + scale_word_at(r128, unit / PER_WORD)) = word;
    }
  }
}

template <typename O, int KIND> __global__ void __launch_bounds__(THREADS) fp4_expand_kernel(const unsigned char* held, const float* factors, O* out, int k, unsigned units,
                                                                                             unsigned long long all, bool words) {
  typedef Format<KIND> F;
  const unsigned long long id = (unsigned long long)blockIdx.x * THREADS + threadIdx.x;
  if (id >= all) return;
  const unsigned long long row = id / units;
  const int i = (int)(id - row * units), unit = i % (INPUTS / UNIT), r128 = (int)(row % ROWS);
  const unsigned char* const block = held + (row / ROWS * blocks_of(k) + i / (INPUTS / UNIT)) * F::BLOCK_BYTES;
  const uint2 c = *reinterpret_cast<const uint2*>(block + F::SCALE_BYTES + code_at(r128, unit));
  const int group = unit * UNIT / F::GROUP;
  const float s = scale_value(block[scale_word_at(r128, group / 4) + group % 4], KIND == NV), g = KIND == NV ? factors[row] : 1.f;
  float v[UNIT];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    unsigned two;
    asm("{ .reg .b8 b; cvt.u8.u32 b, %1; cvt.rn.f16x2.e2m1x2 %0, b; }" : "=r"(two) : "r"((j < 4 ? c.x >> (8 * j) : c.y >> (8 * (j - 4))) & 0xffu));
    const __half2 h = *reinterpret_cast<const __half2*>(&two);
    v[2 * j] = __low2float(h) * s;
    v[2 * j + 1] = __high2float(h) * s;
    if (KIND == NV) {
      v[2 * j] *= g;
      v[2 * j + 1] *= g;
    }
  }
  O* const to = out + row * k + i * UNIT;
  if (words && i * UNIT + UNIT <= k) {
    constexpr int PER = 16 / sizeof(O);
#pragma unroll
    for (int j = 0; j < UNIT; j += PER) {
      O part[PER];
#pragma unroll
      for (int e = 0; e < PER; ++e) part[e] = from_f32<O>(v[j + e]);
      *reinterpret_cast<uint4*>(to + j) = *reinterpret_cast<const uint4*>(part);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < UNIT; ++j)
    if (i * UNIT + j < k) to[j] = from_f32<O>(v[j]);
}

template <typename... P, typename... A> int launch(void (*kern)(P...), dim3 grid, bool dependent, cudaStream_t st, A... a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, (P)a...);
  return e != cudaSuccess ? (int)e : launch_status();
}
}  // namespace

// held: blocks of 128 rows by 256 inputs (fp4.cuh); factors: float [rows] (NV).  x: rows of k numbers, `stride` numbers apart, anywhere.
DRYFT_API int dryft_fp4_quantise(int is_bf16, int kind, const void* x, long long stride, void* held, void* factors, int rows, int k, int pdl, void* stream) {
  if (rows <= 0 || k <= 0) return 0;
  const int item = is_bf16 ? 2 : 4;
  const bool words = ((uintptr_t)x & 15) == 0 && (rows == 1 || stride * item % 16 == 0);
  const int units = blocks_of(k) * (INPUTS / UNIT);
  int span = 32;   // lanes of a row
  while (span < THREADS && span < units) span *= 2;
  const dim3 grid((rows + THREADS / span - 1) / (THREADS / span));
  const cudaStream_t st = (cudaStream_t)stream;
  auto run = [&](auto kern, auto* p) { return launch(kern, grid, pdl, st, p, stride, (unsigned char*)held, (float*)factors, rows, k, span, words); };
  if (is_bf16) return kind == NV ? run(fp4_quantise_kernel<bf16, NV>, (const bf16*)x) : run(fp4_quantise_kernel<bf16, MX>, (const bf16*)x);
  return kind == NV ? run(fp4_quantise_kernel<float, NV>, (const float*)x) : run(fp4_quantise_kernel<float, MX>, (const float*)x);
}

// out [rows, k]: what the codes stand for
DRYFT_API int dryft_fp4_expand(int is_bf16, int kind, const void* held, const void* factors, void* out, int rows, int k, void* stream) {
  if (rows <= 0 || k <= 0) return 0;
  const int item = is_bf16 ? 2 : 4;
  const bool words = ((uintptr_t)out & 15) == 0 && ((long long)k * item % 16 == 0 || rows == 1);
  const unsigned units = (k + UNIT - 1) / UNIT;
  const unsigned long long all = (unsigned long long)rows * units;
  if ((all + THREADS - 1) / THREADS > 0x7fffffffull) return DRYFT_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)((all + THREADS - 1) / THREADS));
  const cudaStream_t st = (cudaStream_t)stream;
  auto run = [&](auto kern, auto* p) { return launch(kern, grid, false, st, (const unsigned char*)held, (const float*)factors, p, k, units, all, words); };
  if (is_bf16) return kind == NV ? run(fp4_expand_kernel<bf16, NV>, (bf16*)out) : run(fp4_expand_kernel<bf16, MX>, (bf16*)out);
  return kind == NV ? run(fp4_expand_kernel<float, NV>, (float*)out) : run(fp4_expand_kernel<float, MX>, (float*)out);
}
