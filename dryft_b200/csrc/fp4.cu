// Rounding rows to microscaled 4-bit floating point (fp4.cuh has the format and the layout) and taking them out again.
#include "fp4.cuh"

namespace {
using namespace fp4;
typedef __nv_bfloat16 bf16;
constexpr int UNIT = 16;        // numbers that a lane has at a time
constexpr int THREADS = 256, WARPS = THREADS / 32, BLOCK_UNITS = INPUTS / UNIT;

// Sixteen numbers as they lie in memory.
template <typename T> struct Raw { unsigned w[UNIT * sizeof(T) / 4]; };
__device__ __forceinline__ float number(const Raw<bf16>& r, int i) { return __uint_as_float(i & 1 ? r.w[i / 2] & 0xffff0000u : r.w[i / 2] << 16); }
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
// SILU: the row holds gate numbers, then as many others: silu(gate) rounded, times the other, rounded (the points of `silu_mul`).
template <typename T, bool SILU> __device__ __forceinline__ Raw<T> load_unit(const T* row, int c, int k, bool words) {
  Raw<T> r = load(row, c, k, words);
  if constexpr (SILU) {
    const Raw<T> up = load(row + k, c, k, words);
#pragma unroll
    for (int i = 0; i < UNIT / 2; ++i) {
      float v[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float g = number(r, 2 * i + e);
        v[e] = rnd<bf16>(__fdividef(g, 1.f + __expf(-g))) * number(up, 2 * i + e);   // (a few 32-bit ulp: far inside the rounding to bfloat16)
      }
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
    for (int i = 0; i < UNIT / 2; ++i) most = __vmaxu2(most, r.w[i] & 0x7fff7fffu);
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

// A row is 1, 2, 4 or 8 warps' (`span` lanes); a lane has HELD units in registers at a time, `span` apart.  NV wants the row's largest number first: a row that is held whole
// (bfloat16: up to 16,384 numbers) is read once.
template <typename T, int KIND, bool SILU>
__global__ void __launch_bounds__(THREADS) fp4_quantise_kernel(const T* x, long long stride, unsigned char* held, float* factors, int rows, int k, int span, bool words) {
  typedef Format<KIND> F;
  constexpr int HELD = sizeof(T) == 2 ? 4 : 2;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  let_next_launch_in();   // (behind the wait: what comes in may rely on all that was written before this launch)
  __shared__ unsigned most_s[WARPS];
  const int at = threadIdx.x & (span - 1), row = blockIdx.x * (THREADS / span) + threadIdx.x / span, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int units = row < rows ? blocks_of(k) * BLOCK_UNITS : 0;   // (a warp is one row's)
  const T* const from = x + (row < rows ? row : 0) * stride;
  auto take = [&](Raw<T> (&r)[HELD], int base) {
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      const int i = base + j * span + at;
      if (i < units) r[j] = load_unit<T, SILU>(from, i * UNIT, k, words);
    }
  };
  Raw<T> r[HELD] = {};
  take(r, 0);
  float factor = 0.f, u = 0.f;
  if (KIND == NV) {
    unsigned most = 0;
#pragma unroll
    for (int j = 0; j < HELD; ++j) most = max(most, size_of(r[j]).most);
    for (int base = HELD * span; base < units; base += HELD * span) {
      Raw<T> more[HELD] = {};
      take(more, base);
#pragma unroll
      for (int j = 0; j < HELD; ++j) most = max(most, size_of(more[j]).most);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (span > 32) {
      if (lane == 0) most_s[warp] = most;
      __syncthreads();
      const int first = warp & ~(span / 32 - 1);
      for (int w = 0; w < span / 32; ++w) most = max(most, most_s[first + w]);
    }
    factor = fmaxf(__fdiv_rn(__uint_as_float(most), 2688.f), __uint_as_float((127u - 112u) << 23));
    u = __frcp_rn(6.f * factor);
    if (at == 0 && row < rows) factors[row] = factor;
  }
  unsigned char* const block_row = held + (size_t)(row / ROWS) * blocks_of(k) * F::BLOCK_BYTES;
  const int r128 = row % ROWS;
  for (int base = 0; base < units; base += HELD * span) {   // (whole warps, for the exchanges)
    if (base > 0) take(r, base);
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      const int i = base + j * span + at;
      if (base + j * span >= units) break;
      Size s = size_of(r[j]);
      unsigned byte, word;
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
      uint2 c = make_uint2(codes8(r[j], 0, by), codes8(r[j], 8, by));
      if (s.bad) c = make_uint2(0x22222222u, 0x22222222u);
      if (i < units) {
        unsigned char* const block = block_row + (size_t)(i / BLOCK_UNITS) * F::BLOCK_BYTES;
        const int unit = i % BLOCK_UNITS;
        *reinterpret_cast<uint2*>(block + F::SCALE_BYTES + code_at(r128, unit)) = c;
        constexpr int PER_WORD = F::WORD_INPUTS / UNIT;
        if (unit % PER_WORD == 0) *reinterpret_cast<unsigned*>(block + scale_word_at(r128, unit / PER_WORD)) = word;
      }
    }
  }
}

// A block of 128 rows by 256 inputs a thread block, two rows a warp at a time: sixteen numbers a lane.
template <typename O, int KIND>
__global__ void __launch_bounds__(THREADS) fp4_expand_kernel(const unsigned char* held, const float* factors, O* out, int rows, int k) {
  typedef Format<KIND> F;
  constexpr int STEPS = ROWS / (2 * WARPS);
  const int KB = blocks_of(k), kb = blockIdx.x % KB, rb = blockIdx.x / KB, unit = threadIdx.x % BLOCK_UNITS, first = threadIdx.x / BLOCK_UNITS;
  const int c0 = kb * INPUTS + unit * UNIT;
  if (c0 >= k) return;
  const unsigned char* const block = held + (size_t)blockIdx.x * F::BLOCK_BYTES;
  constexpr int PER = UNIT / F::GROUP > 0 ? 1 : F::GROUP / UNIT;
  const int group = unit / PER, left = rows - rb * ROWS;
  uint2 c[STEPS];
  unsigned char sb[STEPS];
  float g[STEPS];
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int r = first + i * 2 * WARPS;
    if (r < left) {
      c[i] = *reinterpret_cast<const uint2*>(block + F::SCALE_BYTES + code_at(r, unit));
      sb[i] = block[scale_word_at(r, group / 4) + group % 4];
      g[i] = KIND == NV ? factors[rb * ROWS + r] : 1.f;
    }
  }
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int r = first + i * 2 * WARPS;
    if (r >= left) break;
    const float s = scale_value(sb[i], KIND == NV);
    float v[UNIT];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      unsigned two;
      asm("{ .reg .b8 b; cvt.u8.u32 b, %1; cvt.rn.f16x2.e2m1x2 %0, b; }" : "=r"(two) : "r"((j < 4 ? c[i].x >> (8 * j) : c[i].y >> (8 * (j - 4))) & 0xffu));
      const __half2 h = *reinterpret_cast<const __half2*>(&two);
      v[2 * j] = __low2float(h) * s;
      v[2 * j + 1] = __high2float(h) * s;
      if (KIND == NV) {
        v[2 * j] *= g[i];
        v[2 * j + 1] *= g[i];
      }
    }
    O* const to = out + (size_t)(rb * ROWS + r) * k + c0;
    if (c0 + UNIT <= k) {
      unsigned w[UNIT * sizeof(O) / 4];
#pragma unroll
      for (int j = 0; j < (int)(UNIT * sizeof(O) / 4); ++j) {
        if (sizeof(O) == 4) w[j] = __float_as_uint(v[j]);
        else {
          const __nv_bfloat162 two = __floats2bfloat162_rn(v[2 * j % UNIT], v[(2 * j + 1) % UNIT]);
          w[j] = *reinterpret_cast<const unsigned*>(&two);
        }
      }
#pragma unroll
      for (int j = 0; j < (int)(UNIT * sizeof(O) / 4); j += 8) st_words8(to + 4 * j / sizeof(O), w + j);
    } else {
#pragma unroll
      for (int j = 0; j < UNIT; ++j)
        if (c0 + j < k) to[j] = from_f32<O>(v[j]);
    }
  }
}

// The same where rows of results begin anywhere: a column a thread, so that a warp's results lie behind one another.
template <typename O, int KIND> __global__ void __launch_bounds__(THREADS) fp4_expand_columns_kernel(const unsigned char* held, const float* factors, O* out, int rows, int k) {
  typedef Format<KIND> F;
  static_assert(THREADS == INPUTS, "a thread a column");
  const int KB = blocks_of(k), kb = blockIdx.x % KB, rb = blockIdx.x / KB, in = threadIdx.x, c = kb * INPUTS + in, left = min(ROWS, rows - rb * ROWS), group = in / F::GROUP;
  if (c >= k) return;
  const unsigned char* const block = held + (size_t)blockIdx.x * F::BLOCK_BYTES;
#pragma unroll 8
  for (int r = 0; r < left; ++r) {
    const unsigned code = block[F::SCALE_BYTES + code_at(r, in / UNIT) + in % UNIT / 2] >> in % 2 * 4;
    unsigned two;
    asm("{ .reg .b8 b; cvt.u8.u32 b, %1; cvt.rn.f16x2.e2m1x2 %0, b; }" : "=r"(two) : "r"(code & 15u));
    const float v = __low2float(*reinterpret_cast<const __half2*>(&two)) * scale_value(block[scale_word_at(r, group / 4) + group % 4], KIND == NV);
    out[(size_t)(rb * ROWS + r) * k + c] = from_f32<O>(KIND == NV ? v * factors[rb * ROWS + r] : v);
  }
}

template <typename... P, typename... A> int launch(void (*kern)(P...), unsigned blocks, bool dependent, cudaStream_t st, A... a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
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

// held: blocks of 128 rows by 256 inputs (fp4.cuh); factors: float [rows] (NV).  x: rows of k numbers, `stride` numbers apart, anywhere.  silu (bfloat16): rows of 2 k numbers,
// silu of the first half times the second.
DRYFT_API int dryft_fp4_quantise(int is_bf16, int kind, int silu, const void* x, long long stride, void* held, void* factors, int rows, int k, int pdl, void* stream) {
  if (rows <= 0 || k <= 0) return 0;
  if (silu && !is_bf16) return DRYFT_ERR_UNSUPPORTED;
  const int item = is_bf16 ? 2 : 4, held_units = is_bf16 ? 4 : 2;
  const bool words = ((uintptr_t)x & 15) == 0 && (rows == 1 || stride * item % 16 == 0) && (!silu || (long long)k * item % 16 == 0);
  const int units = blocks_of(k) * BLOCK_UNITS;
  // lanes of a row: as many as hold it, or of few rows as many as it has units for (a row's latency is then what counts)
  int span = 32;
  while (span < THREADS && span * (rows <= 512 ? 1 : held_units) < units) span *= 2;
  const unsigned blocks = (unsigned)((rows + (long long)(THREADS / span) - 1) / (THREADS / span));
  const cudaStream_t st = (cudaStream_t)stream;
  auto run = [&](auto kern, auto* p) { return launch(kern, blocks, pdl, st, p, stride, (unsigned char*)held, (float*)factors, rows, k, span, words); };
  if (silu) return kind == NV ? run(fp4_quantise_kernel<bf16, NV, true>, (const bf16*)x) : run(fp4_quantise_kernel<bf16, MX, true>, (const bf16*)x);
  if (is_bf16) return kind == NV ? run(fp4_quantise_kernel<bf16, NV, false>, (const bf16*)x) : run(fp4_quantise_kernel<bf16, MX, false>, (const bf16*)x);
  return kind == NV ? run(fp4_quantise_kernel<float, NV, false>, (const float*)x) : run(fp4_quantise_kernel<float, MX, false>, (const float*)x);
}

// out [rows, k]: what the codes stand for
DRYFT_API int dryft_fp4_expand(int is_bf16, int kind, const void* held, const void* factors, void* out, int rows, int k, void* stream) {
  if (rows <= 0 || k <= 0) return 0;
  const bool words = ((uintptr_t)out & 31) == 0 && ((long long)k * (is_bf16 ? 2 : 4) % 32 == 0 || rows == 1);
  const long long blocks = (long long)((rows + ROWS - 1) / ROWS) * blocks_of(k);
  if (blocks > 0x7fffffffll) return DRYFT_ERR_UNSUPPORTED;
  const cudaStream_t st = (cudaStream_t)stream;
  auto run = [&](auto kern, auto* p) { return launch(kern, (unsigned)blocks, false, st, (const unsigned char*)held, (const float*)factors, p, rows, k); };
  auto columns = [&](auto kern, auto* p) { return launch(kern, (unsigned)blocks, false, st, (const unsigned char*)held, (const float*)factors, p, rows, k); };
  if (!words && is_bf16) return kind == NV ? columns(fp4_expand_columns_kernel<bf16, NV>, (bf16*)out) : columns(fp4_expand_columns_kernel<bf16, MX>, (bf16*)out);
  if (!words) return kind == NV ? columns(fp4_expand_columns_kernel<float, NV>, (float*)out) : columns(fp4_expand_columns_kernel<float, MX>, (float*)out);
  if (is_bf16) return kind == NV ? run(fp4_expand_kernel<bf16, NV>, (bf16*)out) : run(fp4_expand_kernel<bf16, MX>, (bf16*)out);
  return kind == NV ? run(fp4_expand_kernel<float, NV>, (float*)out) : run(fp4_expand_kernel<float, MX>, (float*)out);
}
