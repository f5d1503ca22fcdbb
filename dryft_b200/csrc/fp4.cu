// Rounding rows to microscaled 4-bit floating point (fp4.cuh has the format and the layout) and taking them out again.
#include "fp4.cuh"

namespace {
using namespace fp4;
typedef __nv_bfloat16 bf16;
constexpr int THREADS = 256, WARPS = THREADS / 32;

// A row is 1, 2, 4 or 8 warps' (`span` lanes); a lane has HELD units in registers at a time, `span` apart.  NV wants the row's largest number first: a row that is held whole
// (bfloat16: up to 12,288 numbers) is read once.  Its blocks wait for their rows' first numbers, then for each other's maxima: four of them a multiprocessor, with three units a
// lane, hide more of that than two with four (2,000 rows of 9,728: 15.6 us and 17.8; of 2,560: 6.4 and 7.6).
template <typename T, int KIND> __host__ __device__ constexpr int held_units() { return sizeof(T) == 4 ? 2 : KIND == NV ? 3 : 4; }
template <typename T, int KIND, bool SILU>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 2 && KIND == NV ? 4 : 1) fp4_quantise_kernel(const T* x, long long stride, unsigned char* held, float* factors, int rows, int k, int span, bool words, bool signal) {
  typedef Format<KIND> F;
  constexpr int HELD = held_units<T, KIND>();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (signal) let_next_launch_in();   // (behind the wait: what comes in may rely on all that was written before this launch)
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
    factor = row_factor(most);
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
      unsigned word;
      const uint2 c = round_unit<KIND>(r[j], factor, u, word);
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

// The same where rows of results begin anywhere: a column of some rows a thread, so that a warp's results lie behind one another.
constexpr int COLUMN_ROWS = 8;
template <typename O, int KIND> __global__ void __launch_bounds__(THREADS) fp4_expand_columns_kernel(const unsigned char* held, const float* factors, O* out, int rows, int k) {
  typedef Format<KIND> F;
  static_assert(THREADS == INPUTS, "a thread a column");
  const int KB = blocks_of(k), kb = blockIdx.x % KB, rb = blockIdx.x / KB, in = threadIdx.x, c = kb * INPUTS + in, group = in / F::GROUP;
  const int first = blockIdx.y * COLUMN_ROWS, left = min(first + COLUMN_ROWS, rows - rb * ROWS);
  if (c >= k) return;
  const unsigned char* const block = held + (size_t)blockIdx.x * F::BLOCK_BYTES;
#pragma unroll
  for (int r = first; r < left; ++r) {
    const unsigned code = block[F::SCALE_BYTES + code_at(r, in / UNIT) + in % UNIT / 2] >> in % 2 * 4;
    unsigned two;
    asm("{ .reg .b8 b; cvt.u8.u32 b, %1; cvt.rn.f16x2.e2m1x2 %0, b; }" : "=r"(two) : "r"(code & 15u));
    const float v = __low2float(*reinterpret_cast<const __half2*>(&two)) * scale_value(block[scale_word_at(r, group / 4) + group % 4], KIND == NV);
    out[(size_t)(rb * ROWS + r) * k + c] = from_f32<O>(KIND == NV ? v * factors[rb * ROWS + r] : v);
  }
}

template <typename... P, typename... A> int launch(void (*kern)(P...), dim3 blocks, bool dependent, cudaStream_t st, A... a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = blocks;
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
// silu of the first half times the second.  pdl: 1, a programmatic dependent of the launch before it; 2, the next
// launch may be one of this (it then reads what this writes behind its own wait).
DRYFT_API int dryft_fp4_quantise(int is_bf16, int kind, int silu, const void* x, long long stride, void* held, void* factors, int rows, int k, int pdl, void* stream) {
  if (rows <= 0 || k <= 0) return 0;
  if (silu && !is_bf16) return DRYFT_ERR_UNSUPPORTED;
  const int item = is_bf16 ? 2 : 4, held_at_a_time = !is_bf16 ? held_units<float, NV>() : kind == NV ? held_units<bf16, NV>() : held_units<bf16, MX>();
  const bool words = ((uintptr_t)x & 15) == 0 && (rows == 1 || stride * item % 16 == 0) && (!silu || (long long)k * item % 16 == 0);
  const int units = blocks_of(k) * BLOCK_UNITS;
  // lanes of a row: as many as hold it, or of few rows as many as it has units for (a row's latency is then what counts)
  int span = 32;
  while (span < THREADS && span * (rows <= 512 ? 1 : held_at_a_time) < units) span *= 2;
  const unsigned blocks = (unsigned)((rows + (long long)(THREADS / span) - 1) / (THREADS / span));
  const cudaStream_t st = (cudaStream_t)stream;
  auto run = [&](auto kern, auto* p) { return launch(kern, blocks, pdl & 1, st, p, stride, (unsigned char*)held, (float*)factors, rows, k, span, words, (pdl & 2) != 0); };
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
  auto columns = [&](auto kern, auto* p) { return launch(kern, dim3((unsigned)blocks, ROWS / COLUMN_ROWS), false, st, (const unsigned char*)held, (const float*)factors, p, rows, k); };
  if (!words && is_bf16) return kind == NV ? columns(fp4_expand_columns_kernel<bf16, NV>, (bf16*)out) : columns(fp4_expand_columns_kernel<bf16, MX>, (bf16*)out);
  if (!words) return kind == NV ? columns(fp4_expand_columns_kernel<float, NV>, (float*)out) : columns(fp4_expand_columns_kernel<float, MX>, (float*)out);
  if (is_bf16) return kind == NV ? run(fp4_expand_kernel<bf16, NV>, (bf16*)out) : run(fp4_expand_kernel<bf16, MX>, (bf16*)out);
  return kind == NV ? run(fp4_expand_kernel<float, NV>, (float*)out) : run(fp4_expand_kernel<float, MX>, (float*)out);
}
