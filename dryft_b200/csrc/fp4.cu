// Rounding rows to microscaled 4-bit floating point (fp4.cuh has the format and the layout) and taking them out again.
#include "fp4.cuh"

namespace {
using namespace fp4;
typedef __nv_bfloat16 bf16;
constexpr int THREADS = 256, WARPS = THREADS / 32;

// A row is 1 to 32 warps' (`span` lanes); a lane has HELD units in registers at a time, `span` apart.  NV wants the row's largest number first: a row that is held whole
// (bfloat16, 256 lanes: up to 12,288 numbers) is read once.  Its blocks wait for their rows' first numbers, then for each other's maxima: 1,024 threads a multiprocessor, of 64 registers,
// hide more of that than fewer with more in them (2,000 rows of 9,728, NV: 15.2 us, with 96 registers 17.8; MX with silu 24.5, 35.9; of 2,560 32-bit numbers, NV, 9.3, 12.0).  The bound of 64
// registers is one for all forms that read words, also where blocks have 256 or 512 threads: 32-bit NV spills 176 bytes a thread, NV with silu 88, MX with silu 4.
//
// What it takes: 2,000 rows of 9,728 in bfloat16 (39 MB read, 10 or 11 written: 7.5 us at a copy's rate) MX 11.7 us, NV 15.2; with silu (78 MB read: 13.4) 24.5 and 29; rows that begin anywhere 16.6 and
// 22.7.  Nothing is full: issue slots two thirds (8.0 and 10.6 million instructions of a warp, without silu: 13 and 17 for a number of each lane), memory 61%; a block's rows come
// first, then are worked on, and what is resident beside it does not cover that.  Blocks of 512 or 1,024 threads and roundings in packed bfloat16 were no faster.
template <typename T, int KIND> __host__ __device__ constexpr int held_units() { return sizeof(T) == 4 ? 2 : KIND == NV ? 3 : 4; }
// WORDS: rows begin on 16-byte boundaries (silu: both halves of them).
constexpr int MOST_LANES = 1024;
template <typename T, int KIND, bool SILU, bool WORDS>
__global__ void __launch_bounds__(WORDS ? MOST_LANES : THREADS, 1) fp4_quantise_kernel(const T* x, long long stride, unsigned char* held, float* factors, int rows, int k, int span, bool signal) {
  typedef Format<KIND> F;
  constexpr int HELD = held_units<T, KIND>();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (signal) let_next_launch_in();   // (behind the wait: what comes in may rely on all that was written before this launch)
  __shared__ unsigned most_s[MOST_LANES / 32];
  const int at = threadIdx.x & (span - 1), row = blockIdx.x * (blockDim.x / span) + threadIdx.x / span, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int units = row < rows ? blocks_of(k) * BLOCK_UNITS : 0;   // (a warp is one row's)
  const T* const from = x + (row < rows ? row : 0) * stride;
  auto take = [&](Raw<T> (&r)[HELD], int base) {
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      const int i = base + j * span + at;
      if (i < units) r[j] = load_unit<T, SILU, !WORDS>(from, i * UNIT, k, true);
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

// A block of 128 rows by 256 inputs a thread block, two rows a warp at a time: sixteen numbers a lane, whose results are whole sectors, all of a lane's codes asked for first.  Bound by
// what it writes: 19,456 rows of 2,560, MX, as bfloat16 (26.5 MB in, 100 out) 22 us, 5,700 GB/s.
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

// The same where rows of results begin anywhere: a row's 256 numbers a warp at a time, eight a lane, by way of shared memory, so that what crosses memory is 16-byte words, but for a
// segment's two ends: 2,000 rows of 9,729 15.3 us as bfloat16 (rows on 32-byte boundaries 9.6), 24.7 in 32 bits; a number a lane straight to memory 46, the lanes' work.
constexpr int SHIFTED_ROWS = 4;   // rows of a warp
template <typename O, int KIND> __global__ void __launch_bounds__(THREADS) fp4_expand_shifted_kernel(const unsigned char* held, const float* factors, O* out, int rows, int k) {
  typedef Format<KIND> F;
  constexpr int PER = INPUTS / 32, BYTES = INPUTS * sizeof(O);
  __shared__ __align__(16) unsigned words_s[WARPS][BYTES / 4 + 4];
  const int KB = blocks_of(k), kb = blockIdx.x % KB, rb = blockIdx.x / KB, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = (blockIdx.y * WARPS + warp) * SHIFTED_ROWS, left = min(SHIFTED_ROWS, rows - rb * ROWS - first), group = lane * PER / F::GROUP;
  const unsigned char* const block = held + (size_t)blockIdx.x * F::BLOCK_BYTES;
  unsigned* const words = words_s[warp];
  unsigned c[SHIFTED_ROWS];
  unsigned char sb[SHIFTED_ROWS];
  float g[SHIFTED_ROWS];
#pragma unroll
  for (int i = 0; i < SHIFTED_ROWS; ++i)
    if (i < left) {
      c[i] = *reinterpret_cast<const unsigned*>(block + F::SCALE_BYTES + code_at(first + i, lane / 2) + lane % 2 * 4);
      sb[i] = block[scale_word_at(first + i, group / 4) + group % 4];
      g[i] = KIND == NV ? factors[rb * ROWS + first + i] : 1.f;
    }
#pragma unroll
  for (int i = 0; i < SHIFTED_ROWS; ++i) {
    if (i >= left) break;
    const float s = scale_value(sb[i], KIND == NV);
    O v[PER];
#pragma unroll
    for (int j = 0; j < PER / 2; ++j) {
      unsigned two;
      asm("{ .reg .b8 b; cvt.u8.u32 b, %1; cvt.rn.f16x2.e2m1x2 %0, b; }" : "=r"(two) : "r"((c[i] >> (8 * j)) & 0xffu));
      const __half2 h = *reinterpret_cast<const __half2*>(&two);
      const float lo = __low2float(h) * s, hi = __high2float(h) * s;
      v[2 * j] = from_f32<O>(KIND == NV ? lo * g[i] : lo);
      v[2 * j + 1] = from_f32<O>(KIND == NV ? hi * g[i] : hi);
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < (int)(PER * sizeof(O) / 16); ++j) reinterpret_cast<uint4*>(words)[lane * (PER * sizeof(O) / 16) + j] = reinterpret_cast<const uint4*>(v)[j];
    __syncwarp();
    O* const to = out + (size_t)(rb * ROWS + first + i) * k + kb * INPUTS;
    const int size = min(INPUTS, k - kb * INPUTS) * (int)sizeof(O);                                  // bytes of the segment
    const int head = min((int)(-reinterpret_cast<uintptr_t>(to) & 15), size), whole = (size - head) / 16, tail = head + 16 * whole;   // up to the first word, words, where the rest begins
    for (int w = lane; w < whole; w += 32) {
      const int from = head + 16 * w, shift = from & 2 ? 16 : 0;
      unsigned a[5], b[4];
#pragma unroll
      for (int j = 0; j < 5; ++j) a[j] = words[from / 4 + j];
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = __funnelshift_r(a[j], a[j + 1], shift);
      *reinterpret_cast<uint4*>(reinterpret_cast<unsigned char*>(to) + from) = make_uint4(b[0], b[1], b[2], b[3]);
    }
    const O* const numbers = reinterpret_cast<const O*>(words);
    if (lane * (int)sizeof(O) < head) to[lane] = numbers[lane];
    const int end = tail / (int)sizeof(O) + lane;
    if (lane < 8 && end * (int)sizeof(O) < size) to[end] = numbers[end];
  }
}

template <typename... P, typename... A> int launch(void (*kern)(P...), dim3 blocks, int threads, bool dependent, cudaStream_t st, A... a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = blocks;
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, (P)a...);
  return e != cudaSuccess ? (int)e : launch_status();
}
// of the current device
int multiprocessors() {
  static int of[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
  if (of[dev] == 0 && cudaDeviceGetAttribute(&of[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) of[dev] = 1;
  return of[dev];
}
}  // namespace

// Lanes of a row: as many as hold it, or of few rows (no more than multiprocessors) as many as it has units for (a row's latency is then what counts): up to 256, from where on NV's maxima cost more
// than units side by side give (48 rows of 9,728: 3.0 us with 256 lanes, 3.7 with 1,024; MX 2.4 either way, but with silu 4.0 and 3.6).  More than 256: for rows that have a multiprocessor each (25,600
// numbers of NV 6.0 and 4.6, with silu 16.0 and 8.3, of MX 4.0 and 3.2), or where NV would work out a row's numbers, or read 32 bits of each, twice (2,000 rows of 25,600, silu: 90 and with 512
// lanes 83, 32-bit numbers 82 and 76; bfloat16 as it is 38 and 44).
DRYFT_API int dryft_fp4_lanes(int is_bf16, int kind, int silu, int words, int rows, int k, int multiprocessors) {
  const int held_at_a_time = !is_bf16 ? held_units<float, NV>() : kind == NV ? held_units<bf16, NV>() : held_units<bf16, MX>(), units = blocks_of(k) * BLOCK_UNITS;
  const bool few = rows <= multiprocessors;
  const int most = !words ? THREADS : few ? MOST_LANES : kind == NV && (silu || !is_bf16) ? 512 : THREADS;
  int span = 32;
  while (span < most && span * ((few && kind == MX && (silu || !is_bf16)) || (rows <= 512 && span < THREADS) ? 1 : held_at_a_time) < units) span *= 2;
  return span;
}

// held: blocks of 128 rows by 256 inputs (fp4.cuh); factors: float [rows] (NV).  x: rows of k numbers, `stride` numbers apart, anywhere.  silu (bfloat16): rows of 2 k numbers,
// silu of the first half times the second.  pdl: 1, a programmatic dependent of the launch before it; 2, the next
// launch may be one of this (it then reads what this writes behind its own wait).
DRYFT_API int dryft_fp4_quantise(int is_bf16, int kind, int silu, const void* x, long long stride, void* held, void* factors, int rows, int k, int pdl, void* stream) {
  if (rows <= 0 || k <= 0) return 0;
  if (silu && !is_bf16) return DRYFT_ERR_UNSUPPORTED;
  const int item = is_bf16 ? 2 : 4;
  const bool words = ((uintptr_t)x & 15) == 0 && (rows == 1 || stride * item % 16 == 0) && (!silu || (long long)k * item % 16 == 0);
  const int span = dryft_fp4_lanes(is_bf16, kind, silu, words, rows, k, multiprocessors());
  const int threads = span > THREADS ? span : THREADS;
  const unsigned blocks = (unsigned)((rows + (long long)(threads / span) - 1) / (threads / span));
  const cudaStream_t st = (cudaStream_t)stream;
  auto run = [&](auto kern, auto* p) { return launch(kern, blocks, threads, pdl & 1, st, p, stride, (unsigned char*)held, (float*)factors, rows, k, span, (pdl & 2) != 0); };
  auto by_words = [&](auto with, auto without, auto* p) { return words ? run(with, p) : run(without, p); };
  const bf16* const xb = (const bf16*)x;
  const float* const xf = (const float*)x;
  if (silu)
    return kind == NV ? by_words(fp4_quantise_kernel<bf16, NV, true, true>, fp4_quantise_kernel<bf16, NV, true, false>, xb)
                      : by_words(fp4_quantise_kernel<bf16, MX, true, true>, fp4_quantise_kernel<bf16, MX, true, false>, xb);
  if (is_bf16)
    return kind == NV ? by_words(fp4_quantise_kernel<bf16, NV, false, true>, fp4_quantise_kernel<bf16, NV, false, false>, xb)
                      : by_words(fp4_quantise_kernel<bf16, MX, false, true>, fp4_quantise_kernel<bf16, MX, false, false>, xb);
  return kind == NV ? by_words(fp4_quantise_kernel<float, NV, false, true>, fp4_quantise_kernel<float, NV, false, false>, xf)
                    : by_words(fp4_quantise_kernel<float, MX, false, true>, fp4_quantise_kernel<float, MX, false, false>, xf);
}

// out [rows, k]: what the codes stand for
DRYFT_API int dryft_fp4_expand(int is_bf16, int kind, const void* held, const void* factors, void* out, int rows, int k, void* stream) {
  if (rows <= 0 || k <= 0) return 0;
  const bool words = ((uintptr_t)out & 31) == 0 && ((long long)k * (is_bf16 ? 2 : 4) % 32 == 0 || rows == 1);
  const long long blocks = (long long)((rows + ROWS - 1) / ROWS) * blocks_of(k);
  if (blocks > 0x7fffffffll) return DRYFT_ERR_UNSUPPORTED;
  const cudaStream_t st = (cudaStream_t)stream;
  auto run = [&](auto kern, auto* p) { return launch(kern, (unsigned)blocks, THREADS, false, st, (const unsigned char*)held, (const float*)factors, p, rows, k); };
  auto shifted = [&](auto kern, auto* p) { return launch(kern, dim3((unsigned)blocks, ROWS / (WARPS * SHIFTED_ROWS)), THREADS, false, st, (const unsigned char*)held, (const float*)factors, p, rows, k); };
  if (!words && is_bf16) return kind == NV ? shifted(fp4_expand_shifted_kernel<bf16, NV>, (bf16*)out) : shifted(fp4_expand_shifted_kernel<bf16, MX>, (bf16*)out);
  if (!words) return kind == NV ? shifted(fp4_expand_shifted_kernel<float, NV>, (float*)out) : shifted(fp4_expand_shifted_kernel<float, MX>, (float*)out);
  if (is_bf16) return kind == NV ? run(fp4_expand_kernel<bf16, NV>, (bf16*)out) : run(fp4_expand_kernel<bf16, MX>, (bf16*)out);
  return kind == NV ? run(fp4_expand_kernel<float, NV>, (float*)out) : run(fp4_expand_kernel<float, MX>, (float*)out);
}
