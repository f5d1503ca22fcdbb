// y = x w^T with both operands in microscaled 4-bit floating point (fp4.cuh), on the 5th-generation tensor cores, which multiply such numbers and scales as they lie:
// tcgen05.mma kind::mxf4 (a scale for 32 inputs) and kind::mxf4nvf4 (for 16), 64 inputs an instruction, summed in 32 bits.  A product of two codes is a multiple of 1/4, so what an
// instruction sums before the scales is exact.  Measured with normal random operands of 25,600 inputs: MX results are the definition's in 32 bits, NV results off by 5e-8 of the whole (a
// product of the same values in 32 bits by the library: 8e-7).  Where groups differ far in size a sum is cut off below 2^-21 of its terms' magnitudes, an instruction, at the most.
//
// Computed transposed: a tile is 128 rows of W, on the M side, against NB rows of x (16 to 128, padded to whole sixteens), its sums in tensor memory, a W row a lane: results are written
// a column at a time, 32 lanes' behind one another.  A stage of the ring is 256 inputs: a block of W and one of x, each one copy of consecutive bytes (the layout is the tensor
// cores' own, so no tensor maps).  The scales go on from shared into tensor memory (tcgen05.cp) in front of the four products of their stage, by the thread that issues those:
// the copies and products of one thread run in the order that they were issued in; two stages' scales have places of their own.
//
// Which form: one tile for up to 128 rows of x; blocks walk the tiles, two a multiprocessor (one's products and copies are the other's time to write), or, where tiles are few, a cluster
// shares a tile's inputs and adds up through distributed shared memory (SPLIT); up to 16 rows are rounded by every block for itself (SRC).  Many rows: pairs of blocks with one
// 256-row tile of W between them (below).  ops/kernels.py:_fp4_plan chooses, with both sides' figures.
//
// What bounds it.  Few rows: W's bytes.  151,936 outputs of 2,560 inputs, 1 row: 33.6 us, 6,500 GB/s, 99% of a copy's rate; with fewer bytes the launch, first bytes and a tile's end: 8 rows,
// 19,456 of 2,560 (MX, 26.5 MB) 7.2 us where the bytes are 4.1; 1 row (NV), 6,144 of 2,560 4.1 and 1.35, 2,560 of 9,728 4.8 and 2.1.  Many rows: what
// enters a multiprocessor.  2,048 rows, 5,120 of 25,600 (pairs with 192 columns): NV 103 us, MX 91.5, 5.9 PFLOP/s, 104 GB/s into each, 15 TB/s in all; 24,576 of 4,096 (256
// columns): 83 us, 5.0 PFLOP/s, and 75.5.  MX has 0.91 and 0.92 of NV's bytes, takes 0.89 and 0.91 of its time, and has the same products; the tensor pipe is 62% busy.  Larger tiles would
// read less for as much work: 512 outputs by 192 rows leave tensor memory room for one set of sums and two stages' scales, so that products wait while sums are read, and there are half as
// many tiles to share out.  Not built.
//
// Warps: 0 copies, 1 issues, the others read the sums out.  Every wait on a barrier is bounded by a clock; a waiter that gives up raises *err, every role leaves its loop, the block lets its
// copies and products end and frees its tensor memory.
#include "fp4.cuh"
#include "drain.h"
#include <type_traits>

namespace {
using namespace fp4;
typedef __nv_bfloat16 bf16;
constexpr long long WAIT_CYCLES = 2000000000LL;
constexpr unsigned SLEEP_NS = 10000;

__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(void* bar, unsigned count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(void* bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(void* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(void* bar, unsigned parity) {
  unsigned ok;
  asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3; selp.u32 %0, 1, 0, p; }"
               : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity), "r"(SLEEP_NS) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_try_wait_cluster(void* bar, unsigned parity) {   // for what other blocks of the cluster arrive at
  unsigned ok;
  asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3; selp.u32 %0, 1, 0, p; }"
               : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity), "r"(SLEEP_NS) : "memory");
  return ok != 0;
}
template <bool CLUSTER = false> __device__ __forceinline__ bool mbar_wait(void* bar, unsigned parity, int* err, volatile int* failed, int site) {
  auto there = [&] { return CLUSTER ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity); };
  if (there()) return true;
  const long long t0 = clock64();
  while (!there()) {
    if (*failed) return false;
    if (clock64() - t0 > WAIT_CYCLES) {
      if (err) atomicCAS(err, 0, 300 + site);   // the first wait that gave up names its place
      *failed = 1;
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, unsigned bytes, void* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// codes: K-major, 128-byte swizzle, rows of 128 bytes (256 numbers), groups of eight rows 1024 bytes apart
__device__ __forceinline__ unsigned long long codes_desc(const void* smem) {
  return (unsigned long long)((smem_u32(smem) & 0x3FFFF) >> 4) | (unsigned long long)1 << 16 | (unsigned long long)(1024 >> 4) << 32 | (unsigned long long)1 << 46 |
         (unsigned long long)2 << 61;
}
// scales: 32 rows of 16 bytes, groups of eight rows 128 bytes apart, not swizzled
__device__ __forceinline__ unsigned long long scales_desc(const void* smem) {
  return (unsigned long long)((smem_u32(smem) & 0x3FFFF) >> 4) | (unsigned long long)(128 >> 4) << 32 | (unsigned long long)1 << 46;
}
// 32 rows of 16 bytes into four columns, the same in each quarter of the lanes
template <int CTAS = 1> __device__ __forceinline__ void scales_to_tmem(unsigned taddr, unsigned long long desc) {
  if (CTAS == 1) asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");   // in both blocks, each from its own shared memory
}
// Instruction descriptor: A and B E2M1, N >> 3 at bit 17 (added by the caller), scales' type at bit 23 (0 E4M3, 1 E8M0), M >> 7 at bit 27; which of a word's scales the instruction takes at
// bits 4 (B) and 29 (A): all four (NV), the first or the second two (MX).
template <int KIND, int M = 128> __device__ __forceinline__ constexpr unsigned idesc(int scale) {
  return (1u << 7) | (1u << 10) | (KIND == MX ? 1u << 23 : 0u) | ((unsigned)(M >> 7) << 27) | ((unsigned)scale << 4) | ((unsigned)scale << 29);
}
// D[tmem] (+)= A[smem] B[smem], 64 inputs
#define DRYFT_FP4_MMA(group, kind)                                                                       \
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                         \
               "tcgen05.mma.cta_group::" group "." kind " [%0], %1, %2, %3, [%4], [%5], p;\n\t}"           \
               ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(sa), "r"(sb), "r"(accumulate) : "memory")
template <int KIND, int CTAS = 1>
__device__ __forceinline__ void umma(unsigned d, unsigned long long a, unsigned long long b, unsigned id, unsigned sa, unsigned sb, unsigned accumulate) {
  if (KIND == NV && CTAS == 1) DRYFT_FP4_MMA("1", "kind::mxf4nvf4.block_scale.scale_vec::4X");
  else if (KIND == NV) DRYFT_FP4_MMA("2", "kind::mxf4nvf4.block_scale.scale_vec::4X");
  else if (CTAS == 1) DRYFT_FP4_MMA("1", "kind::mxf4.block_scale.scale_vec::2X");
  else DRYFT_FP4_MMA("2", "kind::mxf4.block_scale.scale_vec::2X");
}
__device__ __forceinline__ bool elected() {   // one lane of the warp
  unsigned one;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ void umma_commit(void* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_ld16(unsigned taddr, float (&v)[16]) {
  unsigned r[16];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

struct Params {
  const unsigned char *x, *w;          // blocks (fp4.cuh); x: or rows as they are (below)
  const float *x_factors, *w_factors;  // NV
  void* y;
  int* err;
  int m, n, blocks;   // blocks: of 256 inputs
  // of x as it is: numbers of a row, numbers between rows, whether 16-byte words can be read
  int k;
  long long x_stride;
  bool x_words;
};

constexpr int FUSED_ROWS = 16, FUSED_BLOCKS = 12;   // rows, and blocks of 256 inputs, that a block rounds for itself at most
// What x is: held in 4 bits, or rows that every block rounds for itself, of bfloat16 (SILU: of gate numbers and as many others) or 32-bit numbers.
enum Source { HELD = 0, BF16 = 1, SILU = 2, F32 = 3 };

// SPLIT: a tile's inputs are shared out among a cluster's blocks.
template <int KIND, int NB, bool SPLIT, int SRC> struct Layout {
  typedef Format<KIND> F;
  static constexpr bool FUSED = SRC != HELD;
  // warps that read sums: four take a quarter of the rows each, and PARTS fours a part of the columns, so that each scheduler has several to hide their latencies
  static constexpr int PARTS = NB <= 16 ? 1 : NB <= 32 ? 2 : 4, READERS = 4 * PARTS;
  static constexpr int ROUNDERS = FUSED ? READERS + 4 : 0, THREADS = (2 + (FUSED ? ROUNDERS : READERS)) * 32;   // warps that round x, the readers among them
  static constexpr int X_BYTES = F::SCALE_BYTES + NB * (INPUTS / 2), STAGE_BYTES = F::BLOCK_BYTES + (FUSED ? 0 : X_BYTES);   // W's block, as much of x's; multiples of 1024
  static constexpr int X_BLOCKS = FUSED ? FUSED_BLOCKS : 0;                                  // of x, which stay for all tiles
  // (of 64 registers where tiles have 128 columns and are not shared: two forms spill 8 bytes a thread)
  static constexpr int RESIDENT = 2, STAGES = (110 * 1024 - X_BLOCKS * X_BYTES) / STAGE_BYTES;   // RESIDENT: blocks of a multiprocessor
  // tensor memory: sums of ACCS tiles, then the scales of two stages
  static constexpr int ACCS = SPLIT || NB >= 128 ? 1 : 2, SCALE_COLS = 8 * F::WORDS, NEED_COLS = ACCS * NB + 2 * SCALE_COLS;
  static constexpr int TMEM_COLS = NEED_COLS <= 128 ? 128 : NEED_COLS <= 256 ? 256 : 512;
  static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + X_BLOCKS * X_BYTES + 8 * (2 * STAGES + 5) + 16;
  static_assert(RESIDENT * TMEM_COLS <= 512 && RESIDENT * (SMEM_BYTES + 2048) <= 228 * 1024 && STAGES >= 3, "of a block");
  static_assert(!SPLIT || (NB + 7 * 4) * ROWS * 4 <= STAGES * STAGE_BYTES, "sums fit where the stages were");
};

__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ unsigned cluster_size() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
// (relaxed: what the blocks of a cluster hand each other completes barriers of its own.  A release waits until all that the block has written is in place: a microsecond.)
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  cluster_arrive();
  cluster_wait();
}
// 16 bytes into another block's shared memory, at the address that this block has the like at; they complete a barrier there
__device__ __forceinline__ void send(unsigned addr, unsigned bar, unsigned rank, float a, float b, float c, float d) {
  asm volatile("{ .reg .u32 a, b; mapa.shared::cluster.u32 a, %0, %2; mapa.shared::cluster.u32 b, %1, %2;\n\t"
               "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [a], {%3, %4, %5, %6}, [b]; }"
               ::"r"(addr), "r"(bar), "r"(rank), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}
constexpr int MOST_BLOCKS = 8;   // of a cluster

// A row of W's factor (NV), taken in two steps.  A sum of codes times scales is 2^-20 at the least, 2^54 at the most, and the other row's factor 2^-112 to 2^117: times `of` it is far
// from both ends of 32 bits, whatever that other factor makes of it then; `rest` is a power of two, 1 but for rows of very large or small numbers.
// (Asked for early, and looked at where nothing waits for it: a block of a cluster that looked at it in front of its sums took 0.3 us longer.)  `far`: whether a row of the warp's has such a rest.
struct RowFactor { float of, rest; bool far; };
template <int KIND> __device__ __forceinline__ RowFactor in_steps(float f) {
  if (KIND != NV) return {1.f, 1.f, false};
  const RowFactor r = f > 0x1p60f ? RowFactor{f * 0x1p-48f, 0x1p48f, false} : f < 0x1p-80f ? RowFactor{f * 0x1p32f, 0x1p-32f, false} : RowFactor{f, 1.f, false};
  return {r.of, r.rest, __any_sync(0xffffffffu, r.rest != 1.f) != 0};
}

// A warp's results: columns (rows of x) of one row of W a lane.
template <int KIND, int COLS, typename O>
__device__ __forceinline__ void write_columns(const Params& p, O* to, bool there, int cols, float (&v)[COLS / 16][16], RowFactor own, const float (&x_factor)[(COLS + 31) / 32]) {
#pragma unroll
  for (int c = 0; c < COLS / 16; ++c) {
    if (16 * c >= cols) break;
    if (KIND == NV)
#pragma unroll
      for (int j = 0; j < 16; ++j) v[c][j] = v[c][j] * own.of * __shfl_sync(0xffffffffu, x_factor[c / 2], (16 * c + j) % 32);
    if (KIND == NV && own.far)
#pragma unroll
      for (int j = 0; j < 16; ++j) v[c][j] *= own.rest;
    if (there)   // (apart from the exchanges, which are all lanes')
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (16 * c + j < cols) to[(size_t)(16 * c + j) * p.n] = from_f32<O>(v[c][j]);
  }
}

// The rows' largest magnitudes' bits (FUSED, NV): of this block's inputs, then of whole rows; and what the cluster's blocks sent each other.
struct Most { unsigned rows[FUSED_ROWS], of[MOST_BLOCKS][FUSED_ROWS]; unsigned long long full; };

// The rounders' part (FUSED): the rows' inputs that this block multiplies, of blocks k0 to k1, into shared memory as the products want them.  NV wants the largest number of whole
// rows: the blocks of a cluster, which have a row's inputs between them, send each other theirs.  A thread has AHEAD units on their way at a time; its first ones stay in
// registers between looking and rounding, more are read again.
template <typename L, int KIND, int SRC, bool SPLIT>
__device__ __forceinline__ void round_x(const Params& p, int k0, int k1, unsigned char* xs, Most& most_s, unsigned long long* x_full, unsigned rank, unsigned size,
                                        volatile int* failed) {
  typedef typename L::F F;
  typedef typename std::conditional<SRC == F32, float, bf16>::type X;
  constexpr int THREADS = L::ROUNDERS * 32, AHEAD = 2;   // (four: 0.1 to 0.3 us longer for one to four rows, whose instructions a block meets for the first time)
  const int id = threadIdx.x - 64, lane = threadIdx.x & 31, own = (k1 - k0) * BLOCK_UNITS, all = p.m * own;
  const X* const x = reinterpret_cast<const X*>(p.x);
  // i / n, for i + 1/2 and n far below 2^23
  auto over = [](int i, float by) { return (int)(((float)i + 0.5f) * by); };
  const float by_own = 1.f / (float)own;
  auto load = [&](int i, int row) { return load_unit<X, SRC == SILU>(x + row * p.x_stride, (k0 * BLOCK_UNITS + i - row * own) * UNIT, p.k, p.x_words); };
  auto take = [&](Raw<X> (&r)[AHEAD], int base) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (base + j * THREADS + id < all) r[j] = load(base + j * THREADS + id, over(base + j * THREADS + id, by_own));
  };
  Raw<X> r[AHEAD] = {};
  take(r, 0);
  if (KIND == NV) {
    auto look = [&](const Raw<X>& r, bool there, int row) {   // sixteen neighbouring lanes have one row's
      unsigned most = there ? size_of(r).most : 0u;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
      if (there && lane % BLOCK_UNITS == 0) atomicMax(&most_s.rows[row], most);
    };
    auto look_all = [&](const Raw<X> (&r)[AHEAD], int base) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        if (base + j * THREADS < all) look(r[j], base + j * THREADS + id < all, over(base + j * THREADS + id, by_own));
    };
    look_all(r, 0);
    for (int base = AHEAD * THREADS; base < all; base += AHEAD * THREADS) {
      Raw<X> o[AHEAD] = {};
      take(o, base);
      look_all(o, base);
    }
    // the rounders' own barriers: what a rounder waits for in front of one ends, or runs out
    asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
    if constexpr (SPLIT) {
      for (unsigned i = id; i < size * FUSED_ROWS; i += THREADS)
        asm volatile("{ .reg .u32 a, b; mapa.shared::cluster.u32 a, %0, %3; mapa.shared::cluster.u32 b, %1, %3;\n\t"
                     "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [a], %2, [b]; }"
                     ::"r"(smem_u32(&most_s.of[rank][i % FUSED_ROWS])), "r"(smem_u32(&most_s.full)), "r"(most_s.rows[i % FUSED_ROWS]), "r"(i / FUSED_ROWS) : "memory");
      mbar_wait<true>(&most_s.full, 0, p.err, failed, 6);
      asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");   // (everybody has sent what `rows` was)
      if (id < FUSED_ROWS) {
        unsigned most = 0;
        for (unsigned b = 0; b < size; ++b) most = max(most, most_s.of[b][id]);
        most_s.rows[id] = most;
      }
      asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
    }
  }
  for (int base = 0; base < all; base += AHEAD * THREADS) {
    if (base > 0) take(r, base);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (base + j * THREADS >= all) break;
      const int i = base + j * THREADS + id, row = over(min(i, all - 1), by_own), c = i - row * own, unit = c % BLOCK_UNITS;
      const float factor = KIND == NV ? row_factor(most_s.rows[row]) : 1.f;
      unsigned word;
      const uint2 codes = round_unit<KIND>(r[j], factor, KIND == NV ? __frcp_rn(6.f * factor) : 1.f, word);
      if (i < all) {
        unsigned char* const block = xs + (size_t)(c / BLOCK_UNITS) * L::X_BYTES;
        constexpr int PER_WORD = F::WORD_INPUTS / UNIT;
        *reinterpret_cast<uint2*>(block + F::SCALE_BYTES + code_at(row, unit)) = codes;
        if (unit % PER_WORD == 0) *reinterpret_cast<unsigned*>(block + scale_word_at(row, unit / PER_WORD)) = word;
      }
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // what was written is read by the tensor cores
  mbar_arrive(x_full);
}

template <int KIND, int NB, bool SPLIT, int SRC, typename O>
__global__ void __launch_bounds__(Layout<KIND, NB, SPLIT, SRC>::THREADS, Layout<KIND, NB, SPLIT, SRC>::RESIDENT) linear_fp4_kernel(const Params p) {
  typedef Layout<KIND, NB, SPLIT, SRC> L;
  typedef typename L::F F;
  constexpr int STAGES = L::STAGES, READ_THREADS = L::READERS * 32;
  constexpr bool FUSED = L::FUSED;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* const stages = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* const xs = stages + STAGES * L::STAGE_BYTES;                                                  // (FUSED) x's blocks
  unsigned long long* const full = reinterpret_cast<unsigned long long*>(xs + L::X_BLOCKS * L::X_BYTES);       // [S] copies -> products
  unsigned long long* const empty = full + STAGES;                                                             // [S] products -> copies
  unsigned long long* const acc_full = empty + STAGES;                                                         // [2] a tile's sums -> their readers
  unsigned long long* const acc_empty = acc_full + 2;                                                          // [2] read (by every reader) -> products
  unsigned long long* const x_full = acc_empty + 2;                                                            // (FUSED) x is rounded (by every rounder) -> products
  unsigned* const tmem_slot = reinterpret_cast<unsigned*>(x_full + 1);
  __shared__ int failed_s, issued_s;
  __shared__ unsigned long long drained_s, sums_s;   // sums_s: (SPLIT) what the cluster's blocks send this one has come
  __shared__ Most most_s;
  volatile int* const failed = &failed_s;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, KB = p.blocks;
  const int x_tiles = (p.m + NB - 1) / NB, tiles = (p.n + ROWS - 1) / ROWS * x_tiles;   // those of one W row range are behind one another: W crosses memory once
  // this block's tiles, and its share of their inputs
  const unsigned rank = SPLIT ? cluster_rank() : 0, size = SPLIT ? cluster_size() : 1;
  const int first_tile = blockIdx.x / size, step = SPLIT ? tiles : gridDim.x, k0 = SPLIT ? KB * rank / size : 0, k1 = SPLIT ? KB * (rank + 1) / size : KB;

  // (SPLIT) columns that the blocks of a cluster have in turn
  constexpr int GROUP = 4, GROUPS = NB / GROUP;
  // columns of a tile that has so many rows of x left: whole sixteens
  auto columns = [](int left) { return left >= NB ? NB : (left + 15) / 16 * 16; };

  if (threadIdx.x == 0) {
    failed_s = issued_s = 0;
    mbar_init(&drained_s, 1);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], READ_THREADS);
    }
    if (SPLIT) mbar_init(&sums_s, 1);
    if (FUSED) mbar_init(x_full, L::ROUNDERS * 32);
    if (FUSED && SPLIT && KIND == NV) mbar_init(&most_s.full, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (FUSED && threadIdx.x < FUSED_ROWS) most_s.rows[threadIdx.x] = 0;
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(L::TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if constexpr (FUSED && SPLIT && KIND == NV) {   // the others' barriers are there before anything is sent to them
    if (threadIdx.x == 0) mbar_expect_tx(&most_s.full, size * FUSED_ROWS * 4);
    __syncwarp();
    cluster_sync();
  }
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const unsigned tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  let_next_launch_in();

  if (warp == 0) {
    const bool issues = elected();
    auto w_of = [&](int t) { return p.w + ((size_t)(t / x_tiles) * KB + k0) * F::BLOCK_BYTES; };
    auto x_bytes_of = [&](int t) { return FUSED ? 0 : F::SCALE_BYTES + columns(p.m - t % x_tiles * NB) * (INPUTS / 2); };   // scales, and codes of the rows that there are
    auto load_w = [&](int t, int kb, int s) {
      mbar_expect_tx(&full[s], F::BLOCK_BYTES + x_bytes_of(t));
      bulk_load(stages + (size_t)s * L::STAGE_BYTES, w_of(t) + (size_t)(kb - k0) * F::BLOCK_BYTES, F::BLOCK_BYTES, &full[s]);
    };
    // W depends on no launch that may still be running: as much of it as fits is asked for at once
    const int early = first_tile < tiles ? min(STAGES, k1 - k0) : 0;
    if (issues)
      for (int s = 0; s < early; ++s) load_w(first_tile, k0 + s, s);
    __syncwarp();
    if (!FUSED) asm volatile("griddepcontrol.wait;" ::: "memory");
    int i = 0, s = 0;
    unsigned par = 1;   // (the first turn finds every stage free)
    bool ok = true;
    for (int t = first_tile; ok && t < tiles; t += step) {
      const unsigned char* x = p.x + ((size_t)(t % x_tiles) * KB + k0) * F::BLOCK_BYTES;
      const unsigned x_bytes = x_bytes_of(t);
      for (int kb = k0; kb < k1; ++kb, ++i, x += F::BLOCK_BYTES) {
        ok = i < STAGES || __all_sync(0xffffffffu, mbar_wait(&empty[s], par, p.err, failed, 1));
        if (!ok) break;
        if (issues) {
          if (i >= early) load_w(t, kb, s);
          if (!FUSED) bulk_load(stages + (size_t)s * L::STAGE_BYTES + F::BLOCK_BYTES, x, x_bytes, &full[s]);
        }
        __syncwarp();
        if (++s == STAGES) {
          s = 0;
          par ^= 1;
        }
      }
    }
    if (lane == 0) issued_s = i;
  } else if (warp == 1) {
    const bool issues = elected();
    int s = 0, run = 0;
    unsigned par = 0, buffer = 0;
    // stages that this block's products take
    long long left = SPLIT ? k1 - k0 : first_tile < tiles ? (long long)((unsigned)(tiles - first_tile - 1) / (unsigned)step + 1) * (k1 - k0) : 0;
    bool ok = !FUSED || __all_sync(0xffffffffu, mbar_wait(x_full, 0, p.err, failed, 3));
    for (int t = first_tile; ok && t < tiles; t += step, ++run) {
      const int acc = run % L::ACCS;
      const unsigned d = tmem + acc * NB, n_bits = (unsigned)(columns(p.m - t % x_tiles * NB) >> 3) << 17;
      ok = run < L::ACCS || __all_sync(0xffffffffu, mbar_wait(&acc_empty[acc], (unsigned)((run / L::ACCS - 1) & 1), p.err, failed, 4));
      for (int kb = k0; ok && kb < k1; ++kb) {
        ok = __all_sync(0xffffffffu, mbar_wait(&full[s], par, p.err, failed, 2));
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (issues) {
          unsigned char* const at = stages + (size_t)s * L::STAGE_BYTES;
          const unsigned sw = tmem + L::ACCS * NB + buffer * L::SCALE_COLS, sx = sw + 4 * F::WORDS;
          const unsigned char* const x_at = FUSED ? xs + (size_t)(kb - k0) * L::X_BYTES : at + F::BLOCK_BYTES;
          const unsigned long long w_scales = scales_desc(at), x_scales = scales_desc(x_at);
          const unsigned long long w = codes_desc(at + F::SCALE_BYTES), x = codes_desc(x_at + F::SCALE_BYTES);
#pragma unroll
          for (int j = 0; j < F::WORDS; ++j) {
            scales_to_tmem(sw + 4 * j, w_scales + j * (512 >> 4));
            scales_to_tmem(sx + 4 * j, x_scales + j * (512 >> 4));
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int word = j * F::WORDS / 4;
            umma<KIND>(d, w + 2 * j, x + 2 * j, idesc<KIND>(KIND == MX ? 2 * (j & 1) : 0) | n_bits, sw + 4 * word, sx + 4 * word, kb > k0 || j > 0);
          }
          if (left > STAGES) umma_commit(&empty[s]);   // (where a copy waits for it: nothing is on its way to a block that may have ended)
          if (kb == k1 - 1) umma_commit(&acc_full[acc]);
        }
        --left;
        __syncwarp();
        buffer ^= 1;
        if (++s == STAGES) {
          s = 0;
          par ^= 1;
        }
      }
    }
  } else {
    const int q = warp & 3;                              // the quarter of tensor memory that this warp may read
    constexpr int COLS = NB / L::PARTS;                  // columns that this warp reads, from `first` on
    const int first = (warp - 2) / 4 * COLS;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if constexpr (FUSED) round_x<L, KIND, SRC, SPLIT>(p, k0, k1, xs, most_s, x_full, rank, size, failed);
    int run = 0;
    for (int t = warp < 2 + L::READERS ? first_tile : tiles; t < tiles; t += step, ++run) {
      const int acc = run % L::ACCS, row = t / x_tiles * ROWS + q * 32 + lane, col0 = t % x_tiles * NB + first, cols = min(COLS, p.m - col0);   // cols: may be none
      const float own = KIND == NV && row < p.n ? __ldg(p.w_factors + row) : 1.f;
      float x_factor[(COLS + 31) / 32];   // of the columns, a lane each (asked for here, where there is time)
      if constexpr (KIND == NV)
#pragma unroll
        for (int c = 0; c < (COLS + 31) / 32; ++c)
          x_factor[c] = 32 * c + lane >= cols ? 1.f : FUSED ? row_factor(most_s.rows[col0 + 32 * c + lane]) : ld_prev(p.x_factors + col0 + 32 * c + lane);
      const RowFactor steps = in_steps<KIND>(own);   // (here: the products take longer than the factor)
      if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[acc], (unsigned)(run / L::ACCS & 1), p.err, failed, 5))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if constexpr (SPLIT) break;   // (below)
      // into registers all at once, so that the next tile's products may begin
      const unsigned from = tmem + ((unsigned)(q * 32) << 16) + acc * NB + first;
      float v[COLS / 16][16];
#pragma unroll
      for (int c = 0; c < COLS / 16; ++c)
        if (16 * c < cols) tmem_ld16(from + 16 * c, v[c]);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      mbar_arrive(&acc_empty[acc]);
      write_columns<KIND, COLS>(p, reinterpret_cast<O*>(p.y) + (size_t)col0 * p.n + row, row < p.n, cols, v, steps, x_factor);
      __syncwarp();
    }
  }

  if constexpr (SPLIT) {
    // Columns go to the cluster's blocks in turn, GROUP at a time: every block sends the others its sums, into what were the stages ([block][group][row][4], by asynchronous stores), and adds up what it
    // was sent, in the order of the inputs.  All threads come by here, whatever their waits came to; what is sent when one gave up is nobody's result.
    const unsigned per_block = (GROUPS + size - 1) / size;
    const int q = warp & 3, part = (warp - 2) / 4;
    const int row = first_tile / x_tiles * ROWS + q * 32 + lane, col0 = first_tile % x_tiles * NB, cols = min(NB, p.m - col0);
    const bool reads = warp >= 2 && warp < 2 + L::READERS;
    const float own = KIND == NV && reads && row < p.n ? __ldg(p.w_factors + row) : 1.f;
    float x_factor[(NB + 31) / 32];
    if constexpr (KIND == NV)
#pragma unroll
      for (int c = 0; c < (NB + 31) / 32; ++c)
        x_factor[c] = !reads || 32 * c + lane >= cols ? 1.f : FUSED ? row_factor(most_s.rows[col0 + 32 * c + lane]) : ld_prev(p.x_factors + col0 + 32 * c + lane);
    auto place = [&](unsigned block, unsigned group) { return (unsigned)(((block * per_block + group) * GROUP / 4 * ROWS + q * 32 + lane) * 16); };
    __syncwarp();
    if (threadIdx.x == 64) {   // groups rank, rank + size, ... of those that have results, from every block
      const unsigned groups = (cols + GROUP - 1) / GROUP, mine = groups > rank ? (groups - rank + size - 1) / size : 0;
      mbar_expect_tx(&sums_s, mine * size * GROUP * ROWS * 4);
    }
    __syncwarp();
    cluster_sync();   // every block's products have ended, so its stages are free
    if (reads) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const unsigned from = tmem + ((unsigned)(q * 32) << 16);
#pragma unroll 1
      for (int c = part * (NB / L::PARTS); c < min(cols, (part + 1) * (NB / L::PARTS)); c += 16) {
        float v[16];
        tmem_ld16(from + c, v);
#pragma unroll
        for (int j = 0; j < 16; j += 4)
          if (c + j < cols) {
            const unsigned g = (c + j) / GROUP;
            send(smem_u32(stages) + place(rank, g / size), smem_u32(&sums_s), g % size, v[j], v[j + 1], v[j + 2], v[j + 3]);
          }
      }
    }
    const RowFactor steps = in_steps<KIND>(own);
    if (reads) mbar_wait<true>(&sums_s, 0, p.err, failed, 7);
    __syncwarp();
    cluster_arrive();   // (a block whose shared memory others may still send to does not end: below)
    if (reads) {
#pragma unroll 1
      for (unsigned i = part; (rank + size * i) * GROUP < cols; i += L::PARTS) {
        const int c = (rank + size * i) * GROUP;
        float v[GROUP];
#pragma unroll
        for (int j = 0; j < GROUP; ++j) v[j] = 0.f;
#pragma unroll 4
        for (unsigned b = 0; b < size; ++b)
#pragma unroll
          for (int j = 0; j < GROUP; j += 4) {
            const float4 t = *reinterpret_cast<const float4*>(stages + place(b, i));
            v[j] += t.x;
            v[j + 1] += t.y;
            v[j + 2] += t.z;
            v[j + 3] += t.w;
          }
        if (KIND == NV) {
          float f = x_factor[0];
#pragma unroll
          for (int h = 1; h < (NB + 31) / 32; ++h)
            if (c >= 32 * h) f = x_factor[h];
#pragma unroll
          for (int j = 0; j < GROUP; ++j) v[j] = v[j] * steps.of * __shfl_sync(0xffffffffu, f, (c + j) % 32);
          if (steps.far)
#pragma unroll
            for (int j = 0; j < GROUP; ++j) v[j] *= steps.rest;
        }
        if (row < p.n)
#pragma unroll
          for (int j = 0; j < GROUP; ++j)
            if (c + j < cols) reinterpret_cast<O*>(p.y)[(size_t)(col0 + c + j) * p.n + row] = from_f32<O>(v[j]);
      }
    }
    __syncwarp();
    cluster_wait();
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*failed) {
    // a wait ran out: give copies and products that may still be in flight a bounded time to end
    const long long t0 = clock64();
    auto expired = [&] { return clock64() - t0 > WAIT_CYCLES; };
    if (threadIdx.x == 0) ring_drain(issued_s, STAGES, [&](int s, unsigned parity) { return mbar_try_wait(&full[s], parity); }, expired);
    if (warp == 1 && elected()) {   // the thread that issued the products
      umma_commit(&drained_s);
      while (!mbar_try_wait(&drained_s, 0) && !expired()) {}
    }
    __syncthreads();
  }
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::TMEM_COLS) : "memory");
  }
}

// The same for many rows of x: two blocks on neighbouring multiprocessors have a tile of 256 rows of W (128 each) against `nb` rows of x, of which each holds half: a product's
// operands then cross from L2 for twice the work (38 KB of a stage a block instead of 54: tiles of 256 columns by one block took 95 us where pairs take 83).  The first block issues the products of
// both.  The second one's copies complete barriers of its own; its warp 1 passes that on.
template <int KIND> struct PairLayout {
  typedef Format<KIND> F;
  static constexpr int MOST_NB = 256, PARTS = 4, READERS = 4 * PARTS, THREADS = (2 + READERS) * 32, COLS = MOST_NB / PARTS;
  static constexpr int X_AT = F::BLOCK_BYTES + 2 * F::SCALE_BYTES, STAGE_BYTES = X_AT + MOST_NB / 2 * (INPUTS / 2);   // W's block, x's scales (all of the tile's), half of x's codes
  static constexpr int STAGES = 225 * 1024 / STAGE_BYTES;
  static constexpr int SCALE_COLS = 4 * F::WORDS * 3, TMEM_COLS = 512;
  static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + 8 * (3 * STAGES + 4) + 16;
  // tensor memory: sums of two tiles of up to 192 columns, so that a tile's products need not wait until the sums before it are read, or of one of 256; then the scales of two stages
  static constexpr int TWO_NB = 192;
  static_assert(2 * TWO_NB + 2 * SCALE_COLS <= TMEM_COLS, "of tensor memory");
  static_assert(MOST_NB + 2 * SCALE_COLS <= TMEM_COLS && SMEM_BYTES <= 227 * 1024 && STAGE_BYTES % 1024 == 0, "of a block");
};
__device__ __forceinline__ void mbar_arrive_at(void* bar, unsigned rank) {   // of a block of the cluster
  asm volatile("{ .reg .u32 a; mapa.shared::cluster.u32 a, %0, %1; mbarrier.arrive.shared::cluster.b64 _, [a]; }" ::"r"(smem_u32(bar)), "r"(rank) : "memory");
}
__device__ __forceinline__ void umma_commit_both(void* bar) {   // in both blocks
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((unsigned short)3) : "memory");
}

template <int KIND, typename O> __global__ void __launch_bounds__(PairLayout<KIND>::THREADS, 1) linear_fp4_pair_kernel(const Params p, int nb) {
  typedef PairLayout<KIND> L;
  typedef typename L::F F;
  constexpr int STAGES = L::STAGES;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* const stages = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned long long* const full = reinterpret_cast<unsigned long long*>(stages + STAGES * L::STAGE_BYTES);   // [S] this block's copies
  unsigned long long* const peer_full = full + STAGES;                                                         // [S] (of the first block) the other's copies
  unsigned long long* const empty = peer_full + STAGES;                                                        // [S] products -> copies
  unsigned long long* const acc_full = empty + STAGES;                                                         // [2] a tile's sums -> their readers
  unsigned long long* const acc_empty = acc_full + 2;                                                          // [2] (of the first block) read, by every reading warp of both
  unsigned* const tmem_slot = reinterpret_cast<unsigned*>(acc_empty + 2);
  const int accs = nb <= L::TWO_NB ? 2 : 1, acc_cols = nb <= L::TWO_NB ? L::TWO_NB : L::MOST_NB;
  __shared__ int failed_s, issued_s;
  __shared__ unsigned long long drained_s;
  volatile int* const failed = &failed_s;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, KB = p.blocks;
  const unsigned rank = cluster_rank();
  // whole tiles first, those of one W row range behind one another; then the last, shorter ones
  const int w_blocks = (p.n + ROWS - 1) / ROWS, w_tiles = (w_blocks + 1) / 2, whole = p.m / nb, tiles = w_tiles * ((p.m + nb - 1) / nb);
  struct Tile { int w, x0, cols; };
  auto tile_of = [&](int t) {
    const bool short_one = t >= w_tiles * whole;
    Tile r;
    r.w = (short_one ? t - w_tiles * whole : t / whole) * 2;                      // the first of its blocks of W
    r.x0 = (short_one ? whole : t % whole) * nb;                                  // its first row of x
    r.cols = short_one ? (p.m - r.x0 + 31) / 32 * 32 : nb;                          // columns: each block has half of them, whole sixteens
    return r;
  };
  const int first_tile = blockIdx.x / 2, step = gridDim.x / 2;

  if (threadIdx.x == 0) {
    failed_s = issued_s = 0;
    mbar_init(&drained_s, 1);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&peer_full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * L::READERS);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(L::TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();   // both have their barriers and their tensor memory
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const unsigned tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  let_next_launch_in();

  if (warp == 0) {
    const bool issues = elected();
    // of the two blocks of x that a tile's rows are in: rows from..to are this block's half
    struct Half { int from, to; unsigned head, tail; bool second; };   // bytes in either; whether the tile has rows in the second
    auto half_of = [&](const Tile& at) {
      Half h;
      h.from = at.x0 % ROWS + (int)rank * (at.cols / 2);
      h.to = h.from + at.cols / 2;
      h.head = h.from < ROWS ? (min(h.to, ROWS) - h.from) * (INPUTS / 2) : 0;
      h.tail = h.to > ROWS ? (h.to - max(h.from, ROWS)) * (INPUTS / 2) : 0;
      h.second = at.x0 % ROWS + at.cols > ROWS;
      return h;
    };
    auto load_w = [&](const Tile& at, const Half& h, int kb, int s) {
      mbar_expect_tx(&full[s], F::BLOCK_BYTES + (h.second ? 2 : 1) * F::SCALE_BYTES + h.head + h.tail);
      // (an odd number of blocks of W: the last one again, for rows that are nobody's)
      bulk_load(stages + (size_t)s * L::STAGE_BYTES, p.w + ((size_t)min(at.w + (int)rank, w_blocks - 1) * KB + kb) * F::BLOCK_BYTES, F::BLOCK_BYTES, &full[s]);
    };
    // W depends on no launch that may still be running: as much of it as fits is asked for at once
    const int early = first_tile < tiles ? min(STAGES, KB) : 0;
    if (issues && early) {
      const Tile at = tile_of(first_tile);
      const Half h = half_of(at);
      for (int s = 0; s < early; ++s) load_w(at, h, s, s);
    }
    __syncwarp();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int i = 0, s = 0;
    unsigned par = 1;   // (the first turn finds every stage free)
    bool ok = true;
    for (int t = first_tile; ok && t < tiles; t += step) {
      const Tile at = tile_of(t);
      const Half h = half_of(at);
      const unsigned char* x = p.x + (size_t)(at.x0 / ROWS) * KB * F::BLOCK_BYTES;
      for (int kb = 0; kb < KB; ++kb, ++i, x += F::BLOCK_BYTES) {
        ok = i < STAGES || __all_sync(0xffffffffu, mbar_wait(&empty[s], par, p.err, failed, 11));
        if (!ok) break;
        if (issues) {
          unsigned char* const stage = stages + (size_t)s * L::STAGE_BYTES;
          const unsigned char* const next = x + (size_t)KB * F::BLOCK_BYTES;
          if (i >= early) load_w(at, h, kb, s);
          bulk_load(stage + F::BLOCK_BYTES, x, F::SCALE_BYTES, &full[s]);
          if (h.second) bulk_load(stage + F::BLOCK_BYTES + F::SCALE_BYTES, next, F::SCALE_BYTES, &full[s]);
          if (h.head) bulk_load(stage + L::X_AT, x + F::SCALE_BYTES + h.from * (INPUTS / 2), h.head, &full[s]);
          if (h.tail) bulk_load(stage + L::X_AT + h.head, next + F::SCALE_BYTES + (max(h.from, ROWS) - ROWS) * (INPUTS / 2), h.tail, &full[s]);
        }
        __syncwarp();
        if (++s == STAGES) {
          s = 0;
          par ^= 1;
        }
      }
    }
    if (lane == 0) issued_s = i;
  } else if (warp == 1 && rank == 1) {
    int s = 0;
    unsigned par = 0;
    bool ok = true;
    for (int t = first_tile; ok && t < tiles; t += step)
      for (int kb = 0; kb < KB; ++kb) {
        ok = __all_sync(0xffffffffu, mbar_wait(&full[s], par, p.err, failed, 12));
        if (!ok) break;
        if (lane == 0) mbar_arrive_at(&peer_full[s], 0);
        if (++s == STAGES) {
          s = 0;
          par ^= 1;
        }
      }
  } else if (warp == 1) {
    const bool issues = elected();
    int s = 0, run = 0;
    unsigned par = 0, buffer = 0;
    long long left = first_tile < tiles ? (long long)((unsigned)(tiles - first_tile - 1) / (unsigned)step + 1) * KB : 0;   // stages that this pair's products take
    bool ok = true;
    for (int t = first_tile; ok && t < tiles; t += step, ++run) {
      const Tile at = tile_of(t);
      const unsigned n_bits = (unsigned)(at.cols >> 3) << 17, shift = at.x0 % ROWS / 32;   // shift: columns of scales in front of the tile's
      const int acc = run % accs;
      const unsigned d = tmem + acc * acc_cols;
      ok = run < accs || __all_sync(0xffffffffu, mbar_wait<true>(&acc_empty[acc], (unsigned)((run / accs - 1) & 1), p.err, failed, 14));
      for (int kb = 0; ok && kb < KB; ++kb) {
        ok = __all_sync(0xffffffffu, mbar_wait(&full[s], par, p.err, failed, 12) && mbar_wait<true>(&peer_full[s], par, p.err, failed, 13));
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (issues) {
          unsigned char* const stage = stages + (size_t)s * L::STAGE_BYTES;
          const unsigned sw = tmem + accs * acc_cols + buffer * L::SCALE_COLS, sx = sw + 4 * F::WORDS;
          const unsigned long long w_scales = scales_desc(stage), x_scales = scales_desc(stage + F::BLOCK_BYTES);
          const unsigned long long w = codes_desc(stage + F::SCALE_BYTES), x = codes_desc(stage + L::X_AT);
#pragma unroll
          for (int j = 0; j < F::WORDS; ++j) {
            scales_to_tmem<2>(sw + 4 * j, w_scales + j * (512 >> 4));
#pragma unroll
            for (int h = 0; h < 2; ++h) scales_to_tmem<2>(sx + 8 * j + 4 * h, x_scales + ((j * 512 + h * F::SCALE_BYTES) >> 4));
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int word = j * F::WORDS / 4;
            umma<KIND, 2>(d, w + 2 * j, x + 2 * j, idesc<KIND, 256>(KIND == MX ? 2 * (j & 1) : 0) | n_bits, sw + 4 * word, sx + 8 * word + shift, kb > 0 || j > 0);
          }
          if (left > STAGES) umma_commit_both(&empty[s]);   // (as above)
          if (kb == KB - 1) umma_commit_both(&acc_full[acc]);
        }
        --left;
        __syncwarp();
        buffer ^= 1;
        if (++s == STAGES) {
          s = 0;
          par ^= 1;
        }
      }
    }
  } else {
    const int q = warp & 3, first = (warp - 2) / 4 * L::COLS;   // q: the quarter of tensor memory that this warp may read; first: its first column
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int run = 0;
    for (int t = first_tile; t < tiles; t += step, ++run) {
      const Tile at = tile_of(t);
      const int row = (at.w + (int)rank) * ROWS + q * 32 + lane, col0 = at.x0 + first, cols = min(min(L::COLS, at.cols - first), p.m - col0);   // cols: may be none
      const float own = KIND == NV && row < p.n ? __ldg(p.w_factors + row) : 1.f;
      float x_factor[L::COLS / 32];
      if constexpr (KIND == NV)
#pragma unroll
        for (int c = 0; c < L::COLS / 32; ++c) x_factor[c] = 32 * c + lane < cols ? ld_prev(p.x_factors + col0 + 32 * c + lane) : 1.f;
      const int acc = run % accs;
      const RowFactor steps = in_steps<KIND>(own);   // (as above)
      if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[acc], (unsigned)(run / accs & 1), p.err, failed, 15))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const unsigned from = tmem + ((unsigned)(q * 32) << 16) + acc * acc_cols + first;
      float v[L::COLS / 16][16];
#pragma unroll
      for (int c = 0; c < L::COLS / 16; ++c)
        if (16 * c < cols) tmem_ld16(from + 16 * c, v[c]);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0 && t + accs * step < tiles) mbar_arrive_at(&acc_empty[acc], 0);   // (where products wait for it: nothing is on its way to a block that may have ended)
      write_columns<KIND, L::COLS>(p, reinterpret_cast<O*>(p.y) + (size_t)col0 * p.n + row, row < p.n, cols, v, steps, x_factor);
      __syncwarp();
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*failed) {
    // a wait ran out: give copies and products that may still be in flight a bounded time to end
    const long long t0 = clock64();
    auto expired = [&] { return clock64() - t0 > WAIT_CYCLES; };
    if (threadIdx.x == 0) ring_drain(issued_s, STAGES, [&](int s, unsigned parity) { return mbar_try_wait(&full[s], parity); }, expired);
    if (warp == 1 && rank == 0 && elected()) {   // the thread that issued the products
      asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(&drained_s)) : "memory");
      while (!mbar_try_wait(&drained_s, 0) && !expired()) {}
    }
    __syncthreads();
  }
  __syncwarp();
  cluster_sync();   // neither's memory goes before the other is done with it
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::TMEM_COLS) : "memory");
  }
}

template <int KIND, int NB, bool SPLIT, int SRC, typename O> int configured(cudaLaunchConfig_t& cfg, cudaLaunchAttribute (&attr)[2], int blocks, int split, bool dependent, cudaStream_t st) {
  typedef Layout<KIND, NB, SPLIT, SRC> L;
  static bool asked[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return DRYFT_ERR_UNSUPPORTED;
  if (!asked[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(linear_fp4_kernel<KIND, NB, SPLIT, SRC, O>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM_BYTES);
    if (e != cudaSuccess) return (int)e;
    asked[dev] = true;
  }
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(L::THREADS);
  cfg.dynamicSmemBytes = L::SMEM_BYTES;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 0;
  if (dependent) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (SPLIT) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = split;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  return 0;
}
template <int KIND, int NB, bool SPLIT, int SRC, typename O> int run(const Params& p, int blocks, int split, bool dependent, cudaStream_t st) {
  typedef Layout<KIND, NB, SPLIT, SRC> L;
  const long long tiles = ((long long)p.n + ROWS - 1) / ROWS * ((p.m + NB - 1) / NB);
  if (NB < ROWS && p.m > NB) return DRYFT_ERR_UNSUPPORTED;   // (a block of x is 128 rows: only tiles of as many follow one another)
  if (tiles * MOST_BLOCKS > 0x7fffffffll || blocks <= 0 || (SPLIT ? blocks != tiles * split : blocks > tiles)) return DRYFT_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  const int rc = configured<KIND, NB, SPLIT, SRC, O>(cfg, attr, blocks, split, dependent, st);
  if (rc) return rc;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, linear_fp4_kernel<KIND, NB, SPLIT, SRC, O>, p);
  return e != cudaSuccess ? (int)e : launch_status();
}
template <int KIND, typename O> int run_pairs(const Params& p, int nb, int blocks, bool dependent, cudaStream_t st) {
  typedef PairLayout<KIND> L;
  if (nb != 128 && nb != 192 && nb != 256) return DRYFT_ERR_UNSUPPORTED;   // (rows of x of a tile begin at whole or half blocks, and lie in two at most)
  const long long tiles = ((long long)p.n + 2 * ROWS - 1) / (2 * ROWS) * ((p.m + nb - 1) / nb);
  if (tiles > 0x3fffffffll || blocks <= 0 || blocks % 2 || blocks > 2 * tiles) return DRYFT_ERR_UNSUPPORTED;
  auto kern = linear_fp4_pair_kernel<KIND, O>;
  static bool asked[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return DRYFT_ERR_UNSUPPORTED;
  if (!asked[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM_BYTES);
    if (e != cudaSuccess) return (int)e;
    asked[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(L::THREADS);
  cfg.dynamicSmemBytes = L::SMEM_BYTES;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 2 : 1;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p, nb);
  return e != cudaSuccess ? (int)e : launch_status();
}
template <int KIND, bool SPLIT, typename O> int by_rows(const Params& p, int nb, int blocks, int split, bool dependent, cudaStream_t st) {
  switch (nb) {
    case 16: return run<KIND, 16, SPLIT, HELD, O>(p, blocks, split, dependent, st);
    case 32: return run<KIND, 32, SPLIT, HELD, O>(p, blocks, split, dependent, st);
    case 64: return run<KIND, 64, SPLIT, HELD, O>(p, blocks, split, dependent, st);
    case 128: return run<KIND, 128, SPLIT, HELD, O>(p, blocks, split, dependent, st);
  }
  return DRYFT_ERR_UNSUPPORTED;
}
template <int KIND, typename O> int by_split(const Params& p, int nb, int blocks, int split, bool dependent, cudaStream_t st) {
  if (split == 0) return run_pairs<KIND, O>(p, nb, blocks, dependent, st);
  return split > 1 ? by_rows<KIND, true, O>(p, nb, blocks, split, dependent, st) : by_rows<KIND, false, O>(p, nb, blocks, split, dependent, st);
}
template <int KIND, typename O> int by_source(const Params& p, bool is_bf16, bool silu, int blocks, int split, bool dependent, cudaStream_t st) {
  if (!is_bf16) {
    if constexpr (sizeof(O) == 4)
      return split > 1 ? run<KIND, FUSED_ROWS, true, F32, O>(p, blocks, split, dependent, st) : run<KIND, FUSED_ROWS, false, F32, O>(p, blocks, split, dependent, st);
    return DRYFT_ERR_UNSUPPORTED;
  }
  if (!silu) return split > 1 ? run<KIND, FUSED_ROWS, true, BF16, O>(p, blocks, split, dependent, st) : run<KIND, FUSED_ROWS, false, BF16, O>(p, blocks, split, dependent, st);
  if constexpr (sizeof(O) == 2)
    return split > 1 ? run<KIND, FUSED_ROWS, true, SILU, O>(p, blocks, split, dependent, st) : run<KIND, FUSED_ROWS, false, SILU, O>(p, blocks, split, dependent, st);
  return DRYFT_ERR_UNSUPPORTED;
}
template <int KIND, int NB> int clusters_of(int split) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (configured<KIND, NB, true, HELD, bf16>(cfg, attr, split, split, false, nullptr)) return 0;
  return cudaOccupancyMaxActiveClusters(&n, linear_fp4_kernel<KIND, NB, true, HELD, bf16>, &cfg) == cudaSuccess ? n : 0;
}
}  // namespace

extern "C" int dryft_fp4_quantise(int is_bf16, int kind, int silu, const void* x, long long stride, void* held, void* factors, int rows, int k, int pdl, void* stream);

// How many clusters of `split` blocks are resident at a time.
DRYFT_API int dryft_linear_fp4_clusters(int nb, int split) {
  if (split < 2 || split > MOST_BLOCKS) return 0;
  switch (nb) {
    case 16: return clusters_of<NV, 16>(split);
    case 32: return clusters_of<NV, 32>(split);
    case 64: return clusters_of<NV, 64>(split);
    case 128: return clusters_of<NV, 128>(split);
  }
  return 0;
}

// y [m, n] = x w^T; x, w: blocks of 128 rows by 256 inputs (fp4.cuh) with factors for each row (NV); y bfloat16 or float32.  nb: x rows of a tile, 16 to 128 (against 128
// rows of W).  split: blocks that share a tile's inputs, as a cluster (1: none do, and `blocks` walk the tiles; 0: pairs of
// blocks walk tiles of 256 rows of W by nb = 128, 192 or 256 of x).
DRYFT_API int dryft_linear_fp4(int kind, int out_bf16, const void* x, const void* x_factors, const void* w, const void* w_factors, void* y, int m, int n, int k, int nb,
                               int blocks, int split, int pdl, int* err, void* stream) {
  if (m <= 0 || n <= 0) return 0;
  if (k <= 0 || split < 0 || split > MOST_BLOCKS || split > blocks_of(k)) return DRYFT_ERR_UNSUPPORTED;
  const Params p = {(const unsigned char*)x, (const unsigned char*)w, (const float*)x_factors, (const float*)w_factors, y, err, m, n, blocks_of(k), k, 0, false};
  const cudaStream_t st = (cudaStream_t)stream;
  if (kind == NV) return out_bf16 ? by_split<NV, bf16>(p, nb, blocks, split, pdl, st) : by_split<NV, float>(p, nb, blocks, split, pdl, st);
  return out_bf16 ? by_split<MX, bf16>(p, nb, blocks, split, pdl, st) : by_split<MX, float>(p, nb, blocks, split, pdl, st);
}

// The same of x as it is: `stride` numbers between its rows (silu: of 2 k numbers, as for dryft_fp4_quantise).  scratch: its form in 4 bits, then (NV) its rows' factors, `factors_at` bytes on.  pdl: 1, the rounding is a programmatic
// dependent of the launch before it; 2, the product is one of the rounding.  scratch null: one launch, every block of which rounds x for itself (up to 16 rows, nb = 16, up to 12 blocks
// of 256 inputs a block; bfloat16, with silu to bfloat16 results, or 32-bit numbers without, to 32-bit results).
DRYFT_API int dryft_linear_fp4_rows(int kind, int is_bf16, int silu, int out_bf16, const void* x, long long stride, const void* w, const void* w_factors, void* y, int m, int n, int k,
                                    int nb, int blocks, int split, unsigned char* scratch, long long factors_at, int pdl, int* err, void* stream) {
  if (m <= 0 || n <= 0) return 0;
  if (!scratch) {   // rounded by the product's own blocks
    const int kb = blocks_of(k);
    if ((!is_bf16 && (silu || out_bf16)) || m > FUSED_ROWS || nb != FUSED_ROWS || split < 1 || split > MOST_BLOCKS || split > kb || (kb + split - 1) / split > FUSED_BLOCKS || (silu && !out_bf16))
      return DRYFT_ERR_UNSUPPORTED;
    const Params p = {(const unsigned char*)x, (const unsigned char*)w, nullptr, (const float*)w_factors, y, err, m, n, kb, k, stride,
                      ((uintptr_t)x & 15) == 0 && (m == 1 || stride * (is_bf16 ? 2 : 4) % 16 == 0) && (!silu || k % 8 == 0)};
    const cudaStream_t st = (cudaStream_t)stream;
    const bool ahead = pdl & 1;
    if (kind == NV) return out_bf16 ? by_source<NV, bf16>(p, is_bf16, silu, blocks, split, ahead, st) : by_source<NV, float>(p, is_bf16, silu, blocks, split, ahead, st);
    return out_bf16 ? by_source<MX, bf16>(p, is_bf16, silu, blocks, split, ahead, st) : by_source<MX, float>(p, is_bf16, silu, blocks, split, ahead, st);
  }
  const int rc = dryft_fp4_quantise(is_bf16, kind, silu, x, stride, scratch, scratch + factors_at, m, k, pdl, stream);
  if (rc) return rc;
  return dryft_linear_fp4(kind, out_bf16, scratch, scratch + factors_at, w, w_factors, y, m, n, k, nb, blocks, split, pdl & 2, err, stream);
}
