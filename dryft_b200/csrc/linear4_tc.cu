// Products with weights held in 4 bits (four_bit.cuh, linear4.cu has their layout) for up to 256 rows of bfloat16, on the 5th-generation tensor cores.
//
// Computed transposed: a tile is 128 rows of W against all rows of x, padded to NB = 32, 64, 128 or 256, its 128 x NB sums in tensor memory.  A unit is
// 128 inputs of a tile (64 with 256 rows of x): its codes (8 KB) and scales come by TMA into a ring of eight, a team of warps takes them out of their 4 bits, 16 rows
// of W a warp at a time, and stores them into tensor memory, where tcgen05.mma takes its first operand from: a lane's codes are rows r and r + 8 and the inputs of two
// neighbouring columns, which is the shape 16x256b as it stands.  x comes by TMA, K-major in a 128-byte swizzle.  So the weights cross memory at 4.5 bits
// and are multiplied as bfloat16 z + (c - 7.5) s: one rounding, by up to 2^-8, of each weight (2^-9.2 in the mean square).  For 32-bit results (LOW)
// the rest of that rounding is a second operand with a product of its own, which leaves 2^-16 (2^-18), and inputs are summed 512 at a time (`SEGMENT`): in one piece
// 30,000 outputs of 12,288 inputs were off by 22 millionths of the whole, now by 0.9; 32-bit multiply-adds in order are by 1.9.  That takes 128 rows at most; more are two passes.
//
// Work is cut evenly: block i of G takes the units [i U / G, (i + 1) U / G) in (tile, inputs) order.  A run that covers its tile's inputs is finished from tensor
// memory; else its sums go to a workspace, and a second launch adds a tile's pieces in the blocks' order.  No block waits for another.
//
// What bounds it: every tile reads all of x again, from L2, which moves 9 TB/s at 48 rows (issue slots are used at 64% beside it, the tensor cores at 32%) and 10 at 256
// rows (41 and 57%).  48 rows: 2,560 outputs of 9,728 inputs 12.6 us (of which some 3 us the launch and 3 us the join), 19,456 of 2,560 16.8 us, 151,936 of 2,560 78 us
// (32-bit results 188: two products and twice the taking out); 128 and 256 rows, 19,456 of 2,560: 24 and 39 us.
// (Steps on the way, 48 rows, 19,456 of 2,560: weights written into shared memory as the operand 22 us; into tensor memory 21.4, by then bound by the one thread that
// issued products, 500 cycles a unit to put their operands into uniform registers; with a whole warp that walks the loop 17.5; one barrier for weights and x, asked
// ahead of the products before, 16.7.)
//
// Warps: 0 copies x, 1 issues the products, 22 copies codes (a lane each issues), 2 to 5 read the sums, 6 to 21 take weights out.  Every wait on a barrier is bounded by a clock; a
// waiter that gives up raises *err, every role leaves its loop, the block lets its copies and products end and frees its tensor memory.
#include "four_bit.cuh"
#include "drain.h"
#include <cuda.h>
#include <type_traits>

namespace {
typedef __nv_bfloat16 bf16;
constexpr int BM = 128, BK = 64, WARPS = 23, TAKERS = 16;
constexpr long long WAIT_CYCLES = 2000000000LL;
constexpr unsigned SLEEP_NS = 10000;   // a waiter sleeps up to so long before it asks again: asking takes issue slots from those it waits for

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
__device__ __forceinline__ bool mbar_test(void* bar, unsigned parity) {   // (does not sleep)
  unsigned ok;
  asm volatile("{ .reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_wait(void* bar, unsigned parity, int* err, volatile int* failed, int site) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (*failed) return false;
    if (clock64() - t0 > WAIT_CYCLES) {
      if (err) atomicCAS(err, 0, 200 + site);   // the first wait that gave up names its place
      *failed = 1;
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, void* bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y) : "memory");
}
// K-major operand tile, 128-byte swizzle: rows of 64 bf16 (128 bytes), 8-row groups 1024 bytes apart.
__device__ __forceinline__ unsigned long long umma_desc(const void* smem_tile) {
  unsigned long long d = 0;
  d |= (unsigned long long)((smem_u32(smem_tile) & 0x3FFFF) >> 4);
  d |= (unsigned long long)1 << 16;
  d |= (unsigned long long)(1024 >> 4) << 32;
  d |= (unsigned long long)1 << 46;
  d |= (unsigned long long)2 << 61;
  return d;
}
// kind::f16 instruction descriptor: D fp32, A and B bf16, both K-major, N >> 3 at bit 17, M >> 4 at bit 24
__host__ __device__ constexpr unsigned idesc(int m, int n) { return (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(n >> 3) << 17) | ((unsigned)(m >> 4) << 24); }
// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void umma(unsigned d_tmem, unsigned a_tmem, unsigned long long b_desc, unsigned id, unsigned accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(id), "r"(accumulate) : "memory");
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

struct Inputs { const bf16* x; long long x_stride; const uint4* codes; const uint2* scales; int k, group_bits; };
struct Params { void* y; float* pieces; int* err; int m, n, blocks, group_bits, tiles; Inputs in; };

// A 32-bit result that is not finite, worked out again from the definition: an infinity times a weight and times the rest of its rounding, which may be 0 or of the other sign,
// is not what it is times their sum.
__device__ __noinline__ float defined_result(const Inputs in, int row, int m) {   // (a copy: what is handed on by its address is read again behind every barrier)
  const bf16* const x = in.x + m * in.x_stride;
  return defined_product(in.codes, in.scales, row, in.k, in.group_bits, [x](int i) { return ld_prev_bf16(x + i); });
}

// KU: blocks of 64 inputs in a unit, two where enough stages of x fit: every handshake between the roles costs the same for twice the work (48 rows, 19,456
// outputs of 2,560 inputs: 28.6 us with units of 64 inputs).  GN: groups that begin in a unit.
template <int NB> constexpr int units_of() { return NB == 256 ? 1 : 2; }
template <int NB, int GN, bool LOW> struct Layout {
  static constexpr int KU = units_of<NB>(), X_BLOCK = NB * BK * 2, STAGE_BYTES = X_BLOCK * KU;   // a stage of x, block by block; multiples of 1024
  static constexpr int SUMS_BYTES = LOW ? NB * BM * 4 : 0;                                       // of segments (below)
  static constexpr int RING = LOW && NB == 128 ? 6 : 8;                                          // units whose codes are on their way
  static constexpr int CODE_BYTES = 4096 * KU, SCALE_BYTES = 512 * GN, SLOT_BYTES = CODE_BYTES + SCALE_BYTES, RING_BYTES = RING * SLOT_BYTES;   // multiples of 128
  // tensor memory: sums of ACCS runs, then the stages of weights (LOW: and of their rests), two inputs a column
  static constexpr int ACCS = NB == 256 ? 1 : 2, W_COLS = BK / 2 * KU, STAGE_COLS = W_COLS * (LOW ? 2 : 1), W_COL0 = ACCS * NB, TMEM_COLS = 512;
  static constexpr int ROOM = (225 * 1024 - RING_BYTES - SUMS_BYTES) / STAGE_BYTES, COLS = (TMEM_COLS - W_COL0) / STAGE_COLS, FIT = ROOM < COLS ? ROOM : COLS;
  static constexpr int STAGES = FIT < 6 ? FIT : 6;
  // Teams of warps that take units' weights out in turn.  A parity tells two phases of a barrier apart, not three: a team that waits for the products of the unit that
  // had its stage before has to know that those of the unit before that are done.  It has written its last unit, TEAMS before this one, into a stage that the products
  // of the unit TEAMS + STAGES before this one had left; so TEAMS is at most STAGES.
  static constexpr int TEAMS = STAGES >= 4 ? 4 : 2, TEAM = TAKERS / TEAMS;
  // Units that are summed in tensor memory at a time.  Every product there cuts what it adds to off, not rounds it: 2^-26 of the sum each in the mean, always towards zero.
  // For 32-bit results 512 inputs, 64 products, are summed so; their sums are added up in shared memory by the threads that read them, rounded.
  static constexpr int SEGMENT = LOW ? 512 / (BK * KU) : 1 << 30;
  static_assert(!LOW || NB <= 128, "sums of segments fit beside up to 128 rows");
  static_assert(STAGES >= 2 && TEAMS <= STAGES && TEAMS <= RING, "phases of a stage's barrier");
  static_assert(W_COL0 + STAGES * STAGE_COLS <= TMEM_COLS, "of tensor memory");
  static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + RING_BYTES + SUMS_BYTES + 8 * (2 * STAGES + 2 * RING + 4) + 64;
  static_assert(SMEM_BYTES <= 227 * 1024, "of a block");
};
// (32 bits: the launcher sees to U G being below 2^32)
__device__ __forceinline__ unsigned first_unit(unsigned U, unsigned G, unsigned i) { return U * i / G; }
// the block that has unit u: the last one that begins at or before it
__device__ __forceinline__ unsigned block_of(unsigned U, unsigned G, unsigned u) { return ((u + 1) * G - 1) / U; }

__device__ __forceinline__ void tmem_st_16x64(unsigned taddr, const unsigned (&v)[16]) {   // 16 lanes' 32 columns; a lane has rows r, r + 8 and columns 8 s + 2c, + 1
  asm volatile("tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
               ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                 "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
// 16 rows of W of one block of a unit by a warp, into tensor memory: rows r and r + 8, four inputs (two columns) of each of four steps.
template <int GN, bool LOW, int KU> __device__ __forceinline__ void take_out(unsigned to, int block, uint4 raw, const uint2 (&sz)[GN]) {
  const unsigned words[4] = {raw.x, raw.y, raw.z, raw.w};
  const __nv_bfloat162 less = __floats2bfloat162_rn(-CODE_BIAS, -CODE_BIAS);
  unsigned v[16], rest[16];
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int g = (4 * block + s) * GN / (4 * KU);
      const unsigned one = h ? sz[g].y : sz[g].x;
#pragma unroll
      for (int e = 0; e < 2; ++e) {   // inputs 16 s + 4c + 2e, + 1
        const unsigned pair = code_pair(words[s], 2 * e + h);
        if constexpr (!LOW) {
          const unsigned ss = __byte_perm(one, one, 0x1010), zz = __byte_perm(one, one, 0x3232);
          const __nv_bfloat162 x = __hfma2(__hadd2(*reinterpret_cast<const __nv_bfloat162*>(&pair), less), *reinterpret_cast<const __nv_bfloat162*>(&ss),
                                           *reinterpret_cast<const __nv_bfloat162*>(&zz));
          v[4 * s + 2 * h + e] = *reinterpret_cast<const unsigned*>(&x);
        } else {
          const GroupCode code = unpack_code(one);
          const float a = fmaf(__uint_as_float(pair << 16) - CODE_BIAS, code.s, code.z), b = fmaf(__uint_as_float(pair & 0xffff0000u) - CODE_BIAS, code.s, code.z);
          const __nv_bfloat162 x = __floats2bfloat162_rn(a, b), y = __floats2bfloat162_rn(a - __low2float(x), b - __high2float(x));
          v[4 * s + 2 * h + e] = *reinterpret_cast<const unsigned*>(&x);
          rest[4 * s + 2 * h + e] = *reinterpret_cast<const unsigned*>(&y);
        }
      }
    }
  tmem_st_16x64(to, v);
  if constexpr (LOW) tmem_st_16x64(to + BK / 2 * KU, rest);
}

template <int NB, int GN, bool LOW>
__global__ void __launch_bounds__(WARPS * 32, 1) linear4_tc_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_codes,
                                                                   const __grid_constant__ CUtensorMap map_scales, const Params p) {
  typedef Layout<NB, GN, LOW> L;
  constexpr int STAGES = L::STAGES, RING = L::RING, KU = L::KU;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* const stages = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* const ring = stages + STAGES * L::STAGE_BYTES;
  unsigned long long* const full = reinterpret_cast<unsigned long long*>(ring + L::RING_BYTES + L::SUMS_BYTES);  // [S] weights (a team), x (TMA) -> products
  unsigned long long* const empty = full + STAGES;                                                                // [S] products -> both
  unsigned long long* const acc_full = empty + STAGES;                                                            // [2] a run's sums -> their readers
  unsigned long long* const acc_empty = acc_full + 2;                                                             // [2] read (128 arrivals) -> products
  unsigned long long* const c_full = acc_empty + 2;                                                               // [RING] TMA -> weights
  unsigned long long* const c_empty = c_full + RING;                                                              // [RING] taken out (a team) -> TMA
  unsigned* const tmem_slot = reinterpret_cast<unsigned*>(c_empty + RING);
  __shared__ int failed_s, issued_s, codes_issued_s;
  __shared__ unsigned long long drained_s;
  volatile int* const failed = &failed_s;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, KB = p.blocks / KU;
  const int U = p.tiles * KB, u0 = first_unit(U, gridDim.x, blockIdx.x), u1 = first_unit(U, gridDim.x, blockIdx.x + 1), n_units = u1 - u0;

  if (threadIdx.x == 0) {
    failed_s = issued_s = codes_issued_s = 0;
    mbar_init(&drained_s, 1);
    for (int s = 0; s < RING; ++s) {
      mbar_init(&c_full[s], 1);
      mbar_init(&c_empty[s], L::TEAM);
    }
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], L::TEAM + 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 128);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(L::TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const unsigned tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  let_next_launch_in();

  // The warps that copy and the one that issues products walk their units as a whole, and one lane issues: what an instruction is given is then the same for every lane,
  // and stays in uniform registers.  Places are counted up, not worked out: a unit takes 700 cycles, and a division is a tenth of that.
  if (warp == 0) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const bool issues = elected();
    int i = 0, s = 0, kb = u0 % KB;
    unsigned par = 1;   // (the first turn finds every stage free)
    for (; i < n_units; ++i) {
      if (i >= STAGES && !__all_sync(0xffffffffu, mbar_wait(&empty[s], par, p.err, failed, 1))) break;
      if (issues) {
        mbar_expect_tx(&full[s], L::STAGE_BYTES);
        unsigned char* const to = stages + (size_t)s * L::STAGE_BYTES;
#pragma unroll
        for (int b = 0; b < KU; ++b) tma_load_2d(to + b * L::X_BLOCK, &map_x, (kb * KU + b) * BK, 0, &full[s]);
      }
      __syncwarp();
      kb = kb + 1 == KB ? 0 : kb + 1;
      if (++s == STAGES) {
        s = 0;
        par ^= 1;
      }
    }
    if (lane == 0) issued_s = i;
  } else if (warp == 1) {
    constexpr unsigned ID = idesc(BM, NB);
    const unsigned long long x_desc0 = umma_desc(stages);
    const bool issues = elected();
    int run = 0, s = 0, kb = u0 % KB;   // runs of one tile's units that this block has begun
    unsigned par = 0, first = 1;
    int left = LOW ? L::SEGMENT - kb % L::SEGMENT : 0;   // units of the segment
    bool there = false;   // the next unit is, as of the last one's products: asked before they are issued, which hides the answer's way
    for (int i = 0; i < n_units; ++i) {
      bool ok = there || mbar_wait(&full[s], par, p.err, failed, 2);
      if (ok && first && run >= L::ACCS)   // the sums that this buffer held have been read
        ok = mbar_wait(&acc_empty[run % L::ACCS], (unsigned)((run / L::ACCS - 1) & 1), p.err, failed, 4);
      if (!__all_sync(0xffffffffu, ok)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const unsigned long long x_desc = x_desc0 + (unsigned)(s * (L::STAGE_BYTES >> 4));
      const unsigned d = tmem + (unsigned)(run % L::ACCS * NB), w = tmem + L::W_COL0 + (unsigned)(s * L::STAGE_COLS);
      const bool tile_ends = kb + 1 == KB, last = tile_ends || i == n_units - 1 || (LOW && left == 1);
      const int ahead = s + 1 == STAGES ? 0 : s + 1;
      there = mbar_test(&full[ahead], ahead == 0 ? par ^ 1 : par);   // (behind the last unit: of a phase that nobody waits for)
      if (issues) {
#pragma unroll
        for (int b = 0; b < KU; ++b)
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk) {
            const unsigned long long x = x_desc + b * (L::X_BLOCK >> 4) + kk * 2;
            const unsigned from = w + b * (BK / 2) + kk * 8;
            umma(d, from, x, ID, b + kk > 0 ? 1u : first ^ 1u);
            if (LOW) umma(d, from + L::W_COLS, x, ID, 1u);
          }
        umma_commit(&empty[s]);
        if (last) umma_commit(&acc_full[run % L::ACCS]);
      }
      __syncwarp();
      first = last;
      run += last;
      kb = tile_ends ? 0 : kb + 1;
      if (LOW) left = last ? L::SEGMENT : left - 1;
      s = ahead;
      par ^= ahead == 0;
    }
  } else if (warp < 6) {
    const int q = warp & 3, row = q * 32 + lane;   // the quarter of tensor memory that this warp may read; W row of the tile
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int run = 0;
    float* const sums = reinterpret_cast<float*>(ring + L::RING_BYTES) + row;   // (LOW) [NB][128]: of a tile's segments so far; the thread's own row
    for (int u = u0; u < u1; ++run) {
      const int tile = u / KB, b = run % L::ACCS, begin = tile * KB, part_end = min(u1, begin + KB);
      const int end = LOW ? min(part_end, u + L::SEGMENT - (u - begin) % L::SEGMENT) : part_end;
      const bool whole = u0 <= begin && part_end == begin + KB, more = LOW && u > begin && u > u0;   // more: not the first segment
      u = end;
      bool ok = mbar_wait(&acc_full[b], (unsigned)(run / L::ACCS & 1), p.err, failed, 5);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const unsigned from = tmem + ((unsigned)(q * 32) << 16) + (unsigned)(b * NB);
      const int out = tile * BM + row;
      // a piece: of this block, its first tile's (0) or its last one's (1); [slot][NB][128]
      float* const piece = p.pieces + (size_t)(2 * blockIdx.x + (u0 < begin ? 1 : 0)) * BM * NB + row;
      float none[2] = {0.f, 0.f};   // (LOW) of infinities and NaN among the tile's results
#pragma unroll 1
      for (int m0 = 0; m0 < NB; m0 += 16) {
        float v[16];
        tmem_ld16(from + m0, v);
        if (LOW && more) {
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] += sums[(m0 + j) * BM];
        }
        if (LOW && end != part_end) {   // more of this tile's inputs follow
#pragma unroll
          for (int j = 0; j < 16; ++j) sums[(m0 + j) * BM] = v[j];
        } else if (whole) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (m0 + j < p.m && out < p.n) {
              if (LOW) reinterpret_cast<float*>(p.y)[(size_t)(m0 + j) * p.n + out] = v[j];
              else reinterpret_cast<bf16*>(p.y)[(size_t)(m0 + j) * p.n + out] = __float2bfloat16_rn(v[j]);
            }
          if constexpr (LOW) {
#pragma unroll
            for (int j = 0; j < 16; ++j) none[j & 1] = fmaf(v[j], 0.f, none[j & 1]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (m0 + j < p.m) __stcg(piece + (size_t)(m0 + j) * BM, v[j]);
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      mbar_arrive(&acc_empty[b]);
      if (LOW && whole && end == part_end && !(none[0] + none[1] == 0.f) && out < p.n)   // products go on meanwhile
#pragma unroll 1
        for (int m = 0; m < p.m; ++m) {
          float* const at = reinterpret_cast<float*>(p.y) + (size_t)m * p.n + out;
          if (!(fabsf(*at) < INFINITY)) *at = defined_result(p.in, out, m);
        }
      __syncwarp();   // reading tensor memory is the whole warp's
    }
  } else if (warp == 6 + TAKERS) {   // codes depend on no earlier launch
    const bool issues = elected();
    int i = 0, s = 0, kb = u0 % KB, tile = u0 / KB;
    unsigned par = 1;
    for (; i < n_units; ++i) {
      if (i >= RING && !__all_sync(0xffffffffu, mbar_wait(&c_empty[s], par, p.err, failed, 7))) break;
      if (issues) {
        unsigned char* const to = ring + s * L::SLOT_BYTES;
        mbar_expect_tx(&c_full[s], L::SLOT_BYTES);
        tma_load_2d(to, &map_codes, kb * (128 * KU), tile * 8, &c_full[s]);
        tma_load_2d(to + L::CODE_BYTES, &map_scales, ((kb * (64 * KU)) >> p.group_bits) * 16, tile * 8, &c_full[s]);
      }
      __syncwarp();
      if (++kb == KB) {
        kb = 0;
        ++tile;
      }
      if (++s == RING) {
        s = 0;
        par ^= 1;
      }
    }
    if (lane == 0) codes_issued_s = i;
  } else {
    // teams take the units in turn, so that one's waits and fence are another's work
    constexpr int TEAM = L::TEAM;
    const int q = warp & 3, upper = (warp - 6) % TEAM >> 2;   // the quarter of tensor memory that this warp may write; of a team of eight, which half of it
    for (int i = (warp - 6) / TEAM; i < n_units; i += L::TEAMS) {
      const int s = i % STAGES, cs = i % RING;
      bool ok = mbar_wait(&c_full[cs], (unsigned)((i / RING) & 1), p.err, failed, 8);
      if (ok && i >= STAGES) ok = mbar_wait(&empty[s], (unsigned)(((i / STAGES) - 1) & 1), p.err, failed, 6);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const unsigned char* const from = ring + cs * L::SLOT_BYTES;
#pragma unroll
      for (int j = 0; j < 8 / TEAM; ++j) {   // 16 rows of W
        const int t = 2 * q + j + upper;
        uint2 sz[GN];
#pragma unroll
        for (int g = 0; g < GN; ++g) sz[g] = *reinterpret_cast<const uint2*>(from + L::CODE_BYTES + (t * GN + g) * 64 + (lane >> 2) * 8);
#pragma unroll
        for (int b = 0; b < KU; ++b) {
          const uint4 raw = *reinterpret_cast<const uint4*>(from + (t * KU + b) * 512 + lane * 16);
          take_out<GN, LOW, KU>(tmem + ((unsigned)(16 * t) << 16) + (unsigned)(L::W_COL0 + s * L::STAGE_COLS + b * (BK / 2)), b, raw, sz);
        }
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&full[s]);
        mbar_arrive(&c_empty[cs]);
      }
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*failed) {
    // a wait ran out: give copies and products that may still be in flight a bounded time to end
    const long long t0 = clock64();
    auto expired = [&] { return clock64() - t0 > WAIT_CYCLES; };
    if (threadIdx.x == 0) ring_drain(issued_s, STAGES, [&](int s, unsigned parity) { return mbar_try_wait(&full[s], parity); }, expired);   // (or as long, where weights are missing)
    if (threadIdx.x == (6 + TAKERS) * 32) ring_drain(codes_issued_s, RING, [&](int s, unsigned parity) { return mbar_try_wait(&c_full[s], parity); }, expired);
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

// Tiles that several blocks had pieces of: a block per tile and two rows of x, a thread per W row; the pieces in the blocks' order.
constexpr int JOIN_ROWS = 2;
template <int NB, typename O>
__global__ void __launch_bounds__(128) linear4_pieces_kernel(const float* pieces, O* y, int m, int n, unsigned blocks, unsigned tiles, unsigned G,   // blocks: units of a tile
                                                             const Inputs in) {
  const unsigned U = tiles * blocks, begin = blockIdx.x * blocks, first = block_of(U, G, begin), last = block_of(U, G, begin + blocks - 1);
  if (first == last) {   // (what follows this launch takes it that the one before is complete, also where no tile had pieces)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const int out = blockIdx.x * BM + threadIdx.x, m0 = blockIdx.y * JOIN_ROWS;
  constexpr size_t SLOT = (size_t)BM * NB;
  // the first block's last piece if its units began in the tile before; every other block begins with this tile
  const float* const from = pieces + (size_t)m0 * BM + threadIdx.x;
  const float* const head = from + (2 * first + (first_unit(U, G, first) < begin ? 1 : 0)) * SLOT;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float v[JOIN_ROWS];
#pragma unroll
  for (int j = 0; j < JOIN_ROWS; ++j) v[j] = m0 + j < m ? __ldcg(head + j * BM) : 0.f;
#pragma unroll 8
  for (unsigned i = first + 1; i <= last; ++i)
#pragma unroll
    for (int j = 0; j < JOIN_ROWS; ++j)
      if (m0 + j < m) v[j] += __ldcg(from + 2 * i * SLOT + j * BM);
  if (out < n)
#pragma unroll
    for (int j = 0; j < JOIN_ROWS; ++j)
      if (m0 + j < m) {
        if (sizeof(O) == 4 && !(fabsf(v[j]) < INFINITY)) v[j] = defined_result(in, out, m0 + j);
        y[(size_t)(m0 + j) * n + out] = from_f32<O>(v[j]);
      }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess) fn = (EncodeTiledFn)p;
  }
  return fn;
}

int sm_count() {
  static int sms = 0;
  if (sms == 0) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) sms = 148;
  }
  return sms;
}

template <typename... P, typename... A> int launch(void (*kern)(P...), dim3 grid, int threads, size_t bytes, bool dependent, cudaStream_t st, A... a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, (P)a...);
  return e != cudaSuccess ? (int)e : launch_status();
}

struct Operands { EncodeTiledFn enc; const void *x, *codes, *scales; long long x_stride; int k, group; };
// rows of `wide` elements, `step` bytes apart, in boxes of box_wide x box_rows; zeros out of range
bool encode(EncodeTiledFn enc, CUtensorMap* map, CUtensorMapDataType type, const void* base, long long wide, long long rows, long long step, int box_wide, int box_rows,
            CUtensorMapSwizzle swizzle) {
  const cuuint64_t dims[2] = {(cuuint64_t)wide, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)step};
  const cuuint32_t box[2] = {(cuuint32_t)box_wide, (cuuint32_t)box_rows}, ones[2] = {1, 1};
  return enc(map, type, 2, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
int padded_rows(int m) { return m <= 32 ? 32 : m <= 64 ? 64 : m <= 128 ? 128 : 256; }
int blocks_of(int k) { return (k + 127) / 128 * 2; }
// the launch's blocks: one a multiprocessor, if there are as many units
int grid_of(int n, int units) {
  const long long all = (long long)((n + BM - 1) / BM) * units;
  return (int)(all < sm_count() ? all : sm_count());
}

template <int NB, int GN, bool LOW> int run(const Operands& o, const Params& p, int pdl, cudaStream_t st) {
  typedef Layout<NB, GN, LOW> L;
  constexpr int KU = L::KU;
  const int units = p.blocks / KU, G = grid_of(p.n, units), tiles16 = (p.n + 15) / 16, groups = p.blocks * 64 / o.group;
  if ((long long)p.tiles * units * (G + 1) >= 1ll << 31) return DRYFT_ERR_UNSUPPORTED;
  CUtensorMap x, codes, scales;
  if (!encode(o.enc, &x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, o.x, o.k, p.m, o.x_stride * 2, BK, NB, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !encode(o.enc, &codes, CU_TENSOR_MAP_DATA_TYPE_UINT32, o.codes, (long long)p.blocks * 128, tiles16, (long long)p.blocks * 512, 128 * KU, 8, CU_TENSOR_MAP_SWIZZLE_NONE) ||
      !encode(o.enc, &scales, CU_TENSOR_MAP_DATA_TYPE_UINT32, o.scales, (long long)groups * 16, tiles16, (long long)groups * 64, 16 * GN, 8, CU_TENSOR_MAP_SWIZZLE_NONE))
    return DRYFT_ERR_UNSUPPORTED;
  auto kern = linear4_tc_kernel<NB, GN, LOW>;
  static bool asked[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return DRYFT_ERR_UNSUPPORTED;
  if (!asked[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM_BYTES);
    if (e != cudaSuccess) return (int)e;
    asked[dev] = true;
  }
  const int rc = launch(kern, dim3(G), WARPS * 32, L::SMEM_BYTES, pdl & 1, st, x, codes, scales, p);
  if (rc || G == p.tiles) return rc;   // (a tile a block: no pieces)
  typedef typename std::conditional<LOW, float, bf16>::type O;
  return launch(linear4_pieces_kernel<NB, O>, dim3(p.tiles, (p.m + JOIN_ROWS - 1) / JOIN_ROWS), 128, 0, pdl & 2, st, (const float*)p.pieces, (O*)p.y, p.m, p.n,
                units, p.tiles, G, p.in);
}
template <int NB, bool LOW> int by_group(const Operands& o, const Params& p, int pdl, cudaStream_t st) {
  constexpr int WIDE = 64 * units_of<NB>();   // inputs of a unit
  switch (o.group) {
    case 128: return run<NB, 1, LOW>(o, p, pdl, st);
    case 64: return run<NB, WIDE / 64, LOW>(o, p, pdl, st);
    case 32: return run<NB, WIDE / 32, LOW>(o, p, pdl, st);
    case 16: return run<NB, WIDE / 16, LOW>(o, p, pdl, st);
  }
  return DRYFT_ERR_UNSUPPORTED;
}
}  // namespace

// Rows of a pass: with sums of segments in shared memory beside them no more than 128 fit.
static int rows_of_pass(int out_f32, int m) { return out_f32 && m > 128 ? 128 : m; }

// Floats of the workspace that a product needs.
DRYFT_API long long dryft_linear4_tc_pieces(int m, int n, int k) { return 2ll * grid_of(n, blocks_of(k)) * BM * padded_rows(m); }
// Launches that it makes: for each pass one where every block has a whole tile, else a second one for the pieces.
DRYFT_API int dryft_linear4_tc_launches(int out_f32, int m, int n, int k) {
  const int rows = rows_of_pass(out_f32, m), units = blocks_of(k) / (padded_rows(rows) == 256 ? units_of<256>() : units_of<128>());
  return (grid_of(n, units) == (n + BM - 1) / BM ? 1 : 2) * ((m + rows - 1) / rows);
}

// y [m, n] = x [m, k] w^T, m <= 256; x bfloat16, rows x_stride numbers apart on 16-byte boundaries; y bfloat16 or (out_f32) float32.
// pdl: 1, the product is a programmatic dependent of the launch before it; 2, its further launches are, each of the one before; both or neither.
DRYFT_API int dryft_linear4_tc(int out_f32, const void* x, long long x_stride, const void* codes, const void* scales, void* y, float* pieces, int m, int n, int k,
                               int group, int pdl, int* err, void* stream) {
  if (m <= 0 || n <= 0) return 0;
  if (m > 256 || k <= 0 || k % 16) return DRYFT_ERR_UNSUPPORTED;
  const EncodeTiledFn enc = encode_fn();
  if (!enc) return DRYFT_ERR_UNSUPPORTED;
  const cudaStream_t st = (cudaStream_t)stream;
  const int pass = rows_of_pass(out_f32, m);
  for (int m0 = 0; m0 < m; m0 += pass) {
    const bf16* const rows = (const bf16*)x + m0 * x_stride;
    const int count = pass < m - m0 ? pass : m - m0, overlap = m0 == 0 ? pdl : pdl & 2 ? 3 : 0;
    const Operands o = {enc, rows, codes, scales, x_stride, k, group};
    const Params p = {(char*)y + (size_t)m0 * n * (out_f32 ? 4 : 2), pieces, err, count, n, blocks_of(k), __builtin_ctz(group), (n + BM - 1) / BM,
                      {rows, x_stride, (const uint4*)codes, (const uint2*)scales, k, __builtin_ctz(group)}};
    int rc = DRYFT_ERR_UNSUPPORTED;
    switch (padded_rows(count)) {
      case 32: rc = out_f32 ? by_group<32, true>(o, p, overlap, st) : by_group<32, false>(o, p, overlap, st); break;
      case 64: rc = out_f32 ? by_group<64, true>(o, p, overlap, st) : by_group<64, false>(o, p, overlap, st); break;
      case 128: rc = out_f32 ? by_group<128, true>(o, p, overlap, st) : by_group<128, false>(o, p, overlap, st); break;
      case 256: rc = by_group<256, false>(o, p, overlap, st); break;   // (not for 32-bit results)
    }
    if (rc) return rc;
  }
  return 0;
}
