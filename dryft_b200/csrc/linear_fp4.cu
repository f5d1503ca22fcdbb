// y = x w^T with both operands in microscaled 4-bit floating point (fp4.cuh), on the 5th-generation tensor cores, which multiply such numbers and scales as they lie:
// tcgen05.mma kind::mxf4 (a scale for 32 inputs) and kind::mxf4nvf4 (for 16), sums of 64 inputs an instruction in 32 bits.
//
// Computed transposed: a tile is 128 rows of W, on the M side, against NB rows of x (16 to 256, padded), its 128 x NB sums in tensor memory, a W row a lane.  A stage of the ring is
// 256 inputs: a block of W and one or two of x, each a copy of consecutive bytes.  The scales go on from shared into tensor memory (tcgen05.cp), in front of the four products of
// their stage, by the thread that issues those: the copies and products of one thread run in the order that they were issued in.
//
// Warps: 0 copies, 1 issues, 2 to 5 read the sums out.  Every wait on a barrier is bounded by a clock; a waiter that gives up raises *err, every role leaves its loop, the
// block lets its copies and products end and frees its tensor memory.
#include "fp4.cuh"
#include "drain.h"

namespace {
using namespace fp4;
typedef __nv_bfloat16 bf16;
constexpr int THREADS = 6 * 32;
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
__device__ __forceinline__ bool mbar_wait(void* bar, unsigned parity, int* err, volatile int* failed, int site) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity)) {
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
__device__ __forceinline__ void scales_to_tmem(unsigned taddr, unsigned long long desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// Instruction descriptor: A and B E2M1, N >> 3 at bit 17, scales' type at bit 23 (0 E4M3, 1 E8M0), M >> 7 at bit 27; which of a word's scales the instruction takes at
// bits 4 (B) and 29 (A): all four (NV), the first or the second two (MX).
template <int KIND> __device__ __forceinline__ constexpr unsigned idesc(int n, int scale) {
  return (1u << 7) | (1u << 10) | ((unsigned)(n >> 3) << 17) | (KIND == MX ? 1u << 23 : 0u) | (1u << 27) | ((unsigned)scale << 4) | ((unsigned)scale << 29);
}
// D[tmem] (+)= A[smem] B[smem], 64 inputs
template <int KIND> __device__ __forceinline__ void umma(unsigned d, unsigned long long a, unsigned long long b, unsigned id, unsigned sa, unsigned sb, unsigned accumulate) {
  if (KIND == NV)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
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
  const unsigned char *x, *w;          // blocks (fp4.cuh)
  const float *x_factors, *w_factors;  // NV
  void* y;
  int* err;
  int m, n, blocks;   // blocks: of 256 inputs
};

template <int KIND, int NB> struct Layout {
  typedef Format<KIND> F;
  static constexpr int XB = NB > ROWS ? 2 : 1;                                   // blocks of x in a stage
  static constexpr int X_CODES = NB * (INPUTS / 2), X_BYTES = XB * F::SCALE_BYTES + X_CODES, STAGE_BYTES = F::BLOCK_BYTES + X_BYTES;   // multiples of 1024
  static constexpr int ROOM = 225 * 1024 / STAGE_BYTES, STAGES = ROOM < 12 ? ROOM : 12;
  // tensor memory: sums of ACCS tiles, then the scales of two stages
  static constexpr int ACCS = NB > 128 ? 1 : 2, SCALE_COLS = 4 * F::WORDS * (1 + XB), NEED_COLS = ACCS * NB + 2 * SCALE_COLS;
  static constexpr int TMEM_COLS = NEED_COLS <= 128 ? 128 : NEED_COLS <= 256 ? 256 : 512;
  static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + 8 * (2 * STAGES + 4) + 16;
  static_assert(NEED_COLS <= 512 && SMEM_BYTES <= 227 * 1024 && STAGES >= 3, "of a block");
};

template <int KIND, int NB, typename O> __global__ void __launch_bounds__(THREADS, 1) linear_fp4_kernel(const Params p) {
  typedef Layout<KIND, NB> L;
  typedef typename L::F F;
  constexpr int STAGES = L::STAGES, XB = L::XB;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* const stages = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned long long* const full = reinterpret_cast<unsigned long long*>(stages + STAGES * L::STAGE_BYTES);   // [S] copies -> products
  unsigned long long* const empty = full + STAGES;                                                             // [S] products -> copies
  unsigned long long* const acc_full = empty + STAGES;                                                         // [2] a tile's sums -> their readers
  unsigned long long* const acc_empty = acc_full + 2;                                                          // [2] read (128 arrivals) -> products
  unsigned* const tmem_slot = reinterpret_cast<unsigned*>(acc_empty + 2);
  __shared__ int failed_s, issued_s;
  __shared__ unsigned long long drained_s;
  volatile int* const failed = &failed_s;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, KB = p.blocks;
  const int x_tiles = (p.m + NB - 1) / NB, tiles = (p.n + ROWS - 1) / ROWS * x_tiles;   // those of one W row range behind one another: W crosses memory once

  if (threadIdx.x == 0) {
    failed_s = issued_s = 0;
    mbar_init(&drained_s, 1);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
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

  if (warp == 0) {
    const bool issues = elected();
    int i = 0, s = 0;
    unsigned par = 1;   // (the first turn finds every stage free)
    bool ok = true, waited = false;
    for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
      const unsigned char* const w = p.w + (size_t)(t / x_tiles) * KB * F::BLOCK_BYTES;
      const unsigned char* const x = p.x + (size_t)(t % x_tiles) * XB * KB * F::BLOCK_BYTES;
      const bool second = XB == 2 && (t % x_tiles) * NB + ROWS < p.m;   // (rows behind the last block of x: any numbers do)
      for (int kb = 0; kb < KB; ++kb, ++i) {
        ok = i < STAGES || __all_sync(0xffffffffu, mbar_wait(&empty[s], par, p.err, failed, 1));
        if (!ok) break;
        unsigned char* const to = stages + (size_t)s * L::STAGE_BYTES;
        if (issues) {
          mbar_expect_tx(&full[s], XB == 2 && !second ? F::BLOCK_BYTES * 2 : L::STAGE_BYTES);
          bulk_load(to, w + (size_t)kb * F::BLOCK_BYTES, F::BLOCK_BYTES, &full[s]);
        }
        if (!waited) {   // W depends on no launch that may still be running
          asm volatile("griddepcontrol.wait;" ::: "memory");
          waited = true;
        }
        if (issues) {
          const unsigned char* const xb = x + (size_t)kb * F::BLOCK_BYTES;
          if (XB == 1) bulk_load(to + F::BLOCK_BYTES, xb, L::X_BYTES, &full[s]);
          else {
            unsigned char* const scales = to + F::BLOCK_BYTES;
            unsigned char* const codes = scales + XB * F::SCALE_BYTES;
            bulk_load(scales, xb, F::SCALE_BYTES, &full[s]);
            bulk_load(codes, xb + F::SCALE_BYTES, CODE_BYTES, &full[s]);
            if (second) {
              bulk_load(scales + F::SCALE_BYTES, xb + (size_t)KB * F::BLOCK_BYTES, F::SCALE_BYTES, &full[s]);
              bulk_load(codes + CODE_BYTES, xb + (size_t)KB * F::BLOCK_BYTES + F::SCALE_BYTES, CODE_BYTES, &full[s]);
            }
          }
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
    bool ok = true;
    for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x, ++run) {
      const int b = run % L::ACCS;
      const unsigned d = tmem + b * NB;
      ok = run < L::ACCS || __all_sync(0xffffffffu, mbar_wait(&acc_empty[b], (unsigned)((run / L::ACCS - 1) & 1), p.err, failed, 4));
      for (int kb = 0; ok && kb < KB; ++kb) {
        ok = __all_sync(0xffffffffu, mbar_wait(&full[s], par, p.err, failed, 2));
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (issues) {
          unsigned char* const at = stages + (size_t)s * L::STAGE_BYTES;
          const unsigned sw = tmem + L::ACCS * NB + buffer * L::SCALE_COLS, sx = sw + 4 * F::WORDS;
          const unsigned long long w_scales = scales_desc(at), x_scales = scales_desc(at + F::BLOCK_BYTES);
          const unsigned long long w = codes_desc(at + F::SCALE_BYTES), x = codes_desc(at + F::BLOCK_BYTES + XB * F::SCALE_BYTES);
#pragma unroll
          for (int j = 0; j < F::WORDS; ++j) {
            scales_to_tmem(sw + 4 * j, w_scales + j * (512 >> 4));
#pragma unroll
            for (int h = 0; h < XB; ++h) scales_to_tmem(sx + 4 * XB * j + 4 * h, x_scales + (j * 512 + h * F::SCALE_BYTES >> 4));
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int word = j * F::WORDS / 4;
            umma<KIND>(d, w + 2 * j, x + 2 * j, idesc<KIND>(NB, KIND == MX ? 2 * (j & 1) : 0), sw + 4 * word, sx + 4 * XB * word, kb > 0 || j > 0);
          }
          umma_commit(&empty[s]);
          if (kb == KB - 1) umma_commit(&acc_full[b]);
        }
        __syncwarp();
        buffer ^= 1;
        if (++s == STAGES) {
          s = 0;
          par ^= 1;
        }
      }
    }
  } else {
    const int q = warp & 3;   // the quarter of tensor memory that this warp may read
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int run = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++run) {
      const int b = run % L::ACCS, row = t / x_tiles * ROWS + q * 32 + lane, m0 = t % x_tiles * NB;
      const float wf = KIND == NV && row < p.n ? p.w_factors[row] : 1.f;
      if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[b], (unsigned)(run / L::ACCS & 1), p.err, failed, 5))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const unsigned from = tmem + ((unsigned)(q * 32) << 16) + b * NB;
#pragma unroll 1
      for (int j0 = 0; j0 < NB && m0 + j0 < p.m; j0 += 16) {
        float v[16];
        tmem_ld16(from + j0, v);
        const float xf = KIND == NV && m0 + j0 + (lane & 15) < p.m ? ld_prev(p.x_factors + m0 + j0 + (lane & 15)) : 1.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float f = __shfl_sync(0xffffffffu, xf, j);
          if (m0 + j0 + j < p.m && row < p.n) reinterpret_cast<O*>(p.y)[(size_t)(m0 + j0 + j) * p.n + row] = from_f32<O>(KIND == NV ? v[j] * wf * f : v[j]);
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      mbar_arrive(&acc_empty[b]);
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

int sm_count() {
  static int sms = 0;
  if (sms == 0) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) sms = 148;
  }
  return sms;
}

template <int KIND, int NB, typename O> int run(const Params& p, bool dependent, cudaStream_t st) {
  typedef Layout<KIND, NB> L;
  auto kern = linear_fp4_kernel<KIND, NB, O>;
  static bool asked[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return DRYFT_ERR_UNSUPPORTED;
  if (!asked[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM_BYTES);
    if (e != cudaSuccess) return (int)e;
    asked[dev] = true;
  }
  const long long tiles = (long long)((p.n + ROWS - 1) / ROWS) * ((p.m + NB - 1) / NB);
  if (tiles > 0x7ffffff0ll) return DRYFT_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles < sm_count() ? tiles : sm_count()));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = L::SMEM_BYTES;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  return e != cudaSuccess ? (int)e : launch_status();
}
template <int KIND, typename O> int by_rows(const Params& p, bool dependent, cudaStream_t st) {
  if (p.m <= 16) return run<KIND, 16, O>(p, dependent, st);
  if (p.m <= 32) return run<KIND, 32, O>(p, dependent, st);
  if (p.m <= 64) return run<KIND, 64, O>(p, dependent, st);
  if (p.m <= 128) return run<KIND, 128, O>(p, dependent, st);
  return run<KIND, 256, O>(p, dependent, st);
}
}  // namespace

// y [m, n] = x w^T; x, w: blocks of 128 rows by 256 inputs (fp4.cuh) with factors for each row (NV); y bfloat16 or float32
DRYFT_API int dryft_linear_fp4(int kind, int out_bf16, const void* x, const void* x_factors, const void* w, const void* w_factors, void* y, int m, int n, int k, int pdl,
                               int* err, void* stream) {
  if (m <= 0 || n <= 0) return 0;
  if (k <= 0) return DRYFT_ERR_UNSUPPORTED;
  const Params p = {(const unsigned char*)x, (const unsigned char*)w, (const float*)x_factors, (const float*)w_factors, y, err, m, n, blocks_of(k)};
  const cudaStream_t st = (cudaStream_t)stream;
  if (kind == NV) return out_bf16 ? by_rows<NV, bf16>(p, pdl, st) : by_rows<NV, float>(p, pdl, st);
  return out_bf16 ? by_rows<MX, bf16>(p, pdl, st) : by_rows<MX, float>(p, pdl, st);
}
