// Attention of query rows over the paged cache held in 4 bits (four_bit.cuh).  Compiled per model with -DDRYFT_HEAD_DIM, -DDRYFT_GROUP (query heads per key
// head), -DDRYFT_PAGE and -DDRYFT_BITS_GROUP (numbers that share a scale).
//
// Row n at position p of slot s sees the keys j with  max(0, p + 1 - window) <= j <= p  (window <= 0: all of them); a row of slot -1 is padding, its output zeros.
// A block takes up to eight query heads of a (row, key head) and one split of its keys.  Splits are whole tiles of 16 keys.  Up to eight splits are the blocks of
// a thread-block cluster and meet in its shared memory; more leave (acc, m, l) in memory and a second launch joins them.  Either way in the splits' order.
#include "four_bit.cuh"

#if !defined(DRYFT_HEAD_DIM) || !defined(DRYFT_GROUP) || !defined(DRYFT_PAGE) || !defined(DRYFT_BITS_GROUP)
#error "compile with -DDRYFT_HEAD_DIM=.. -DDRYFT_GROUP=.. -DDRYFT_PAGE=.. -DDRYFT_BITS_GROUP=.."
#endif

namespace {
constexpr int D = DRYFT_HEAD_DIM, G = DRYFT_GROUP, PAGE = DRYFT_PAGE, BG = DRYFT_BITS_GROUP;
constexpr int UNITS = kv4_units(D), ROW = kv4_row_bytes(D), GROUPS = D / BG;
constexpr size_t TILE = kv4_tile_bytes(PAGE, D, BG);
static_assert(D % 16 == 0 && D <= 256 && D % BG == 0 && BG % 16 == 0 && BG <= 128, "head size in steps of 16, whole groups");
static_assert(G >= 1 && G <= 16 && PAGE % 16 == 0, "1..16 query heads per key head, pages of whole tiles of 16 tokens");

struct Span { int first, end; };   // keys of a split: whole tiles of 16, `least` of them at least, cut at the row's first and last key
__device__ __forceinline__ Span span_of(int pos, int window, int split, int splits, int least) {
  const int lo = window > 0 && pos + 1 > window ? pos + 1 - window : 0;
  const int t0 = lo / 16, tiles = pos / 16 + 1 - t0, per = max(least, (tiles + splits - 1) / splits);
  const int a = t0 + min(tiles, split * per), b = t0 + min(tiles, (split + 1) * per);
  return {max(lo, a * 16), min(pos + 1, b * 16)};
}

// What a block knows of its work: head tile `ht` (of eight query heads) of a key head of a row, and its split.
constexpr int HEAD_TILES = (G + 7) / 8, HEADS = G < 8 ? G : 8;   // (query heads of a block; the last tile may have fewer)
struct Work { int n, head, ht, split; };
__device__ __forceinline__ Work work_of(unsigned block, int n_kv, int splits) {
  const unsigned i = block / splits, j = i / HEAD_TILES;
  return {(int)(j / n_kv), (int)(j % n_kv), (int)(i % HEAD_TILES), (int)(block % splits)};
}

// ---------------------------------------------------------------------------------------------- bfloat16: tensor cores
// S^T = K Q^T and O^T = V^T P^T on mma.sync.m16n8k16, the codes as bfloat16 16 + c straight out of the cache's words (`code_pair`):
//   score  = s_k (sum (16 + c) q - 23.5 sum q) + z_k sum q          group by group, in 32 bits; sum q is the query's own
//   output = sum p' (16 + c) + sum p z_v - 23.5 sum p'              p' = bf16(p s_v): the weight rounded with its scale, one rounding of 2^-9 as for plain P
// Scores, running maximum and sums are 32-bit.  A warp walks tiles of 16 keys of its own, copied STAGES - 1 tiles ahead into its own ring.  The maximum
// of a column follows the scores only when one exceeds it by more than 2^8: what is summed stays below 2^8 times the number of keys.
typedef __nv_bfloat16 bf16;
constexpr int STEPS = D / 16, WARPS = 8, STAGES = D <= 128 ? 4 : 3;
constexpr int CODES = 256 * UNITS, SCALES = 64 * GROUPS, STAGE = 2 * (CODES + SCALES);   // bytes of a tile's keys (or values), of their scales, of both
constexpr int PART = D * 8 + 16;                                                           // floats: O^T [dim][head], maxima, sums
constexpr size_t RING = (size_t)WARPS * STAGES * STAGE, JOIN = (size_t)(WARPS + 1) * PART * 4, SMEM = RING > JOIN ? RING : JOIN;

__device__ __forceinline__ unsigned transposed(unsigned v) {   // an 8 x 8 fragment of 16-bit values
  unsigned r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
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
__device__ __forceinline__ float of_block(const float* p, int block) {   // *p in another block of the cluster
  unsigned at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((unsigned)__cvta_generic_to_shared(p)), "r"(block));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

__global__ void __launch_bounds__(WARPS * 32, D <= 128 ? 2 : 1) attn4_mma_kernel(const bf16* __restrict__ q, const unsigned char* __restrict__ k_pages,
                                                                                 const unsigned char* __restrict__ v_pages, const int* __restrict__ page_table,
                                                                                 int max_pages, const int* __restrict__ tok_slot, const int* __restrict__ tok_pos,
                                                                                 bf16* out, float* part_o, float* part_ml, int n_kv, int splits, int cluster, float scale,
                                                                                 int window) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
  const Work w = work_of(blockIdx.x, n_kv, splits);
  const int slot = tok_slot[w.n], pos = tok_pos[w.n], heads = min(8, G - 8 * w.ht);
  const size_t head0 = ((size_t)w.n * n_kv + w.head) * G + 8 * w.ht;   // the block's first query head
  if (slot < 0) {                                                      // (the whole cluster)
    if (w.split == 0)
      for (int i = threadIdx.x; i < heads * D; i += WARPS * 32) out[head0 * D + i] = from_f32<bf16>(0.f);
    return;
  }
  const Span keys = span_of(pos, window, w.split, splits, WARPS);
  const int t0 = keys.first / 16, t1 = (keys.end + 15) / 16;
  const int* const pages = page_table + (size_t)slot * max_pages;

  float acc[STEPS][4], off[GROUPS][2], top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < STEPS; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) off[g][0] = off[g][1] = 0.f;

  if (keys.first < keys.end) {
    unsigned char* const ring = smem + warp * STAGES * STAGE;
    const unsigned ring_at = (unsigned)__cvta_generic_to_shared(ring) + lane * 16;
    // page numbers of 32 pages, one a lane
    int page0 = t0 * 16 / PAGE, held = 0;
    auto fetch = [&](int p) { held = p + lane <= (t1 - 1) * 16 / PAGE ? pages[p + lane] : 0; };
    fetch(page0);
    int ask = t0 + warp, put = 0;
    auto request = [&] {
      const int p = ask * 16 / PAGE;
      if (ask < t1 && p - page0 >= 32) fetch(page0 = p);
      const int page = __shfl_sync(0xffffffffu, held, (p - page0) & 31);
      if (ask < t1) {
        const size_t at = ((size_t)page * n_kv + w.head) * TILE;
        const unsigned char *k = k_pages + at, *v = v_pages + at;
        const int in_page = ask % (PAGE / 16);
        const unsigned to = ring_at + put * STAGE;
#pragma unroll
        for (int i = 0; i < (CODES + 511) / 512; ++i)
          if (CODES % 512 == 0 || i * 512 + lane * 16 < CODES) {
            copy16(to + i * 512, k + in_page * CODES + i * 512 + lane * 16);
            copy16(to + CODES + i * 512, v + in_page * CODES + i * 512 + lane * 16);
          }
#pragma unroll
        for (int i = 0; i < (2 * SCALES + 511) / 512; ++i) {   // keys' scales, then values'
          const int x = i * 512 + lane * 16;
          if (x < 2 * SCALES) copy16(to + 2 * CODES + i * 512, (x < SCALES ? k : v - SCALES) + (size_t)ROW * PAGE + in_page * SCALES + x);
        }
        put = put + 1 == STAGES ? 0 : put + 1;
        ask += WARPS;
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
      qf[j] = r < heads ? *reinterpret_cast<const uint2*>(q + (head0 + r) * D + 16 * j + 4 * c) : make_uint2(0, 0);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      float s = 0.f;
#pragma unroll
      for (int j = g * BG / 16; j < (g + 1) * BG / 16; ++j)
        s += (__uint_as_float(qf[j].x << 16) + __uint_as_float(qf[j].x & 0xffff0000u)) + (__uint_as_float(qf[j].y << 16) + __uint_as_float(qf[j].y & 0xffff0000u));
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      s += __shfl_xor_sync(0xffffffffu, s, 2);
      qs[g][0] = __shfl_sync(0xffffffffu, s, 8 * c);
      qs[g][1] = __shfl_sync(0xffffffffu, s, 8 * c + 4);
    }
    const float scale2 = scale * 1.4426950408889634f;   // scores in powers of two

    int get = 0;
#pragma unroll 1
    for (int t = t0 + warp; t < t1; t += WARPS) {
      __syncwarp();   // every lane has read the stage that the next request writes
      request();
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1));
      __syncwarp();
      const unsigned char* const st = ring + get * STAGE;
      get = get + 1 == STAGES ? 0 : get + 1;
      const bool seen[2] = {t * 16 + r >= keys.first && t * 16 + r < keys.end, t * 16 + r + 8 >= keys.first && t * 16 + r + 8 < keys.end};
      float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        float part[4] = {-CODE_BIAS * qs[g][0], -CODE_BIAS * qs[g][1], -CODE_BIAS * qs[g][0], -CODE_BIAS * qs[g][1]};
#pragma unroll
        for (int j = g * BG / 16; j < (g + 1) * BG / 16; ++j) {
          const unsigned lo = *reinterpret_cast<const unsigned*>(st + r * ROW + (c * UNITS + j / 2) * 4);
          const unsigned hi = *reinterpret_cast<const unsigned*>(st + (r + 8) * ROW + (c * UNITS + j / 2) * 4);
          mma_16816(part, code_pair(lo, 2 * (j & 1)), code_pair(hi, 2 * (j & 1)), code_pair(lo, 2 * (j & 1) + 1), code_pair(hi, 2 * (j & 1) + 1), qf[j].x, qf[j].y);
        }
        const GroupCode lo = unpack_code(*reinterpret_cast<const unsigned*>(st + 2 * CODES + (r * GROUPS + g) * 4));
        const GroupCode hi = unpack_code(*reinterpret_cast<const unsigned*>(st + 2 * CODES + ((r + 8) * GROUPS + g) * 4));
        s[0] = fmaf(lo.s, part[0], fmaf(lo.z, qs[g][0], s[0]));
        s[1] = fmaf(lo.s, part[1], fmaf(lo.z, qs[g][1], s[1]));
        s[2] = fmaf(hi.s, part[2], fmaf(hi.z, qs[g][0], s[2]));
        s[3] = fmaf(hi.s, part[3], fmaf(hi.z, qs[g][1], s[3]));
      }
      float p[4];
      bool over = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[i] = seen[i >> 1] ? s[i] * scale2 : -INFINITY;
        over |= s[i] > top[i & 1] + 8.f;
      }
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float m = fmaxf(top[i], fmaxf(s[i], s[i + 2]));
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
          const float lower = m == top[i] ? 1.f : exp2_fast(top[i] - m);
          top[i] = m;
          sum[i] *= lower;
#pragma unroll
          for (int g = 0; g < GROUPS; ++g) off[g][i] *= lower;
#pragma unroll
          for (int j = 0; j < STEPS; ++j) {
            acc[j][i] *= lower;
            acc[j][i + 2] *= lower;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = s[i] == -INFINITY ? 0.f : exp2_fast(s[i] - top[i & 1]);
        sum[i & 1] += p[i];
      }
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        // a key that is not seen may hold anything: its scale and middle are taken for zeros
        const unsigned lo_w = *reinterpret_cast<const unsigned*>(st + 2 * CODES + SCALES + (r * GROUPS + g) * 4);
        const unsigned hi_w = *reinterpret_cast<const unsigned*>(st + 2 * CODES + SCALES + ((r + 8) * GROUPS + g) * 4);
        const GroupCode lo = unpack_code(seen[0] ? lo_w : 0u), hi = unpack_code(seen[1] ? hi_w : 0u);
        const __nv_bfloat162 w0 = __floats2bfloat162_rn(p[0] * lo.s, p[1] * lo.s), w1 = __floats2bfloat162_rn(p[2] * hi.s, p[3] * hi.s);
        const unsigned b0 = *reinterpret_cast<const unsigned*>(&w0), b1 = *reinterpret_cast<const unsigned*>(&w1);
        off[g][0] = fmaf(p[0], lo.z, fmaf(p[2], hi.z, off[g][0]));
        off[g][1] = fmaf(p[1], lo.z, fmaf(p[3], hi.z, off[g][1]));
        off[g][0] = fmaf(-CODE_BIAS, __uint_as_float(b0 << 16) + __uint_as_float(b1 << 16), off[g][0]);
        off[g][1] = fmaf(-CODE_BIAS, __uint_as_float(b0 & 0xffff0000u) + __uint_as_float(b1 & 0xffff0000u), off[g][1]);
        const unsigned t0_ = transposed(b0), t1_ = transposed(b1);
#pragma unroll
        for (int j = g * BG / 16; j < (g + 1) * BG / 16; ++j) {
          const uint2 v = *reinterpret_cast<const uint2*>(st + CODES + (lane * UNITS + j / 2) * 8);
          const int h = 2 * (j & 1);
          mma_16816(acc[j], code_pair(v.x, h), code_pair(v.x, h + 1), code_pair(v.y, h), code_pair(v.y, h + 1), t0_, t1_);
        }
      }
    }
    asm volatile("cp.async.wait_group 0;");
    // what the lanes of a column have of its sums
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) off[g][i] += __shfl_xor_sync(0xffffffffu, off[g][i], o);
      }
  }

  // the block's part: the warps' sums in the warps' order.  A warp leaves its own in shared memory as they are, [dim][head] and the maxima and sums.
  __syncthreads();
  float* const parts = reinterpret_cast<float*>(smem);
  {
    float* const mine = parts + (warp + 1) * PART;
#pragma unroll
    for (int j = 0; j < STEPS; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) mine[(16 * j + 2 * r + (i >> 1)) * 8 + 2 * c + (i & 1)] = acc[j][i] + off[16 * j / BG][i & 1];
    if (r == 0)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mine[D * 8 + 2 * c + i] = top[i];
        mine[D * 8 + 8 + 2 * c + i] = sum[i];
      }
  }
  __syncthreads();
  const bool alone = splits == 1;
  const int h = threadIdx.x & 7;
  {
    float m = -INFINITY, l = 0.f, by[WARPS];
#pragma unroll
    for (int x = 0; x < WARPS; ++x) m = fmaxf(m, parts[(x + 1) * PART + D * 8 + h]);
#pragma unroll
    for (int x = 0; x < WARPS; ++x) {
      const float mx = parts[(x + 1) * PART + D * 8 + h];
      by[x] = mx == -INFINITY ? 0.f : exp2_fast(mx - m);
      l = fmaf(by[x], parts[(x + 1) * PART + D * 8 + 8 + h], l);
    }
    const float inv = 1.f / l;
    for (int dim = threadIdx.x >> 3; dim < D; dim += WARPS * 4) {
      float v = 0.f;
#pragma unroll
      for (int x = 0; x < WARPS; ++x) v = fmaf(by[x], parts[(x + 1) * PART + dim * 8 + h], v);
      if (h >= heads) continue;
      if (alone)
        out[(head0 + h) * D + dim] = from_f32<bf16>(v * inv);
      else if (cluster)
        parts[dim * 8 + h] = v;
      else
        part_o[((head0 + h) * splits + w.split) * D + dim] = v;
    }
    if (!alone && threadIdx.x < heads) {
      float* const to = cluster ? parts + D * 8 + h : part_ml + ((head0 + h) * splits + w.split) * 2;
      to[0] = m;
      to[cluster ? 8 : 1] = l;
    }
  }
  if (alone || !cluster) return;
  // every block of the cluster joins its share of the dims, over the splits in their order
  cluster_barrier();
  if (h < heads) {
    float m = -INFINITY, l = 0.f, by[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      by[x] = x < splits ? of_block(parts + D * 8 + h, x) : -INFINITY;
      m = fmaxf(m, by[x]);
    }
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      by[x] = by[x] == -INFINITY ? 0.f : exp2_fast(by[x] - m);
      if (x < splits) l = fmaf(by[x], of_block(parts + D * 8 + 8 + h, x), l);
    }
    for (int dim = (threadIdx.x >> 3) * splits + w.split; dim < D; dim += WARPS * 4 * splits) {
      float v = 0.f;
#pragma unroll
      for (int x = 0; x < 8; ++x)
        if (x < splits) v = fmaf(by[x], of_block(parts + dim * 8 + h, x), v);
      out[(head0 + h) * D + dim] = from_f32<bf16>(v / l);
    }
  }
  cluster_barrier();   // a block's shared memory stays until the others have read it
}

// ---------------------------------------------------------------------------------------------- 32-bit
// A thread per key for the scores, a thread per dim for the values, everything in 32-bit multiply-adds.
constexpr int THREADS = 128, DIMS = (D + THREADS - 1) / THREADS;

__global__ void __launch_bounds__(THREADS) attn4_f32_kernel(const float* __restrict__ q, const unsigned char* __restrict__ k_pages,
                                                            const unsigned char* __restrict__ v_pages, const int* __restrict__ page_table, int max_pages,
                                                            const int* __restrict__ tok_slot, const int* __restrict__ tok_pos, float* out, float* part_o,
                                                            float* part_ml, int n_kv, int splits, float scale, int window) {
  __shared__ float qs[HEADS][D], ps[HEADS][THREADS], red[THREADS / 32][HEADS], total[THREADS / 32][HEADS], top[HEADS], sum[HEADS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Work w = work_of(blockIdx.x, n_kv, splits);
  const int slot = tok_slot[w.n], pos = tok_pos[w.n], heads = min(8, G - 8 * w.ht);
  const size_t head0 = ((size_t)w.n * n_kv + w.head) * G + 8 * w.ht;
  if (slot < 0) {
    if (w.split == 0)
      for (int i = tid; i < heads * D; i += THREADS) out[head0 * D + i] = 0.f;
    return;
  }
  const Span keys = span_of(pos, window, w.split, splits, 1);
  for (int i = tid; i < HEADS * D; i += THREADS) qs[i / D][i % D] = i / D < heads ? q[head0 * D + i] : 0.f;
  if (tid < HEADS) {
    top[tid] = -INFINITY;
    sum[tid] = 0.f;
  }
  float acc[DIMS][HEADS];
#pragma unroll
  for (int i = 0; i < DIMS; ++i)
#pragma unroll
    for (int g = 0; g < HEADS; ++g) acc[i][g] = 0.f;
  __syncthreads();
  const int* pages = page_table + (size_t)slot * max_pages;
  for (int j0 = keys.first; j0 < keys.end; j0 += THREADS) {
    const int j = j0 + tid;
    float s[HEADS];
#pragma unroll
    for (int g = 0; g < HEADS; ++g) s[g] = j < keys.end ? 0.f : -INFINITY;
    if (j < keys.end) {
      const unsigned char* kt = k_pages + ((size_t)pages[j / PAGE] * n_kv + w.head) * TILE;
      const unsigned* sz = reinterpret_cast<const unsigned*>(kt + (size_t)ROW * PAGE) + (j % PAGE) * GROUPS;
      const unsigned* words = reinterpret_cast<const unsigned*>(kt + (size_t)(j % PAGE) * ROW);
      for (int i = 0; i < D / 4; ++i) {   // four numbers of one step and quarter
        const int c = i & 3, step = i >> 2;
        const unsigned word = words[c * UNITS + step / 2] >> (8 * (step & 1));
        const GroupCode gc = unpack_code(sz[step * 16 / BG]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = value_of(word >> (4 * (e >> 1) + 16 * (e & 1)) & 15u, gc);
#pragma unroll
          for (int g = 0; g < HEADS; ++g) s[g] = fmaf(v, qs[g][step * 16 + 4 * c + e], s[g]);
        }
      }
#pragma unroll
      for (int g = 0; g < HEADS; ++g) s[g] *= scale;
    }
#pragma unroll
    for (int g = 0; g < HEADS; ++g) {
      const float m = warp_max(s[g]);
      if (lane == 0) red[warp][g] = m;
    }
    __syncthreads();
    float lower[HEADS], most[HEADS];
#pragma unroll
    for (int g = 0; g < HEADS; ++g) {
      float m = top[g];
#pragma unroll
      for (int x = 0; x < THREADS / 32; ++x) m = fmaxf(m, red[x][g]);
      lower[g] = m == top[g] ? 1.f : expf(top[g] - m);
      most[g] = m;
      s[g] = s[g] == -INFINITY ? 0.f : expf(s[g] - m);
      ps[g][tid] = s[g];
      const float l = warp_sum(s[g]);
      if (lane == 0) total[warp][g] = l;
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < HEADS; ++g)
      if (tid == g) {
        float l = 0.f;
#pragma unroll
        for (int x = 0; x < THREADS / 32; ++x) l += total[x][g];
        sum[g] = sum[g] * lower[g] + l;
        top[g] = most[g];
      }
    const int count = min(THREADS, keys.end - j0);
#pragma unroll
    for (int i = 0; i < DIMS; ++i) {
      const int x = tid + i * THREADS;
#pragma unroll
      for (int g = 0; g < HEADS; ++g) acc[i][g] *= lower[g];
      if (x < D)
        for (int t = 0; t < count; ++t) {
          const int key = j0 + t;
          const unsigned char* vt = v_pages + ((size_t)pages[key / PAGE] * n_kv + w.head) * TILE;
          const unsigned word = *reinterpret_cast<const unsigned short*>(vt + kv4_value_at(key % PAGE, (x & 15) >> 1, x >> 5, UNITS));
          const unsigned sz = reinterpret_cast<const unsigned*>(vt + (size_t)ROW * PAGE)[(key % PAGE) * GROUPS + x / BG];
          const float v = value_of(word >> (8 * ((x >> 4) & 1) + 4 * (x & 1)) & 15u, unpack_code(sz));
#pragma unroll
          for (int g = 0; g < HEADS; ++g) acc[i][g] = fmaf(ps[g][t], v, acc[i][g]);
        }
    }
  }
  __syncthreads();
  for (int g = 0; g < HEADS; ++g) {
    if (g >= heads) break;
#pragma unroll
    for (int i = 0; i < DIMS; ++i) {
      const int x = tid + i * THREADS;
      if (x >= D) continue;
      float a = 0.f;
#pragma unroll
      for (int e = 0; e < HEADS; ++e) a = e == g ? acc[i][e] : a;
      if (splits == 1)
        out[(head0 + g) * D + x] = a / sum[g];
      else
        part_o[((head0 + g) * splits + w.split) * D + x] = a;
    }
    if (splits > 1 && tid == 0) {
      part_ml[((head0 + g) * splits + w.split) * 2] = top[g] * 1.4426950408889634f;   // in powers of two, as the join takes them
      part_ml[((head0 + g) * splits + w.split) * 2 + 1] = sum[g];
    }
  }
}

// A block per (row, query head): the splits' sums joined in their order.  Maxima are powers of two.
template <typename T>
__global__ void __launch_bounds__(THREADS) attn4_join_kernel(const float* part_o, const float* part_ml, const int* __restrict__ tok_slot, T* out, int n_heads, int splits) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const unsigned n = blockIdx.x / n_heads;
  if (tok_slot[n] < 0) return;   // the first launch wrote its zeros
  const size_t h = blockIdx.x;
  float m = -INFINITY, l = 0.f;
  for (int s = 0; s < splits; ++s) m = fmaxf(m, __ldcg(part_ml + (h * splits + s) * 2));
  for (int s = 0; s < splits; ++s) {
    const float ms = __ldcg(part_ml + (h * splits + s) * 2);
    l = fmaf(__ldcg(part_ml + (h * splits + s) * 2 + 1), ms == -INFINITY ? 0.f : exp2f(ms - m), l);   // (a split of NaN alone has no maximum, its sum is NaN)
  }
  for (int x = threadIdx.x; x < D; x += THREADS) {
    float a = 0.f;
    for (int s = 0; s < splits; ++s) {
      const float ms = __ldcg(part_ml + (h * splits + s) * 2);
      a = fmaf(__ldcg(part_o + (h * splits + s) * D + x), ms == -INFINITY ? 0.f : exp2f(ms - m), a);
    }
    out[h * D + x] = from_f32<T>(a / l);
  }
}

struct Args {
  const void *q, *k_pages, *v_pages;
  const int* page_table;
  int max_pages;
  const int *tok_slot, *tok_pos;
  void* out;
  float *part_o, *part_ml;
  int n, n_kv, splits;
  float scale;
  int window;
  cudaStream_t st;
};

template <typename... P, typename... A>
int launch(void (*kern)(P...), unsigned grid, int threads, size_t bytes, int cluster, bool dependent, cudaStream_t st, A... a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
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

template <typename T> int join(const Args& a) {
  return launch(attn4_join_kernel<T>, (unsigned)a.n * a.n_kv * G, THREADS, 0, 1, true, a.st, a.part_o, a.part_ml, a.tok_slot, (T*)a.out, a.n_kv * G, a.splits);
}

int rows_f32(const Args& a) {
  const int rc = launch(attn4_f32_kernel, (unsigned)a.n * a.n_kv * HEAD_TILES * a.splits, THREADS, 0, 1, false, a.st, (const float*)a.q,
                        (const unsigned char*)a.k_pages, (const unsigned char*)a.v_pages, a.page_table, a.max_pages, a.tok_slot, a.tok_pos, (float*)a.out, a.part_o,
                        a.part_ml, a.n_kv, a.splits, a.scale, a.window);
  return rc || a.splits == 1 ? rc : join<float>(a);
}

int rows_bf16(const Args& a) {
  static bool asked = false;
  if (!asked) {   // (asking twice does no harm)
    const cudaError_t e = cudaFuncSetAttribute(attn4_mma_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM);
    if (e != cudaSuccess) return (int)e;
    asked = true;
  }
  const int cluster = a.splits > 1 && a.splits <= 8;
  const int rc = launch(attn4_mma_kernel, (unsigned)a.n * a.n_kv * HEAD_TILES * a.splits, WARPS * 32, SMEM, cluster ? a.splits : 1, false, a.st, (const bf16*)a.q,
                        (const unsigned char*)a.k_pages, (const unsigned char*)a.v_pages, a.page_table, a.max_pages, a.tok_slot, a.tok_pos, (bf16*)a.out, a.part_o,
                        a.part_ml, a.n_kv, a.splits, cluster, a.scale, a.window);
  return rc || a.splits == 1 || cluster ? rc : join<bf16>(a);
}
}  // namespace

DRYFT_API int dryft_attn4_rows(int is_bf16, const void* q, const void* k_pages, const void* v_pages, const int* page_table, int max_pages, const int* tok_slot,
                               const int* tok_pos, void* out, float* part_o, float* part_ml, int n, int n_kv, int splits, float scale, int window, void* stream) {
  if (n <= 0) return 0;
  return (is_bf16 ? rows_bf16 : rows_f32)({q, k_pages, v_pages, page_table, max_pages, tok_slot, tok_pos, out, part_o, part_ml, n, n_kv, splits, scale, window,
                                           (cudaStream_t)stream});
}
DRYFT_API int dryft_attn4_sizes(int which) { return which == 0 ? D : which == 1 ? G : which == 2 ? PAGE : BG; }
