// Attention of query rows over the paged cache held in 4 bits (four_bit.cuh).  Compiled per model with -DDRYFT_HEAD_DIM, -DDRYFT_GROUP (query heads per key
// head), -DDRYFT_PAGE and -DDRYFT_BITS_GROUP (numbers that share a scale).
//
// Row n at position p of slot s sees the keys j with  max(0, p + 1 - window) <= j <= p  (window <= 0: all of them); a row of slot -1 is padding, its output zeros.
// Grid (rows, key heads, splits).  With one split a block writes its output; otherwise it leaves (acc, m, l) and a second launch joins them in the splits' order.
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

struct Span { int first, end; };   // keys of a split: whole tiles of 16, cut at the row's first and last key
__device__ __forceinline__ Span span_of(int pos, int window, int split, int splits) {
  const int lo = window > 0 && pos + 1 > window ? pos + 1 - window : 0;
  const int t0 = lo / 16, tiles = pos / 16 + 1 - t0, per = (tiles + splits - 1) / splits;
  const int a = t0 + min(tiles, split * per), b = t0 + min(tiles, (split + 1) * per);
  return {max(lo, a * 16), min(pos + 1, b * 16)};
}

constexpr int THREADS = 128, DIMS = (D + THREADS - 1) / THREADS;

template <typename T>
__global__ void __launch_bounds__(THREADS) attn4_rows_kernel(const T* __restrict__ q, const unsigned char* __restrict__ k_pages,
                                                             const unsigned char* __restrict__ v_pages, const int* __restrict__ page_table, int max_pages,
                                                             const int* __restrict__ tok_slot, const int* __restrict__ tok_pos, T* out, float* part_o, float* part_ml,
                                                             float scale, int window) {
  __shared__ float qs[G][D], ps[G][THREADS], red[THREADS / 32][G], total[THREADS / 32][G], top[G], sum[G];
  const int n = blockIdx.x, head = blockIdx.y, split = blockIdx.z, splits = gridDim.z, n_kv = gridDim.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slot = tok_slot[n], pos = tok_pos[n];
  T* const o = out + ((size_t)n * n_kv + head) * G * D;
  if (slot < 0) {
    if (split == 0)
      for (int i = tid; i < G * D; i += THREADS) o[i] = from_f32<T>(0.f);
    return;
  }
  const Span keys = span_of(pos, window, split, splits);
  for (int i = tid; i < G * D; i += THREADS) qs[i / D][i % D] = to_f32<T>(q[((size_t)n * n_kv + head) * G * D + i]);
  if (tid < G) {
    top[tid] = -INFINITY;
    sum[tid] = 0.f;
  }
  float acc[DIMS][G];
#pragma unroll
  for (int i = 0; i < DIMS; ++i)
#pragma unroll
    for (int g = 0; g < G; ++g) acc[i][g] = 0.f;
  __syncthreads();
  const int* pages = page_table + (size_t)slot * max_pages;
  for (int j0 = keys.first; j0 < keys.end; j0 += THREADS) {
    const int j = j0 + tid;
    float s[G];
#pragma unroll
    for (int g = 0; g < G; ++g) s[g] = j < keys.end ? 0.f : -INFINITY;
    if (j < keys.end) {
      const unsigned char* kt = k_pages + ((size_t)pages[j / PAGE] * n_kv + head) * TILE;
      const unsigned* sz = reinterpret_cast<const unsigned*>(kt + (size_t)ROW * PAGE) + (j % PAGE) * GROUPS;
      const unsigned* words = reinterpret_cast<const unsigned*>(kt + (size_t)(j % PAGE) * ROW);
      for (int i = 0; i < D / 4; ++i) {   // four numbers of one step and quarter
        const int c = i & 3, step = i >> 2;
        const unsigned w = words[c * UNITS + step / 2] >> (8 * (step & 1));
        const GroupCode gc = unpack_code(sz[step * 16 / BG]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = value_of(w >> (4 * (e >> 1) + 16 * (e & 1)) & 15u, gc);
#pragma unroll
          for (int g = 0; g < G; ++g) s[g] = fmaf(v, qs[g][step * 16 + 4 * c + e], s[g]);
        }
      }
#pragma unroll
      for (int g = 0; g < G; ++g) s[g] *= scale;
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float m = warp_max(s[g]);
      if (lane == 0) red[warp][g] = m;
    }
    __syncthreads();
    float lower[G], most[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float m = top[g];
#pragma unroll
      for (int w = 0; w < THREADS / 32; ++w) m = fmaxf(m, red[w][g]);
      lower[g] = m == top[g] ? 1.f : expf(top[g] - m);
      most[g] = m;
      s[g] = s[g] == -INFINITY ? 0.f : expf(s[g] - m);
      ps[g][tid] = s[g];
      const float l = warp_sum(s[g]);
      if (lane == 0) total[warp][g] = l;
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < G; ++g)
      if (tid == g) {
        float l = 0.f;
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) l += total[w][g];
        sum[g] = sum[g] * lower[g] + l;
        top[g] = most[g];
      }
    const int count = min(THREADS, keys.end - j0);
#pragma unroll
    for (int i = 0; i < DIMS; ++i) {
      const int x = tid + i * THREADS;
#pragma unroll
      for (int g = 0; g < G; ++g) acc[i][g] *= lower[g];
      if (x < D)
        for (int t = 0; t < count; ++t) {
          const int key = j0 + t;
          const unsigned char* vt = v_pages + ((size_t)pages[key / PAGE] * n_kv + head) * TILE;
          const unsigned w = *reinterpret_cast<const unsigned short*>(vt + kv4_value_at(key % PAGE, (x & 15) >> 1, x >> 5, UNITS));
          const unsigned sz = reinterpret_cast<const unsigned*>(vt + (size_t)ROW * PAGE)[(key % PAGE) * GROUPS + x / BG];
          const float v = value_of(w >> (8 * ((x >> 4) & 1) + 4 * (x & 1)) & 15u, unpack_code(sz));
#pragma unroll
          for (int g = 0; g < G; ++g) acc[i][g] = fmaf(ps[g][t], v, acc[i][g]);
        }
    }
  }
  __syncthreads();
  const size_t h0 = ((size_t)n * n_kv + head) * G;
#pragma unroll
  for (int g = 0; g < G; ++g) {
#pragma unroll
    for (int i = 0; i < DIMS; ++i) {
      const int x = tid + i * THREADS;
      if (x >= D) continue;
      if (splits == 1)
        o[g * D + x] = from_f32<T>(acc[i][g] / sum[g]);
      else
        part_o[((h0 + g) * splits + split) * D + x] = acc[i][g];
    }
    if (splits > 1 && tid == 0) {
      part_ml[((h0 + g) * splits + split) * 2] = top[g];
      part_ml[((h0 + g) * splits + split) * 2 + 1] = sum[g];
    }
  }
}

// A block per (row, query head): the splits' sums joined in their order.
template <typename T>
__global__ void __launch_bounds__(THREADS) attn4_join_kernel(const float* part_o, const float* part_ml, const int* __restrict__ tok_slot, T* out, int n_heads, int splits) {
  const int n = blockIdx.x;
  if (tok_slot[n] < 0) return;   // the first launch wrote its zeros
  const size_t h = (size_t)n * n_heads + blockIdx.y;
  float m = -INFINITY, l = 0.f;
  for (int s = 0; s < splits; ++s) m = fmaxf(m, part_ml[(h * splits + s) * 2]);
  for (int s = 0; s < splits; ++s) {
    const float ms = part_ml[(h * splits + s) * 2];
    if (ms != -INFINITY) l += part_ml[(h * splits + s) * 2 + 1] * expf(ms - m);
  }
  for (int x = threadIdx.x; x < D; x += THREADS) {
    float a = 0.f;
    for (int s = 0; s < splits; ++s) {
      const float ms = part_ml[(h * splits + s) * 2];
      if (ms != -INFINITY) a = fmaf(part_o[(h * splits + s) * D + x], expf(ms - m), a);
    }
    out[h * D + x] = from_f32<T>(a / l);
  }
}

template <typename T>
int rows(const void* q, const void* k_pages, const void* v_pages, const int* page_table, int max_pages, const int* tok_slot, const int* tok_pos, void* out, float* part_o,
         float* part_ml, int n, int n_kv, int splits, float scale, int window, cudaStream_t st) {
  attn4_rows_kernel<T><<<dim3(n, n_kv, splits), THREADS, 0, st>>>((const T*)q, (const unsigned char*)k_pages, (const unsigned char*)v_pages, page_table, max_pages,
                                                                 tok_slot, tok_pos, (T*)out, part_o, part_ml, scale, window);
  int rc = launch_status();
  if (rc || splits == 1) return rc;
  attn4_join_kernel<T><<<dim3(n, n_kv * G), THREADS, 0, st>>>(part_o, part_ml, tok_slot, (T*)out, n_kv * G, splits);
  return launch_status();
}
}  // namespace

DRYFT_API int dryft_attn4_rows(int is_bf16, const void* q, const void* k_pages, const void* v_pages, const int* page_table, int max_pages, const int* tok_slot,
                               const int* tok_pos, void* out, float* part_o, float* part_ml, int n, int n_kv, int splits, float scale, int window, void* stream) {
  if (n <= 0) return 0;
  return (is_bf16 ? rows<__nv_bfloat16> : rows<float>)(q, k_pages, v_pages, page_table, max_pages, tok_slot, tok_pos, out, part_o, part_ml, n, n_kv, splits, scale,
                                                      window, (cudaStream_t)stream);
}
DRYFT_API int dryft_attn4_sizes(int which) { return which == 0 ? D : which == 1 ? G : which == 2 ? PAGE : BG; }
