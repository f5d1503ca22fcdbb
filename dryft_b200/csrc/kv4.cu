// Keys and values of new tokens into the paged cache in 4 bits, and pages back as values (four_bit.cuh has the format).
#include "four_bit.cuh"

namespace {
constexpr int WARPS = 4;

// Lowest and highest of a lane's numbers in steps 0 and 1 of its unit, over the group: `near` lanes next to one another hold a unit.
__device__ __forceinline__ void group_range(float (&lo)[2], float (&hi)[2], int near, int group) {
  if (group >= 32) {
    lo[0] = lo[1] = fminf(lo[0], lo[1]);
    hi[0] = hi[1] = fmaxf(hi[0], hi[1]);
  }
  const int lanes = group > 32 ? near * (group / 32) : near;
  for (int o = 1; o < lanes; o <<= 1) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      lo[p] = fminf(lo[p], __shfl_xor_sync(0xffffffffu, lo[p], o));
      hi[p] = fmaxf(hi[p], __shfl_xor_sync(0xffffffffu, hi[p], o));
    }
  }
}
// fminf and fmaxf pass over NaN: a number that is not finite makes the range infinite
__device__ __forceinline__ void widen(float x, float& lo, float& hi) {
  const bool fine = fabsf(x) < INFINITY;
  lo = fminf(lo, fine ? x : -INFINITY);
  hi = fmaxf(hi, fine ? x : INFINITY);
}

// Where a token's rows of one head go.
struct Place { unsigned char *k, *v; int t; };
__device__ __forceinline__ Place place_of(unsigned char* k_pages, unsigned char* v_pages, const int* page_table, int max_pages, int slot, int pos, int page, int n_kv,
                                          int head, size_t tile) {
  const size_t at = ((size_t)page_table[(size_t)slot * max_pages + pos / page] * n_kv + head) * tile;
  return {k_pages + at, v_pages + at, pos % page};
}

// A token's key of one head, by a warp: 4 U lanes of eight dims.
template <typename T>
__device__ __forceinline__ void store_key(const T* row, unsigned char* tile, int t, int d, int group, int page) {
  const int lane = threadIdx.x & 31, u = lane >> 2, c = lane & 3, units = kv4_units(d);
  float x[2][4], lo[2], hi[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    lo[p] = INFINITY;
    hi[p] = -INFINITY;
    const int at = 32 * u + 16 * p + 4 * c;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[p][e] = at < d ? to_f32<T>(row[at + e]) : 0.f;
      if (at < d) widen(x[p][e], lo[p], hi[p]);
    }
  }
  group_range(lo, hi, 4, group);
  unsigned* const scales = reinterpret_cast<unsigned*>(tile + (size_t)kv4_row_bytes(d) * page) + t * (d / group);
  unsigned word = 0;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const GroupCode g = group_code(lo[p], hi[p]);
    const int at = 32 * u + 16 * p;
    if (at < d) {
#pragma unroll
      for (int e = 0; e < 4; ++e) word |= code_of(x[p][e], g) << (8 * p + 4 * (e >> 1) + 16 * (e & 1));
      if (c == 0 && at % group == 0) scales[at / group] = pack_code(g);
    }
  }
  if (u < units) *reinterpret_cast<unsigned*>(tile + (size_t)t * kv4_row_bytes(d) + (c * units + u) * 4) = word;
}

// A token's value of one head, by a warp: 8 U lanes of four dims.
template <typename T>
__device__ __forceinline__ void store_value(const T* row, unsigned char* tile, int t, int d, int group, int page) {
  const int lane = threadIdx.x & 31, units = kv4_units(d);
  unsigned* const scales = reinterpret_cast<unsigned*>(tile + (size_t)kv4_row_bytes(d) * page) + t * (d / group);
  for (int u0 = 0; u0 < units; u0 += 4) {
    const int u = u0 + (lane >> 3), r = lane & 7;
    float x[2][2], lo[2], hi[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      lo[p] = INFINITY;
      hi[p] = -INFINITY;
      const int at = 32 * u + 16 * p + 2 * r;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        x[p][e] = at < d ? to_f32<T>(row[at + e]) : 0.f;
        if (at < d) widen(x[p][e], lo[p], hi[p]);
      }
    }
    group_range(lo, hi, 8, group);
    unsigned bits = 0;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const GroupCode g = group_code(lo[p], hi[p]);
      const int at = 32 * u + 16 * p;
      if (at < d) {
        bits |= (code_of(x[p][0], g) | code_of(x[p][1], g) << 4) << (8 * p);
        if (r == 0 && at % group == 0) scales[at / group] = pack_code(g);
      }
    }
    if (u < units) *reinterpret_cast<unsigned short*>(tile + kv4_value_at(t, r, u, units)) = (unsigned short)bits;
  }
}

// A warp per (token, key head).
template <typename T>
__global__ void __launch_bounds__(WARPS * 32) kv4_store_kernel(const T* k, const T* v, long long stride, const int* __restrict__ tok_slot,
                                                               const int* __restrict__ tok_pos, unsigned char* k_pages, unsigned char* v_pages,
                                                               const int* __restrict__ page_table, int max_pages, int n_kv, int d, int group, int page) {
  const int head = blockIdx.y * WARPS + (threadIdx.x >> 5);
  const long long n = blockIdx.x;
  const int slot = tok_slot[n], pos = tok_pos[n];
  if (slot < 0 || head >= n_kv) return;
  const Place at = place_of(k_pages, v_pages, page_table, max_pages, slot, pos, page, n_kv, head, kv4_tile_bytes(page, d, group));
  store_key(k + n * stride + (size_t)head * d, at.k, at.t, d, group, page);
  store_value(v + n * stride + (size_t)head * d, at.v, at.t, d, group, page);
}

// The same behind a fused projection (rows q | k | v): per-head norm and rotation of queries and keys first, a warp per (token, head).  Formulas and
// rounding points are those of rope_kv.cu.
template <typename T>
__global__ void __launch_bounds__(WARPS * 32) kv4_rope_store_kernel(const T* qkv, int stride, const float* __restrict__ wq, const float* __restrict__ wk,
                                                                    const float* __restrict__ inv_freq, const T* cs_table, const int* __restrict__ tok_slot,
                                                                    const int* __restrict__ tok_pos, T* q_out, unsigned char* k_pages, unsigned char* v_pages,
                                                                    const int* __restrict__ page_table, int max_pages, int n_heads, int n_kv, int d, int rot,
                                                                    int group, int page, float eps, int has_norm) {
  __shared__ T rows[WARPS][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, head = blockIdx.y * WARPS + warp, half = rot >> 1;
  const long long n = blockIdx.x;
  if (head >= n_heads + 2 * n_kv) return;
  const int slot = tok_slot[n], pos = tok_pos[n];
  const T* src = qkv + n * stride + (size_t)head * d;
  T* const q_row = q_out + ((size_t)n * n_heads + head) * d;
  if (slot < 0) {   // padding: a defined query, nothing cached
    if (head < n_heads)
      for (int i = lane; i < d; i += 32) q_row[i] = from_f32<T>(0.f);
    return;
  }
  Place at = {};
  if (head >= n_heads) at = place_of(k_pages, v_pages, page_table, max_pages, slot, pos, page, n_kv, (head - n_heads) % n_kv, kv4_tile_bytes(page, d, group));
  if (head >= n_heads + n_kv) return store_value(src, at.v, at.t, d, group, page);
  T* const row = rows[warp];
  const float* w = head < n_heads ? wq : wk;
  float x[8], ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = lane + 32 * i < d ? to_f32<T>(src[lane + 32 * i]) : 0.f;
    ss = fmaf(x[i], x[i], ss);
  }
  const float inv = has_norm ? rsqrtf(warp_sum(ss) / (float)d + eps) : 1.f;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (lane + 32 * i < d) row[lane + 32 * i] = from_f32<T>(has_norm ? rnd<T>(x[i] * inv) * w[lane + 32 * i] : x[i]);
  __syncwarp();
  for (int j = lane; j < half; j += 32) {
    float sn, cs;
    if (cs_table != nullptr) {
      cs = to_f32<T>(cs_table[n * rot + j]);
      sn = to_f32<T>(cs_table[n * rot + half + j]);
    } else {
      sincosf((float)pos * inv_freq[j], &sn, &cs);
      cs = rnd<T>(cs);
      sn = rnd<T>(sn);
    }
    const float a = to_f32<T>(row[j]), b = to_f32<T>(row[j + half]);   // the products and their sum are rounded one by one
    row[j] = from_f32<T>(__fadd_rn(rnd<T>(__fmul_rn(a, cs)), -rnd<T>(__fmul_rn(b, sn))));
    row[j + half] = from_f32<T>(__fadd_rn(rnd<T>(__fmul_rn(b, cs)), rnd<T>(__fmul_rn(a, sn))));
  }
  __syncwarp();
  if (head >= n_heads) return store_key(row, at.k, at.t, d, group, page);
  for (int i = lane; i < d; i += 32) q_row[i] = row[i];
}

// Blocks per (sequence, key head), each every gridDim.x-th page of it: the page's tokens as values, those behind the sequence's end as zeros.  Pages before the
// first key that the step's first token of the sequence sees (window <= 0: every key) are left alone: they may be another sequence's by now.
template <typename T>
__global__ void __launch_bounds__(256) kv4_expand_kernel(const unsigned char* k_pages, const unsigned char* v_pages, const int* __restrict__ page_table,
                                                         int max_pages, const int* __restrict__ cu_q, const int* __restrict__ seq_slot,
                                                         const int* __restrict__ tok_pos, T* k_out, T* v_out, int n_kv, int d, int group, int page, int window) {
  const int b = blockIdx.z, head = blockIdx.y, slot = seq_slot[b];
  if (slot < 0 || cu_q[b + 1] <= cu_q[b]) return;
  const int end = tok_pos[cu_q[b + 1] - 1] + 1, first = window > 0 ? max(0, tok_pos[cu_q[b]] + 1 - window) / page : 0;
  const int units = kv4_units(d), groups = d / group;
  for (int p = first + blockIdx.x; p * page < end; p += gridDim.x) {
    const size_t at_page = (size_t)page_table[(size_t)slot * max_pages + p] * n_kv + head;
    const unsigned char *kt = k_pages + at_page * kv4_tile_bytes(page, d, group), *vt = v_pages + at_page * kv4_tile_bytes(page, d, group);
    const unsigned *ks = reinterpret_cast<const unsigned*>(kt + (size_t)kv4_row_bytes(d) * page), *vs = reinterpret_cast<const unsigned*>(vt + (size_t)kv4_row_bytes(d) * page);
    T *ko = k_out + at_page * page * d, *vo = v_out + at_page * page * d;
    for (int i = threadIdx.x; i < page * d; i += blockDim.x) {
      const int t = i / d, x = i % d, u = x / 32, h = (x >> 4) & 1;
      float kv = 0.f, vv = 0.f;
      if (p * page + t < end) {
        const int c = (x & 15) >> 2, e = x & 3, r = (x & 15) >> 1;
        const unsigned kw = *reinterpret_cast<const unsigned*>(kt + (size_t)t * kv4_row_bytes(d) + (c * units + u) * 4);
        const unsigned vw = *reinterpret_cast<const unsigned short*>(vt + kv4_value_at(t, r, u, units));
        kv = value_of(kw >> (8 * h + 4 * (e >> 1) + 16 * (e & 1)) & 15u, unpack_code(ks[t * groups + x / group]));
        vv = value_of(vw >> (8 * h + 4 * (x & 1)) & 15u, unpack_code(vs[t * groups + x / group]));
      }
      ko[i] = from_f32<T>(kv);
      vo[i] = from_f32<T>(vv);
    }
  }
}

template <typename T>
int store(const void* k, const void* v, long long stride, const int* tok_slot, const int* tok_pos, void* k_pages, void* v_pages, const int* page_table,
          int max_pages, int n, int n_kv, int d, int group, int page, cudaStream_t st) {
  kv4_store_kernel<T><<<dim3(n, (n_kv + WARPS - 1) / WARPS), WARPS * 32, 0, st>>>((const T*)k, (const T*)v, stride, tok_slot, tok_pos, (unsigned char*)k_pages,
                                                                                 (unsigned char*)v_pages, page_table, max_pages, n_kv, d, group, page);
  return launch_status();
}
template <typename T>
int expand(const void* k_pages, const void* v_pages, const int* page_table, int max_pages, const int* cu_q, const int* seq_slot, const int* tok_pos, void* k_out,
           void* v_out, int n_seqs, int pages, int n_kv, int d, int group, int page, int window, cudaStream_t st) {
  const int blocks = 4096 / (n_kv * n_seqs) + 1;   // of a sequence and head: a few thousand blocks, however long the sequences may be
  kv4_expand_kernel<T><<<dim3(blocks < pages ? blocks : pages, n_kv, n_seqs), 256, 0, st>>>((const unsigned char*)k_pages, (const unsigned char*)v_pages, page_table, max_pages, cu_q,
                                                                  seq_slot, tok_pos, (T*)k_out, (T*)v_out, n_kv, d, group, page, window);
  return launch_status();
}
template <typename T>
int rope_store(const void* qkv, int stride, const float* wq, const float* wk, const float* inv_freq, const void* cs_table, const int* tok_slot, const int* tok_pos,
               void* q_out, void* k_pages, void* v_pages, const int* page_table, int max_pages, int n, int n_heads, int n_kv, int d, int rot, int group, int page,
               float eps, int has_norm, cudaStream_t st) {
  kv4_rope_store_kernel<T><<<dim3(n, (n_heads + 2 * n_kv + WARPS - 1) / WARPS), WARPS * 32, 0, st>>>(
      (const T*)qkv, stride, wq, wk, inv_freq, (const T*)cs_table, tok_slot, tok_pos, (T*)q_out, (unsigned char*)k_pages, (unsigned char*)v_pages, page_table,
      max_pages, n_heads, n_kv, d, rot, group, page, eps, has_norm);
  return launch_status();
}
}  // namespace

DRYFT_API int dryft_kv4_rope_store(int is_bf16, const void* qkv, int stride, const float* wq, const float* wk, const float* inv_freq, const void* cs_table,
                                   const int* tok_slot, const int* tok_pos, void* q_out, void* k_pages, void* v_pages, const int* page_table, int max_pages, int n,
                                   int n_heads, int n_kv, int d, int rot, int group, int page, float eps, int has_norm, void* stream) {
  if (n <= 0) return 0;
  return (is_bf16 ? rope_store<__nv_bfloat16> : rope_store<float>)(qkv, stride, wq, wk, inv_freq, cs_table, tok_slot, tok_pos, q_out, k_pages, v_pages, page_table,
                                                                  max_pages, n, n_heads, n_kv, d, rot, group, page, eps, has_norm, (cudaStream_t)stream);
}

DRYFT_API int dryft_kv4_store(int is_bf16, const void* k, const void* v, long long stride, const int* tok_slot, const int* tok_pos, void* k_pages, void* v_pages,
                              const int* page_table, int max_pages, int n, int n_kv, int d, int group, int page, void* stream) {
  if (n <= 0) return 0;
  return (is_bf16 ? store<__nv_bfloat16> : store<float>)(k, v, stride, tok_slot, tok_pos, k_pages, v_pages, page_table, max_pages, n, n_kv, d, group, page,
                                                        (cudaStream_t)stream);
}

DRYFT_API int dryft_kv4_expand(int is_bf16, const void* k_pages, const void* v_pages, const int* page_table, int max_pages, const int* cu_q, const int* seq_slot,
                               const int* tok_pos, void* k_out, void* v_out, int n_seqs, int pages, int n_kv, int d, int group, int page, int window,
                               void* stream) {
  if (n_seqs <= 0 || pages <= 0) return 0;
  return (is_bf16 ? expand<__nv_bfloat16> : expand<float>)(k_pages, v_pages, page_table, max_pages, cu_q, seq_slot, tok_pos, k_out, v_out, n_seqs, pages, n_kv, d,
                                                          group, page, window, (cudaStream_t)stream);
}
