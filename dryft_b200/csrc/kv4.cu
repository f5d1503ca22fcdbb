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

// A warp per (token, key head): the key's row by 4 U lanes of eight dims, the value's by 8 U lanes of four.
template <typename T>
__global__ void __launch_bounds__(WARPS * 32) kv4_store_kernel(const T* k, const T* v, long long stride, const int* __restrict__ tok_slot,
                                                               const int* __restrict__ tok_pos, unsigned char* k_pages, unsigned char* v_pages,
                                                               const int* __restrict__ page_table, int max_pages, int n_kv, int d, int group, int page) {
  const int lane = threadIdx.x & 31, head = blockIdx.y * WARPS + (threadIdx.x >> 5);
  const long long n = blockIdx.x;
  const int slot = tok_slot[n], pos = tok_pos[n];
  if (slot < 0 || head >= n_kv) return;
  const int units = kv4_units(d), groups = d / group, t = pos % page;
  const size_t tile = ((size_t)page_table[(size_t)slot * max_pages + pos / page] * n_kv + head) * kv4_tile_bytes(page, d, group);
  const size_t codes = (size_t)kv4_row_bytes(d) * page;
  {
    const T* row = k + n * stride + (size_t)head * d;
    const int u = lane >> 2, c = lane & 3;
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
    unsigned word = 0;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const GroupCode g = group_code(lo[p], hi[p]);
      const int at = 32 * u + 16 * p;
      if (at < d) {
#pragma unroll
        for (int e = 0; e < 4; ++e) word |= code_of(x[p][e], g) << (8 * p + 4 * (e >> 1) + 16 * (e & 1));
        if (c == 0 && at % group == 0) *reinterpret_cast<unsigned*>(k_pages + tile + codes + ((size_t)t * groups + at / group) * 4) = pack_code(g);
      }
    }
    if (u < units) *reinterpret_cast<unsigned*>(k_pages + tile + (size_t)t * kv4_row_bytes(d) + (c * units + u) * 4) = word;
  }
  const T* row = v + n * stride + (size_t)head * d;
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
        if (r == 0 && at % group == 0) *reinterpret_cast<unsigned*>(v_pages + tile + codes + ((size_t)t * groups + at / group) * 4) = pack_code(g);
      }
    }
    if (u < units) *reinterpret_cast<unsigned short*>(v_pages + tile + kv4_value_at(t, r, u, units)) = (unsigned short)bits;
  }
}

// A block per (page of a sequence, key head): the page's tokens as values, those behind the sequence's end as zeros.  Pages before the first key that the
// step's first token of the sequence sees (window <= 0: every key) are left alone: they may be another sequence's by now.
template <typename T>
__global__ void __launch_bounds__(256) kv4_expand_kernel(const unsigned char* k_pages, const unsigned char* v_pages, const int* __restrict__ page_table,
                                                         int max_pages, const int* __restrict__ cu_q, const int* __restrict__ seq_slot,
                                                         const int* __restrict__ tok_pos, T* k_out, T* v_out, int n_kv, int d, int group, int page, int window) {
  const int b = blockIdx.z, head = blockIdx.y, slot = seq_slot[b];
  if (slot < 0 || cu_q[b + 1] <= cu_q[b]) return;
  const int left = tok_pos[cu_q[b + 1] - 1] + 1 - (int)blockIdx.x * page;   // tokens from this page's first one on
  if (left <= 0 || (window > 0 && ((int)blockIdx.x + 1) * page <= tok_pos[cu_q[b]] + 1 - window)) return;
  const size_t at_page = (size_t)page_table[(size_t)slot * max_pages + blockIdx.x] * n_kv + head;
  const int units = kv4_units(d), groups = d / group;
  const unsigned char *kt = k_pages + at_page * kv4_tile_bytes(page, d, group), *vt = v_pages + at_page * kv4_tile_bytes(page, d, group);
  const unsigned *ks = reinterpret_cast<const unsigned*>(kt + (size_t)kv4_row_bytes(d) * page), *vs = reinterpret_cast<const unsigned*>(vt + (size_t)kv4_row_bytes(d) * page);
  T *ko = k_out + at_page * page * d, *vo = v_out + at_page * page * d;
  for (int i = threadIdx.x; i < page * d; i += blockDim.x) {
    const int t = i / d, x = i % d, u = x / 32, p = (x >> 4) & 1;
    float kv = 0.f, vv = 0.f;
    if (t < left) {
      const int c = (x & 15) >> 2, e = x & 3, r = (x & 15) >> 1;
      const unsigned kw = *reinterpret_cast<const unsigned*>(kt + (size_t)t * kv4_row_bytes(d) + (c * units + u) * 4);
      const unsigned vw = *reinterpret_cast<const unsigned short*>(vt + kv4_value_at(t, r, u, units));
      kv = value_of(kw >> (8 * p + 4 * (e >> 1) + 16 * (e & 1)) & 15u, unpack_code(ks[t * groups + x / group]));
      vv = value_of(vw >> (8 * p + 4 * (x & 1)) & 15u, unpack_code(vs[t * groups + x / group]));
    }
    ko[i] = from_f32<T>(kv);
    vo[i] = from_f32<T>(vv);
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
  kv4_expand_kernel<T><<<dim3(pages, n_kv, n_seqs), 256, 0, st>>>((const unsigned char*)k_pages, (const unsigned char*)v_pages, page_table, max_pages, cu_q,
                                                                  seq_slot, tok_pos, (T*)k_out, (T*)v_out, n_kv, d, group, page, window);
  return launch_status();
}
}  // namespace

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
