// Keys and values of new tokens into the paged cache in 4 bits, and pages back as values (four_bit.cuh has the format).
#include "four_bit.cuh"

namespace {
constexpr int WARPS = 4;

// The range of a lane's numbers.  fminf and fmaxf pass over NaN, so whether there was one is kept beside them: x * 0 is NaN for it (and for an infinity).
struct Range {
  float lo = INFINITY, hi = -INFINITY, not_finite = 0.f;
  __device__ __forceinline__ void add(float x) {
    lo = fminf(lo, x);
    hi = fmaxf(hi, x);
    not_finite = fmaf(x, 0.f, not_finite);
  }
  __device__ __forceinline__ void close() {   // a range with such a number is everything
    lo = not_finite == 0.f ? lo : -INFINITY;
    hi = not_finite == 0.f ? hi : INFINITY;
  }
};

// Two numbers that follow one another, as they lie in memory, and the range of many such, which lanes can share.  Of bfloat16 numbers both ends are kept for two
// numbers at once, by instructions that hand a NaN on, and (upper end, lower end with its sign turned) are shared as one word.
__device__ __forceinline__ unsigned min2(unsigned a, unsigned b) {
  unsigned r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ unsigned max2(unsigned a, unsigned b) {
  unsigned r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <typename T> struct Pairs;
template <> struct Pairs<float> {
  typedef float2 two;
  typedef float4 four;
  static __device__ __forceinline__ two half(four v, int i) { return i ? make_float2(v.z, v.w) : make_float2(v.x, v.y); }
  Range r;
  static __device__ __forceinline__ float first(two v) { return v.x; }
  static __device__ __forceinline__ float second(two v) { return v.y; }
  __device__ __forceinline__ void add(two v) {
    r.add(v.x);
    r.add(v.y);
  }
  __device__ __forceinline__ void close() { r.close(); }
  __device__ __forceinline__ void share(int apart) {
    r.lo = fminf(r.lo, __shfl_xor_sync(0xffffffffu, r.lo, apart));
    r.hi = fmaxf(r.hi, __shfl_xor_sync(0xffffffffu, r.hi, apart));
  }
  __device__ __forceinline__ float2 ends() const { return make_float2(r.lo, r.hi); }
};
template <> struct Pairs<__nv_bfloat16> {
  typedef unsigned two;
  typedef uint2 four;
  static __device__ __forceinline__ two half(four v, int i) { return i ? v.y : v.x; }
  unsigned lo = 0x7f807f80u, hi = 0xff80ff80u;   // infinities; after `close`, hi is the word to share
  static __device__ __forceinline__ float first(two v) { return __uint_as_float(v << 16); }
  static __device__ __forceinline__ float second(two v) { return __uint_as_float(v & 0xffff0000u); }
  __device__ __forceinline__ void add(two v) {
    lo = min2(lo, v);
    hi = max2(hi, v);
  }
  __device__ __forceinline__ void close() {
    const unsigned l = min2(lo, __byte_perm(lo, lo, 0x1032)), h = max2(hi, __byte_perm(hi, hi, 0x1032));
    hi = __byte_perm(h, l ^ 0x80008000u, 0x5410);
  }
  __device__ __forceinline__ void share(int apart) { hi = max2(hi, __shfl_xor_sync(0xffffffffu, hi, apart)); }
  __device__ __forceinline__ float2 ends() const {   // a range with an infinity or a NaN is everything
    const float h = first(hi), l = -second(hi);
    return h < INFINITY && l > -INFINITY ? make_float2(l, h) : make_float2(-INFINITY, INFINITY);
  }
};

// The codes of a group's numbers without a division each.  The definition (`code_of`) rounds t / s, t = x - z, and then t / s + 7.5, to 32 bits, and that to a whole
// number.  With j the whole number nearest to t times 1 / s and e = t - j s (j s is exact, so e is rounded once, and 0 where t is a multiple of s), j + e / s is
// t / s up to 2^-22, and exact where e is 0 -- which is every tie.  Only where e is neither 0 nor beyond 10^-5 s could those roundings decide: then the group's numbers
// are divided after all.  (Three numbers in a thousand are ties where x is bfloat16.)
constexpr float ROUND = 12582912.f;   // 1.5 * 2^23: adding it rounds to whole numbers, ties to even
struct Coder {
  GroupCode g;
  float inv;
  unsigned closest = ~0u;   // twice the bits of the least |e| that is not 0, less 1 (which drops the sign, and makes 0 the largest)
  __device__ __forceinline__ Coder(float lo, float hi) : g(group_code(lo, hi)), inv(inverse(g.s)) {}
  __device__ __forceinline__ Coder(GroupCode code, float inverse) : g(code), inv(inverse) {}
  static __device__ __forceinline__ float inverse(float s) { return s > 1e-36f ? __fdividef(1.f, s) : 0.f; }   // (its last bits do not matter)
  // `word` + code << shift + ROUND's bits << shift, which the caller takes out (`round_bits`)
  __device__ __forceinline__ unsigned add(unsigned word, float x, int shift) {
    const float t = __fadd_rn(x, -g.z), j = __fadd_rn(__fadd_rn(__fmul_rn(t, inv), ROUND), -ROUND), e = fmaf(-j, g.s, t);
    closest = min(closest, 2u * __float_as_uint(e) - 1u);
    const float y = __fadd_rn(fmaf(e, inv, j), 7.5f);
    return word + (__float_as_uint(__fadd_rn(fminf(fmaxf(y, 0.f), 15.f), ROUND)) << shift);
  }
  __device__ __forceinline__ bool undecided() const { return closest < 2u * __float_as_uint(g.s * 1e-5f) || (inv == 0.f && g.s > 0.f); }
};
__device__ __forceinline__ constexpr unsigned round_bits(unsigned places) {   // ROUND's bits at every nibble of `places` (a bit each)
  unsigned sum = 0;
  for (int i = 0; i < 8; ++i)
    if (places >> i & 1) sum += 0x4b400000u << (4 * i);
  return sum;
}

// Four consecutive numbers of a row in shared memory, on a boundary of as many
template <typename T> __device__ __forceinline__ void load_four(float (&x)[4], const T* p) {
  if constexpr (sizeof(T) == 4) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const unsigned v = reinterpret_cast<const unsigned*>(p)[i / 2];
      x[i] = __uint_as_float(v << 16);
      x[i + 1] = __uint_as_float(v & 0xffff0000u);
    }
  }
}
// What the launch before wrote: a number, or two on a boundary of as many.  DEPENDENT: past L1 (`ld_prev`)
template <bool DEPENDENT> __device__ __forceinline__ float prev(const float* p) { return DEPENDENT ? ld_prev(p) : *p; }
template <bool DEPENDENT> __device__ __forceinline__ float prev(const __nv_bfloat16* p) { return DEPENDENT ? ld_prev_bf16(p) : __bfloat162float(*p); }
template <bool DEPENDENT, typename T> __device__ __forceinline__ void prev_two(float (&x)[2], const T* p) {
  if constexpr (sizeof(T) == 4) {
    const float2* const at = reinterpret_cast<const float2*>(p);
    const float2 v = DEPENDENT ? ld_prev(at) : *at;
    x[0] = v.x; x[1] = v.y;
  } else {
    const unsigned* const at = reinterpret_cast<const unsigned*>(p);
    const unsigned v = DEPENDENT ? ld_prev(at) : *at;
    x[0] = __uint_as_float(v << 16);
    x[1] = __uint_as_float(v & 0xffff0000u);
  }
}

// Where a token's rows of one head go.
struct Place { unsigned char *k, *v; int t; };
__device__ __forceinline__ Place place_of(unsigned char* k_pages, unsigned char* v_pages, const int* page_table, int max_pages, int slot, int pos, int page, int n_kv,
                                          int head, size_t tile) {
  const int whole = page == 64 ? pos >> 6 : pos / page;
  const size_t at = ((size_t)page_table[(size_t)slot * max_pages + whole] * n_kv + head) * tile;
  return {k_pages + at, v_pages + at, pos - whole * page};
}

// The range of a lane's numbers, which `near` lanes at a distance of `apart` share, over the group: of the two steps of a unit, and of further lanes for groups
// of more than a unit.
__device__ __forceinline__ void group_range(float (&lo)[2], float (&hi)[2], int near, int apart, int group) {
  if (group >= 32) {
    lo[0] = lo[1] = fminf(lo[0], lo[1]);
    hi[0] = hi[1] = fmaxf(hi[0], hi[1]);
  }
  const int lanes = group > 32 ? near * (group / 32) : near;
  for (int o = 1; o < lanes; o <<= 1) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      lo[p] = fminf(lo[p], __shfl_xor_sync(0xffffffffu, lo[p], o * apart));
      hi[p] = fmaxf(hi[p], __shfl_xor_sync(0xffffffffu, hi[p], o * apart));
    }
  }
}

// A token's key of one head: 4 U lanes of eight dims, `part` this lane's number among them (of as many as the next power of two).  Every lane of the warp
// calls this; `have` false: for nothing.
template <typename T> __device__ __forceinline__ void load_key(float (&x)[2][4], const T* row, int part, int d, bool have) {
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int at = 32 * (part >> 2) + 16 * p + 4 * (part & 3);
    x[p][0] = x[p][1] = x[p][2] = x[p][3] = 0.f;
    if (have && at < d) load_four<T>(x[p], row + at);
  }
}
template <int GS> __device__ __forceinline__ void store_key(const float (&x)[2][4], bool have, int part, unsigned char* tile, int t, int d, int page) {
  constexpr int group = 16 * GS;
  const int u = part >> 2, c = part & 3, units = kv4_units(d);
  float lo[2], hi[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    Range range;
    if (have && 32 * u + 16 * p < d) {
#pragma unroll
      for (int e = 0; e < 4; ++e) range.add(x[p][e]);
    }
    range.close();
    lo[p] = range.lo;
    hi[p] = range.hi;
  }
  group_range(lo, hi, 4, 1, group);
  if (!have || u >= units) return;
  unsigned* const scales = reinterpret_cast<unsigned*>(tile + (size_t)kv4_row_bytes(d) * page) + t * (d / group);
  unsigned word = 0;
  constexpr int STEPS = GS == 1 ? 1 : 2;   // of the unit that share a scale
#pragma unroll
  for (int p = 0; p < 2; p += STEPS) {
    const int at = 32 * u + 16 * p;
    if (at >= d) continue;
    Coder code(lo[p], hi[p]);
    unsigned steps = 0u - (STEPS == 2 ? round_bits(0xff) : p ? round_bits(0xcc) : round_bits(0x33));
    const auto place = [](int q, int e) { return 8 * q + 4 * (e >> 1) + 16 * (e & 1); };
#pragma unroll
    for (int q = p; q < p + STEPS; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) steps = code.add(steps, x[q][e], place(q, e));
    if (code.undecided()) {
      steps = 0;
#pragma unroll
      for (int q = p; q < p + STEPS; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) steps |= code_of(x[q][e], code.g) << place(q, e);
    }
    word |= steps;
    if (c == 0 && at % group == 0) scales[at / group] = pack_code(code.g);
  }
  *reinterpret_cast<unsigned*>(tile + (size_t)t * kv4_row_bytes(d) + (c * units + u) * 4) = word;
}

// A token's value of one head, by a warp: 8 U lanes of four dims.
template <bool DEPENDENT, typename T>
__device__ __forceinline__ void store_value(const T* row, unsigned char* tile, int t, int d, int group, int page) {
  const int lane = threadIdx.x & 31, units = kv4_units(d);
  unsigned* const scales = reinterpret_cast<unsigned*>(tile + (size_t)kv4_row_bytes(d) * page) + t * (d / group);
  for (int u0 = 0; u0 < units; u0 += 4) {
    const int u = u0 + (lane >> 3), r = lane & 7;
    float x[2][2] = {}, lo[2], hi[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      Range range;
      const int at = 32 * u + 16 * p + 2 * r;
      if (at < d) {
        prev_two<DEPENDENT>(x[p], row + at);
        range.add(x[p][0]);
        range.add(x[p][1]);
      }
      range.close();
      lo[p] = range.lo;
      hi[p] = range.hi;
    }
    group_range(lo, hi, 8, 1, group);
    if (u >= units) continue;
    unsigned bits = 0;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int at = 32 * u + 16 * p;
      if (at < d) {
        Coder code(lo[p], hi[p]);
        unsigned both = code.add(code.add(0u - round_bits(3), x[p][0], 0), x[p][1], 4);
        if (code.undecided()) both = code_of(x[p][0], code.g) | code_of(x[p][1], code.g) << 4;
        bits |= both << (8 * p);
        if (r == 0 && at % group == 0) scales[at / group] = pack_code(code.g);
      }
    }
    *reinterpret_cast<unsigned short*>(tile + kv4_value_at(t, r, u, units)) = (unsigned short)bits;
  }
}

// Up to 16 tokens that follow one another in a tile of 16, tile places i0 to i0 + count - 1: the UB units from u0 on of their values of one head, by a warp.
// Lane (r, c) takes what it would read, four tokens; GS: steps of 16 dims that share a scale.
template <typename T, int UB, int GS>
__device__ __forceinline__ void store_tile_values(const T* rows, long long stride, unsigned char* tile, int t0, int i0, int count, int u0, int d, int page) {
  constexpr int NG = 2 * UB / GS;   // groups of UB units
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3, units = kv4_units(d), groups = d / (16 * GS);
  unsigned* const scales = reinterpret_cast<unsigned*>(tile + (size_t)kv4_row_bytes(d) * page);
  unsigned bits[UB][2];
#pragma unroll
  for (int b = 0; b < UB; ++b) bits[b][0] = bits[b][1] = 0;
  const bool all = 2 * c >= i0 && 2 * c + 9 < i0 + count;   // the lane's four tokens are written together
  typedef Pairs<T> P;
  typename P::two x[4][2 * UB] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int s = 0; s < 2 * UB; ++s) {
      const int k = 2 * c + (i & 1) + 8 * (i >> 1), at = 32 * u0 + 16 * s + 2 * r;
      if (k >= i0 && k < i0 + count && at < d) x[i][s] = *reinterpret_cast<const typename P::two*>(rows + (k - i0) * stride + at);
    }
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    // the ranges of the lane's four tokens, over the lanes of the group; lane row r & 3 works out one token's scale for all
    float lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      P range;
#pragma unroll
      for (int s = g * GS; s < (g + 1) * GS; ++s)
        if (32 * u0 + 16 * s < d) range.add(x[i][s]);
      range.close();
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) range.share(o);
      const float2 ends = range.ends();
      if ((r & 3) == i) {
        lo = ends.x;
        hi = ends.y;
      }
    }
    const GroupCode one = group_code(lo, hi);
    const unsigned packed = pack_code(one);
    const float inverse = Coder::inverse(one.s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = 2 * c + (i & 1) + 8 * (i >> 1);
      const unsigned sz = __shfl_sync(0xffffffffu, packed, i * 4 + c);
      Coder code(unpack_code(sz), __shfl_sync(0xffffffffu, inverse, i * 4 + c));
      if (k < i0 || k >= i0 + count || 32 * u0 + 16 * GS * g >= d) continue;
      unsigned half[(GS + 1) / 2] = {};   // the 16 bits of each unit of the group (or of one step of it)
#pragma unroll
      for (int s = g * GS; s < (g + 1) * GS; ++s) {
        unsigned& h = half[s / 2 - g * GS / 2];
        h = code.add(code.add(h - round_bits(s & 1 ? 0xc : 0x3), P::first(x[i][s]), 8 * (s & 1)), P::second(x[i][s]), 8 * (s & 1) + 4);
      }
      if (code.undecided()) {
#pragma unroll
        for (int s = g * GS; s < (g + 1) * GS; ++s) {
          unsigned& h = half[s / 2 - g * GS / 2];
          if (GS == 1 || (s & 1) == 0) h = 0;
          h |= (code_of(P::first(x[i][s]), code.g) | code_of(P::second(x[i][s]), code.g) << 4) << (8 * (s & 1));
        }
      }
#pragma unroll
      for (int s = g * GS; s < (g + 1) * GS; s += 2) bits[s / 2][i >> 1] |= half[s / 2 - g * GS / 2] << (16 * (i & 1));
      if (r == 0) scales[(t0 + k) * groups + (32 * u0) / (16 * GS) + g] = sz;
    }
  }
  if (!all) {   // ... or 16 bits each
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = 2 * c + (i & 1) + 8 * (i >> 1);
      if (k < i0 || k >= i0 + count) continue;
#pragma unroll
      for (int b = 0; b < UB; ++b)
        *reinterpret_cast<unsigned short*>(tile + kv4_value_at(t0 + k, r, u0 + b, units)) = (unsigned short)(bits[b][i >> 1] >> (16 * (i & 1)));
    }
  }
  if (all) {
#pragma unroll
    for (int b = 0; b < UB; ++b) *reinterpret_cast<uint2*>(tile + kv4_value_at(t0 + 2 * c, r, u0 + b, units)) = make_uint2(bits[b][0], bits[b][1]);
  }
}

// KEY_TOKENS tokens' keys of one head, by each thread of the lanes that share a token: four dims of each step of a unit.  Quarter c of a unit works out the scale of
// token c for all of them.
constexpr int KEY_TOKENS = 4;
template <typename T, int GS>
__device__ __forceinline__ void store_keys(const typename Pairs<T>::two (&x)[KEY_TOKENS][2][2], const int (&slot)[KEY_TOKENS], const int (&pos)[KEY_TOKENS], int part,
                                           unsigned char* k_pages, unsigned char* v_pages, const int* page_table, int max_pages, int n_kv, int head, int d, int page,
                                           size_t tile_bytes) {
  typedef Pairs<T> P;
  constexpr int GROUP = 16 * GS, STEPS = GS == 1 ? 1 : 2, RANGES = 2 / STEPS;   // steps of the unit that share a scale; scales of a unit
  const int lane = threadIdx.x & 31, u = part >> 2, c = part & 3, units = kv4_units(d);
  unsigned packed[RANGES];
  float inverse[RANGES];
#pragma unroll
  for (int p = 0; p < RANGES; ++p) {
    float2 ends = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < KEY_TOKENS; ++i) {
      P range;
#pragma unroll
      for (int q = p * STEPS; q < (p + 1) * STEPS; ++q)
        if (32 * u + 16 * q < d) {
          range.add(x[i][q][0]);
          range.add(x[i][q][1]);
        }
      range.close();
#pragma unroll
      for (int o = 1; o < (GS > 2 ? 2 * GS : 4); o <<= 1) range.share(o);
      const float2 e = range.ends();
      if (c == i) ends = e;
    }
    const GroupCode one = group_code(ends.x, ends.y);
    packed[p] = pack_code(one);
    inverse[p] = Coder::inverse(one.s);
  }
#pragma unroll
  for (int i = 0; i < KEY_TOKENS; ++i) {
    unsigned sz[RANGES];
    float inv[RANGES];
#pragma unroll
    for (int p = 0; p < RANGES; ++p) {
      sz[p] = __shfl_sync(0xffffffffu, packed[p], (lane & ~3) + i);
      inv[p] = __shfl_sync(0xffffffffu, inverse[p], (lane & ~3) + i);
    }
    if (slot[i] < 0 || u >= units) continue;
    const Place at = place_of(k_pages, v_pages, page_table, max_pages, slot[i], pos[i], page, n_kv, head, tile_bytes);
    unsigned word = 0;
#pragma unroll
    for (int p = 0; p < RANGES; ++p) {
      const int dim = 32 * u + 16 * p * STEPS;
      if (dim >= d) continue;
      Coder code(unpack_code(sz[p]), inv[p]);
      unsigned steps = 0u - (STEPS == 2 ? round_bits(0xff) : p ? round_bits(0xcc) : round_bits(0x33));
      const auto place = [](int q, int e) { return 8 * q + 4 * (e >> 1) + 16 * (e & 1); };
#pragma unroll
      for (int q = p * STEPS; q < (p + 1) * STEPS; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) steps = code.add(steps, e & 1 ? P::second(x[i][q][e >> 1]) : P::first(x[i][q][e >> 1]), place(q, e));
      if (code.undecided()) {
        steps = 0;
#pragma unroll
        for (int q = p * STEPS; q < (p + 1) * STEPS; ++q)
#pragma unroll
          for (int e = 0; e < 4; ++e) steps |= code_of(e & 1 ? P::second(x[i][q][e >> 1]) : P::first(x[i][q][e >> 1]), code.g) << place(q, e);
      }
      word |= steps;
      if (c == 0 && dim % GROUP == 0) reinterpret_cast<unsigned*>(at.k + (size_t)kv4_row_bytes(d) * page)[at.t * (d / GROUP) + dim / GROUP] = sz[p];
    }
    *reinterpret_cast<unsigned*>(at.k + (size_t)at.t * kv4_row_bytes(d) + (c * units + u) * 4) = word;
  }
}

// Bound by issue, 81% of its slots: 31 instructions a number, 15 of them for its code.  12,829 tokens, eight key heads of 128: 30.7 us, 2,200 GB/s (with
// each number's range and every lane's scale for itself 37.6); eight tokens 2.5 us, a launch.
// Grid (blocks, key heads).  Keys by the first `key_blocks` blocks, values by the others.
// Keys: as many lanes for a token as a row has words of eight dims, or the next power of two; a thread takes KEY_TOKENS tokens.
// Values: a warp per `span` consecutive tokens of the launch and UB units.  Tokens that follow one another in one tile of 16 places of a page are
// stored together, by the warp that has the first of them.
template <typename T, int UB, int GS>
__global__ void __launch_bounds__(WARPS * 32) kv4_store_kernel(const T* k, const T* v, long long stride, const int* __restrict__ tok_slot,
                                                               const int* __restrict__ tok_pos, unsigned char* k_pages, unsigned char* v_pages,
                                                               const int* __restrict__ page_table, int max_pages, int n, int d, int page, int span, int key_blocks,
                                                               int lane_bits) {
  const int lane = threadIdx.x & 31, head = blockIdx.y, n_kv = gridDim.y;
  constexpr int GROUP = 16 * GS;
  const size_t tile_bytes = kv4_tile_bytes(page, d, GROUP);
  if ((int)blockIdx.x < key_blocks) {
    const int at_once = (WARPS * 32) >> lane_bits, part = threadIdx.x & ((1 << lane_bits) - 1);
    const int t0 = blockIdx.x * (at_once * KEY_TOKENS) + (threadIdx.x >> lane_bits);
    typename Pairs<T>::two x[KEY_TOKENS][2][2] = {};
    int slot[KEY_TOKENS], pos[KEY_TOKENS];
#pragma unroll
    for (int i = 0; i < KEY_TOKENS; ++i) {
      const int t = t0 + i * at_once;
      slot[i] = t < n ? tok_slot[t] : -1;
      pos[i] = t < n ? tok_pos[t] : 0;
      const T* const row = k + (long long)t * stride + (size_t)head * d;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int at = 32 * (part >> 2) + 16 * q + 4 * (part & 3);
        if (t < n && at < d) {   // four numbers at once
          const auto v = *reinterpret_cast<const typename Pairs<T>::four*>(row + at);
          x[i][q][0] = Pairs<T>::half(v, 0);
          x[i][q][1] = Pairs<T>::half(v, 1);
        }
      }
    }
    store_keys<T, GS>(x, slot, pos, part, k_pages, v_pages, page_table, max_pages, n_kv, head, d, page, tile_bytes);
    return;
  }
  const int job = (blockIdx.x - key_blocks) * WARPS + (threadIdx.x >> 5), parts = kv4_units(d) / UB;
  const long long n0 = (long long)(job / parts) * span;
  if (n0 >= n) return;
  // the launch's tokens from n0 on, one a lane: those that begin a run, and (of the 32 that are looked at) where runs go on
  const long long mine = n0 + lane;
  const int slot = mine < n ? tok_slot[mine] : -1, pos = mine < n ? tok_pos[mine] : 0;
  const bool goes_on = mine < n && mine > 0 && slot >= 0 && tok_slot[mine - 1] == slot && tok_pos[mine - 1] == pos - 1 && pos % 16 != 0;
  const unsigned on = __ballot_sync(0xffffffffu, goes_on);
  unsigned first = __ballot_sync(0xffffffffu, lane < span && slot >= 0 && !goes_on);
  while (first) {
    const int i = __ffs(first) - 1;
    first &= first - 1;
    const unsigned behind = i == 31 ? 0u : ~(on >> (i + 1));   // a run has at most 16 tokens, and begins among the first 16
    const int count = behind ? min(16, __ffs(behind)) : 16;
    const int s = __shfl_sync(0xffffffffu, slot, i), p = __shfl_sync(0xffffffffu, pos, i);
    const Place at = place_of(k_pages, v_pages, page_table, max_pages, s, p, page, n_kv, head, tile_bytes);
    store_tile_values<T, UB, GS>(v + (n0 + i) * stride + (size_t)head * d, stride, at.v, at.t / 16 * 16, at.t % 16, count, (job % parts) * UB, d, page);
  }
}

// The same behind a fused projection (rows q | k | v): per-head norm and rotation of queries and keys first, a warp per (token, head).  Formulas and
// rounding points are those of rope_kv.cu.  A decode step's launch is some 3 us of latency (loads, a norm's sum, angles,
// a range), no rate, and overlaps the one before it (DEPENDENT); a prompt's, 2,000 tokens of 32 / 8 heads of 128 in 52 us, does not, and its heads share a token's angles in L1.
template <typename T, bool DEPENDENT>
__global__ void __launch_bounds__(WARPS * 32) kv4_rope_store_kernel(const T* qkv, int stride, const float* __restrict__ wq, const float* __restrict__ wk,
                                                                    const float* __restrict__ inv_freq, const T* cs_table, const int* __restrict__ tok_slot,
                                                                    const int* __restrict__ tok_pos, T* q_out, unsigned char* k_pages, unsigned char* v_pages,
                                                                    const int* __restrict__ page_table, int max_pages, int n_heads, int n_kv, int d, int rot,
                                                                    int group, int page, float eps, int has_norm) {
  __shared__ __align__(16) T rows[WARPS][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, head = blockIdx.y * WARPS + warp, half = rot >> 1;
  const long long n = blockIdx.x;
  if (gridDim.x <= SIGNAL_ROWS) let_next_launch_in();
  if (DEPENDENT) asm volatile("griddepcontrol.wait;" ::: "memory");
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
  if (head >= n_heads + n_kv) return store_value<DEPENDENT>(src, at.v, at.t, d, group, page);
  T* const row = rows[warp];
  const float* w = head < n_heads ? wq : wk;
  float x[8], ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = lane + 32 * i < d ? prev<DEPENDENT>(src + lane + 32 * i) : 0.f;
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
      cs = prev<DEPENDENT>(cs_table + n * rot + j);
      sn = prev<DEPENDENT>(cs_table + n * rot + half + j);
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
  if (head >= n_heads) {
    float k[2][4];
    load_key<T>(k, row, lane, d, true);
    if (group == 16) return store_key<1>(k, true, lane, at.k, at.t, d, page);
    if (group == 32) return store_key<2>(k, true, lane, at.k, at.t, d, page);
    if (group == 64) return store_key<4>(k, true, lane, at.k, at.t, d, page);
    return store_key<8>(k, true, lane, at.k, at.t, d, page);
  }
  for (int i = lane; i < d; i += 32) q_row[i] = row[i];
}

// What a pair of codes (`code_pair`) stands for, in T: z + (c - 7.5) s, rounded once.  c - 7.5 is exact in bfloat16.
template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> { typedef unsigned type; };
template <> struct Pair<float> { typedef float2 type; };
template <typename T> __device__ __forceinline__ typename Pair<T>::type values_of(unsigned pair, unsigned sz_lo, unsigned sz_hi) {
  if constexpr (sizeof(T) == 2) {
    const __nv_bfloat162 less = __floats2bfloat162_rn(-CODE_BIAS, -CODE_BIAS);
    const unsigned s = __byte_perm(sz_lo, sz_hi, 0x5410), z = __byte_perm(sz_lo, sz_hi, 0x7632);
    const __nv_bfloat162 v = __hfma2(__hadd2(*reinterpret_cast<const __nv_bfloat162*>(&pair), less), *reinterpret_cast<const __nv_bfloat162*>(&s),
                                     *reinterpret_cast<const __nv_bfloat162*>(&z));
    return *reinterpret_cast<const unsigned*>(&v);
  } else {
    const GroupCode a = unpack_code(sz_lo), b = unpack_code(sz_hi);
    return make_float2(fmaf(__uint_as_float(pair << 16) - CODE_BIAS, a.s, a.z), fmaf(__uint_as_float(pair & 0xffff0000u) - CODE_BIAS, b.s, b.z));
  }
}

// Blocks per (sequence, key head), each every gridDim.x-th chunk of it (a page, or part of a long one): the chunk's tokens as values, those behind the sequence's end
// as zeros.  Pages before the first key that the step's first token of the sequence sees (window <= 0: every key) are left alone: they may be another sequence's by now.
// A chunk's codes and scales are copied into shared memory while the one before is taken out; then a thread takes a word of a key (eight dims of a token) or a unit
// of a lane's values (four dims of four tokens), and neighbours fill whole sectors.  Bound by issue (81% of its slots) and, where pages are few, by the way to the first bytes: 64 sequences of up
// to 8,192 tokens, eight key heads of 128, 286 us, 4,990 GB/s (read straight from memory 411); 13 prompts, 12,829 tokens, 21.8 us, 3,180 GB/s; 8 of 100, 4.6 us.
__host__ __device__ inline int chunk_of(int page) { return page <= 64 ? page : page % 64 ? 16 : 64; }
__device__ __forceinline__ void copy16(unsigned to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from)); }
template <typename T>
__global__ void __launch_bounds__(256, 4) kv4_expand_kernel(const unsigned char* __restrict__ k_pages, const unsigned char* __restrict__ v_pages,
                                                            const int* __restrict__ page_table, int max_pages, const int* __restrict__ cu_q,
                                                            const int* __restrict__ seq_slot, const int* __restrict__ tok_pos, T* k_out, T* v_out, int n_kv, int d,
                                                            int group_bits, int page, int window) {
  typedef typename Pair<T>::type P;
  extern __shared__ __align__(16) unsigned char held[];   // two chunks: keys' codes, keys' scales, values' codes, values' scales
  const int b = blockIdx.z, head = blockIdx.y, slot = seq_slot[b], q0 = cu_q[b], q1 = cu_q[b + 1];
  if (slot < 0 || q1 <= q0) return;
  const int chunk = chunk_of(page), per_page = page / chunk, end = tok_pos[q1 - 1] + 1, first = window > 0 ? max(0, tok_pos[q0] + 1 - window) / page * per_page : 0;
  const int units = kv4_units(d), groups = d >> group_bits, row = kv4_row_bytes(d), words = 4 * units;
  const int codes = chunk * row, side = codes + chunk * groups * 4;   // bytes of a chunk's keys (or values)
  const size_t tile_bytes = kv4_tile_bytes(page, d, 1 << group_bits);
  const unsigned held_at = (unsigned)__cvta_generic_to_shared(held);
  const auto page_of = [&](int p) { return (size_t)page_table[(size_t)slot * max_pages + p / per_page] * n_kv + head; };
  const auto request = [&](int p, int buffer) {
    if (p * chunk < end) {
      const size_t at = page_of(p) * tile_bytes;
      const int t0 = p % per_page * chunk;
      for (int i = threadIdx.x * 16; i < side; i += 256 * 16) {
        const size_t from = at + (i < codes ? (size_t)t0 * row + i : (size_t)row * page + (size_t)t0 * groups * 4 + (i - codes));
        copy16(held_at + buffer * 2 * side + i, k_pages + from);
        copy16(held_at + (buffer * 2 + 1) * side + i, v_pages + from);
      }
    }
    asm volatile("cp.async.commit_group;");
  };
  // keys: the thread's word, and its tokens, `t_step` apart.  Values: its lane row r, unit u, and its (tile, c), `j_step` apart.
  const int t_step = 256 / words, kt0 = threadIdx.x / words, kx = threadIdx.x % words, ku = kx >> 2, kc = kx & 3;
  const int j_step = 32 / units, j0 = (threadIdx.x >> 3) / units, u = (threadIdx.x >> 3) % units, r = threadIdx.x & 7;
  request(first + blockIdx.x, 0);
  int buffer = 0;
  const int last = (end + page - 1) / page * per_page;   // (the last page is filled up, by zeros)
  for (int p = first + blockIdx.x; p < last; p += gridDim.x, buffer ^= 1) {
    request(p + gridDim.x, buffer ^ 1);
    const size_t out_at = (page_of(p) * page + p % per_page * chunk) * d;
    asm volatile("cp.async.wait_group 1;");
    __syncthreads();
    const unsigned char *kt = held + buffer * 2 * side, *vt = kt + side;
    const unsigned *ks = reinterpret_cast<const unsigned*>(kt + codes), *vs = reinterpret_cast<const unsigned*>(vt + codes);
    T *ko = k_out + out_at, *vo = v_out + out_at;
    const int left = end - p * chunk;
    if (kt0 < t_step)
#pragma unroll 2
      for (int t = kt0; t < chunk; t += t_step) {
        const bool have = t < left;
        const unsigned w = have ? *reinterpret_cast<const unsigned*>(kt + t * row + (kc * units + ku) * 4) : 0u;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int at = 32 * ku + 16 * s;
          if (at >= d) continue;
          const unsigned sz = have ? ks[t * groups + (at >> group_bits)] : 0u;
          P* const to = reinterpret_cast<P*>(ko + t * d + at + 4 * kc);
          const P a = values_of<T>(code_pair(w, 2 * s), sz, sz), e = values_of<T>(code_pair(w, 2 * s + 1), sz, sz);
          if constexpr (sizeof(T) == 2)
            *reinterpret_cast<uint2*>(to) = make_uint2(a, e);
          else
            *reinterpret_cast<float4*>(to) = make_float4(a.x, a.y, e.x, e.y);
        }
      }
    if (j0 < j_step)
#pragma unroll 2
      for (int j = j0; j < chunk / 4; j += j_step) {
        const int c = j & 3, tile = j >> 2, k0 = tile * 16 + 2 * c;
        const uint2 w = *reinterpret_cast<const uint2*>(vt + (tile * 256 + (r * 4 + c) * 8) * units + u * 8);
#pragma unroll
        for (int h = 0; h < 2; ++h)   // tokens k0, k0 + 1 and k0 + 8, k0 + 9
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const int at = 32 * u + 16 * s;
            if (at >= d) continue;
            const unsigned x = h ? w.y : w.x, a = code_pair(x, 2 * s), e = code_pair(x, 2 * s + 1);
#pragma unroll
            for (int o = 0; o < 2; ++o) {
              const int t = k0 + 8 * h + o;
              const unsigned sz = t < left ? vs[t * groups + (at >> group_bits)] : 0u;
              *reinterpret_cast<P*>(vo + t * d + at + 2 * r) = values_of<T>(__byte_perm(a, e, o ? 0x7632 : 0x5410), sz, sz);
            }
          }
      }
    __syncthreads();   // the next but one chunk goes where this one was
  }
  asm volatile("cp.async.wait_group 0;");
}

template <typename T, int UB, int GS>
int store_as(const void* k, const void* v, long long stride, const int* tok_slot, const int* tok_pos, void* k_pages, void* v_pages, const int* page_table,
             int max_pages, int n, int n_kv, int d, int page, cudaStream_t st) {
  // few tokens: a warp each, so that none waits for another; many: a warp for 16, most of which begin one run
  const int span = n > 512 ? 16 : 1, lane_bits = d > 128 ? 5 : d > 64 ? 4 : d > 32 ? 3 : 2;
  const int key_tokens = (WARPS * 32 >> lane_bits) * KEY_TOKENS, key_blocks = (n + key_tokens - 1) / key_tokens;
  const int warps = (n + span - 1) / span * (kv4_units(d) / UB), value_blocks = (warps + WARPS - 1) / WARPS;
  kv4_store_kernel<T, UB, GS><<<dim3(key_blocks + value_blocks, n_kv), WARPS * 32, 0, st>>>(
      (const T*)k, (const T*)v, stride, tok_slot, tok_pos, (unsigned char*)k_pages, (unsigned char*)v_pages, page_table, max_pages, n, d, page, span, key_blocks, lane_bits);
  return launch_status();
}
template <typename T>
int store(const void* k, const void* v, long long stride, const int* tok_slot, const int* tok_pos, void* k_pages, void* v_pages, const int* page_table,
          int max_pages, int n, int n_kv, int d, int group, int page, cudaStream_t st) {
#define DRYFT_STORE(UB, GS) return store_as<T, UB, GS>(k, v, stride, tok_slot, tok_pos, k_pages, v_pages, page_table, max_pages, n, n_kv, d, page, st)
  switch (group) {   // units that a warp takes: those of a group
    case 16: DRYFT_STORE(1, 1);
    case 32: DRYFT_STORE(1, 2);
    case 64: DRYFT_STORE(2, 4);
    case 128: DRYFT_STORE(4, 8);
  }
#undef DRYFT_STORE
  return DRYFT_ERR_UNSUPPORTED;
}
template <typename T>
int expand(const void* k_pages, const void* v_pages, const int* page_table, int max_pages, const int* cu_q, const int* seq_slot, const int* tok_pos, void* k_out,
           void* v_out, int n_seqs, int pages, int n_kv, int d, int group, int page, int window, cudaStream_t st) {
  const int chunk = chunk_of(page), chunks = pages * (page / chunk), bytes = 4 * chunk * (kv4_row_bytes(d) + 4 * (d / group));   // 48 KB at most
  const int blocks = 4096 / (n_kv * n_seqs) + 1;   // of a sequence and head: a few thousand blocks, however long the sequences may be (1,500: 64 ragged ones 345 us, not 286)
  kv4_expand_kernel<T><<<dim3(blocks < chunks ? blocks : chunks, n_kv, n_seqs), 256, bytes, st>>>((const unsigned char*)k_pages, (const unsigned char*)v_pages, page_table,
                                                                                                 max_pages, cu_q, seq_slot, tok_pos, (T*)k_out, (T*)v_out, n_kv, d,
                                                                                                 __builtin_ctz(group), page, window);
  return launch_status();
}
template <typename T>
int rope_store(const void* qkv, int stride, const float* wq, const float* wk, const float* inv_freq, const void* cs_table, const int* tok_slot, const int* tok_pos,
               void* q_out, void* k_pages, void* v_pages, const int* page_table, int max_pages, int n, int n_heads, int n_kv, int d, int rot, int group, int page,
               float eps, int has_norm, int pdl, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(n, (n_heads + 2 * n_kv + WARPS - 1) / WARPS);
  cfg.blockDim = dim3(WARPS * 32);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  const bool dependent = pdl && n <= (int)SIGNAL_ROWS;
  cfg.numAttrs = dependent ? 1 : 0;
  const auto kern = dependent ? kv4_rope_store_kernel<T, true> : kv4_rope_store_kernel<T, false>;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, (const T*)qkv, stride, wq, wk, inv_freq, (const T*)cs_table, tok_slot, tok_pos, (T*)q_out,
                                           (unsigned char*)k_pages, (unsigned char*)v_pages, page_table, max_pages, n_heads, n_kv, d, rot, group, page, eps, has_norm);
  return e != cudaSuccess ? (int)e : launch_status();
}
}  // namespace

DRYFT_API int dryft_kv4_rope_store(int is_bf16, const void* qkv, int stride, const float* wq, const float* wk, const float* inv_freq, const void* cs_table,
                                   const int* tok_slot, const int* tok_pos, void* q_out, void* k_pages, void* v_pages, const int* page_table, int max_pages, int n,
                                   int n_heads, int n_kv, int d, int rot, int group, int page, float eps, int has_norm, int pdl, void* stream) {
  if (n <= 0) return 0;
  return (is_bf16 ? rope_store<__nv_bfloat16> : rope_store<float>)(qkv, stride, wq, wk, inv_freq, cs_table, tok_slot, tok_pos, q_out, k_pages, v_pages, page_table,
                                                                  max_pages, n, n_heads, n_kv, d, rot, group, page, eps, has_norm, pdl, (cudaStream_t)stream);
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
