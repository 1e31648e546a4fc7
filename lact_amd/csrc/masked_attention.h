// Softmax attention of a sequence with itself under a mask of intervals, bf16 and fp32, head sizes 64 and 128, forward and backward:
//
//   s_ij = f(q_i . k_j / sqrt(D)) - slope_h |i - j|,   f(x) = cap tanh(x / cap) or x,   o_i = sum_j softmax_j(s_ij) v_j
//
// over the keys j in [lo_i, hi_i).  Every mask here is such an interval: a causal window (i - window < j <= i), packed documents (both
// ends cut at the document's) and prefixes (hi_i reaches the end of the prefix).  For a key the queries that see it are an interval too.
// k_attn_ranges writes both where there are documents; a causal window needs no memory for them.  A row that sees nothing has output 0.
//
// q: [B, L, H, D], k, v: [B, L, HK, D] with strides; a head's D elements are contiguous and heads follow each other; H is a multiple of
// HK, and query heads h * H / HK ... share key head h.  out: [B, L, H, D] contiguous.  lse: [B, H, L] fp32, log2 of the row's sum of 2^s.
//
// One wave owns 32 rows (queries in the forward and in dq, keys in dk/dv) as the columns of 32x32 matrix products, so that a lane holds
// one row and the softmax needs no exchange but where the row's maximum is moved; it walks the 64-row tiles of the other side that its
// intervals touch, which travel through a ring of asynchronous global -> LDS copies shared by the block.  The scores feed the next
// product as they lie: k slots 0..3 / 4..7 of lane half h stand for rows 4h + i / 8 + 4h + i of 16, on both operands.  fp32 runs the same
// code: eight 32x32x2 products for one 32x32x16.
//
// A masked place weighs exactly nothing, whatever lies there: scores, probabilities and their gradients are selected, not multiplied, and rows that
// are not finite throughout are taken out of the products (0 * inf is NaN); a row that sees one of them has NaN for an output (Spoilt).
#pragma once
#include "gemm_dma.h"
#include "window_attention.h"

namespace lact {

template <typename T>
struct MaskedAttnParams {
  int B, L, H, HK, group, window;    // group = H / HK; window >= L: none
  const T* q; const T* k; const T* v;
  int ldq, ldk, ldv;                 // elements between tokens
  long long bsq, bsk, bsv;           // elements between batch entries
  const int2* rows;                  // [B, L]: the keys that a query sees, null: those of the causal window
  const int2* cols;                  // [B, L]: the queries that see a key
  const float* slopes;               // [H] or null
  float scale, cap;                  // cap 0: none
  T* out;                            // [B, L, H, D]
  float* lse;                        // [B, H, L]
  // backward
  const T* dout; int lddo; long long bsdo;
  const T* o;
  float* delta;                      // [B, H, L]: sum_d dout * out, written by dq, read by dk/dv
  T* dq; T* dk; T* dv;               // contiguous
  float* part;                       // [2][splits][B, L, HK, D]: dk and dv of every split, where there are several
  int splits;
  UDiv by_heads, by_kv;              // blocks at one place of the sequence: B * H, or splits * B * HK; B * HK
  __device__ __forceinline__ void locate(int& x, int& z) const {
    x = by_heads.div(blockIdx.x);
    z = blockIdx.x - x * (int)by_heads.d;
  }
  // Query heads that share a key head lie B * HK blocks apart: on one die, whose L2 then holds their keys, where that is a multiple of eight.
  __device__ __forceinline__ void query_head(int z, int& b, int& h, int& hk) const {
    const int g = by_kv.div(z), e = z - g * (int)by_kv.d;
    b = e / HK;
    hk = e - b * HK;
    h = hk * group + g;
  }
  __device__ __forceinline__ int2 row_range(int b, int i) const {      // empty: {INT_MAX, 0}
    if (i >= L) return make_int2(0x7fffffff, 0);
    if (rows) {
      const int2 r = rows[(size_t)b * L + i];
      return r.x < r.y ? r : make_int2(0x7fffffff, 0);
    }
    return make_int2(max(0, i - window + 1), i + 1);
  }
  // A row sees itself: of one key, its softmax is constant, and the scores' gradients are 0 (dp - delta would leave what the two sums round differently).
  __device__ __forceinline__ static bool alone(int2 r) { return r.y - r.x == 1; }
  __device__ __forceinline__ int2 col_range(int b, int j) const {
    if (j >= L) return make_int2(0x7fffffff, 0);
    if (cols) {
      const int2 r = cols[(size_t)b * L + j];
      return r.x < r.y ? r : make_int2(0x7fffffff, 0);
    }
    return make_int2(j, window >= L ? L : min(L, j + window));
  }
};

// Intervals from the documents' bounds [B, n + 1] (null: one document) and the lengths of their prefixes [B, n] (null: none).  Whatever the bounds hold, the
// intervals lie inside [0, L).
__global__ void k_attn_ranges(int L, int n, int window, const int* __restrict__ bounds, const int* __restrict__ prefixes, int2* rows, int2* cols) {
  const int b = blockIdx.y, t = blockIdx.x * blockDim.x + threadIdx.x;
  if (t >= L) return;
  int lo = 1, start = 0, end = L;
  if (bounds) {
    const int* bd = bounds + (size_t)b * (n + 1);
    lo = 0;
    for (int hi = n + 1; lo < hi;) {      // the first bound past t
      const int m = (lo + hi) >> 1;
      if (bd[m] <= t) lo = m + 1;
      else hi = m;
    }
    start = lo > 0 ? bd[lo - 1] : 0;
    end = lo <= n ? bd[lo] : 0;
  }
  int2 r = make_int2(0, 0), c = make_int2(0, 0);
  if (lo > 0 && lo <= n) {
    const int s = min(max(start, 0), L), e = min(max(end, 0), L);
    if (s <= t && t < e) {
      const int p = s + (prefixes ? min(max(prefixes[(size_t)b * n + lo - 1], 0), e - s) : 0);
      r = make_int2(max(s, t - window + 1), max(t + 1, p));
      c = make_int2(t < p ? s : t, window >= L ? e : min(e, t + window));
    }
  }
  rows[(size_t)b * L + t] = r;
  cols[(size_t)b * L + t] = c;
}

// ---- what depends on the element type ---------------------------------------------------------------
typedef float f32x8 __attribute__((ext_vector_type(8)));
template <typename T> struct AttnType;
template <> struct AttnType<uint16_t> { using Frag = bf16x8; };
template <> struct AttnType<float> { using Frag = f32x8; };

__device__ __forceinline__ f32x16 mma32(const f32x8& a, const f32x8& b, f32x16 c) {
#pragma unroll
  for (int i = 0; i < 8; ++i) c = mma32(a[i], b[i], c);
  return c;
}

// A row maximum before there is one: below every score that is finite, and 2^(-infinity - it) is 0.
constexpr float ATTN_LOWEST = -3e38f;
constexpr int MASK_WAVES = 4;     // of a block; two blocks of the forward and of dq to a compute unit

template <typename T, int D>
struct MaskTile {       // 64 x D, the 16-byte granule g of row r at slot g ^ key(r): 16 rows of one granule fall into different banks
  static constexpr int ROWB = D * (int)sizeof(T), G = ROWB / 16, BYTES = 64 * ROWB;
  __device__ static __forceinline__ int key(int r) {
    if constexpr (sizeof(T) == 2) return AttnTile<D>::key(r);
    else return r & 15;
  }
};

template <typename T, int D, int NW = MASK_WAVES>
struct MaskCopy {
  using S = MaskTile<T, D>;
  static constexpr int NC = S::G / NW;      // copies of a wave and tile
  static_assert(S::G % NW == 0, "copies must split evenly over the waves");
  uint32_t voff[NC];
  const T* base;
  int ld, last, rows;
  __device__ __forceinline__ int row(int wave, int i) const { return ((wave + i * NW) * 64 + (int)(threadIdx.x & 63)) / S::G; }
  // the 64-row tiles [0, n) from row `first` on of a head whose rows end at L
  __device__ __forceinline__ void init(int wave, const T* head, int ld_, int first, int n, int L) {
    base = uniform(head + (size_t)first * ld_);
    ld = ld_; last = n - 1;
    rows = L - 1 - (first + last * 64);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int r = row(wave, i), slot = (threadIdx.x & 63) % S::G;
      voff[i] = (uint32_t)r * ld * sizeof(T) + (uint32_t)(slot ^ S::key(r)) * 16;
    }
  }
  __device__ __forceinline__ void issue(int t, const T* from, uint32_t lds, int wave) const {
    const T* at = from + (long long)t * 64 * ld;
    if (t < last || rows >= 63) {
#pragma unroll
      for (int i = 0; i < NC; ++i) dma16<false>(at, voff[i], lds + (wave + i * NW) * 1024);
    } else {      // rows past the end repeat the last one
#pragma unroll
      for (int i = 0; i < NC; ++i)
        dma16<false>(at, voff[i] - (uint32_t)max(0, row(wave, i) - rows) * ld * (uint32_t)sizeof(T), lds + (wave + i * NW) * 1024);
    }
  }
};

template <typename T, int D> struct MaskFrag;
template <int D> struct MaskFrag<uint16_t, D> : AttnFrag<D> {};
template <int D>
struct MaskFrag<float, D> {
  using S = MaskTile<float, D>;
  uint32_t row_base, row_key, col_off[8];
  __device__ __forceinline__ void init() {
    const int l = threadIdx.x & 63, h = l >> 5;
    row_base = (l & 31) * S::ROWB;
    row_key = (l & 15) << 4;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int r = (j < 4 ? 0 : 4) + 4 * h + j;      // tile row of slot j: 4h + j, 8 + 4h + j - 4
      col_off[j] = r * S::ROWB + (((((l & 31) >> 2) ^ r) << 4) | ((l & 3) << 2));
    }
  }
  __device__ __forceinline__ f32x8 rows(const char* tile, int rt, int ks) const {
    const uint32_t g = (uint32_t)(ks * 4 + 2 * ((threadIdx.x & 63) >> 5)) << 4;
    const char* p = tile + rt * 32 * S::ROWB + row_base;
    const float4 a = *reinterpret_cast<const float4*>(p + (g ^ row_key)), b = *reinterpret_cast<const float4*>(p + ((g + 16) ^ row_key));
    return f32x8{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  }
  __device__ __forceinline__ f32x8 cols(const char* tile, int dt, int st) const {
    f32x8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      v[j] = *reinterpret_cast<const float*>(tile + st * 16 * S::ROWB + (dt >> 1) * 256 + (col_off[j] ^ (uint32_t)((dt & 1) << 7)));
    return v;
  }
};

template <typename T, int D>
__device__ __forceinline__ void mask_own_rows(typename AttnType<T>::Frag (&f)[D / 16], const T* base, int ld, int row, int L) {
  if constexpr (sizeof(T) == 2) {
    attn_own_rows<D>(f, base, ld, row, L);
  } else {
    const T* p = base + (size_t)min(row, L - 1) * ld + 8 * ((threadIdx.x & 63) >> 5);
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      const float4 a = *reinterpret_cast<const float4*>(p + s * 16), b = *reinterpret_cast<const float4*>(p + s * 16 + 4);
      f[s] = f32x8{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    }
  }
}
// See attn_arrived: what was loaded is there behind this, so that no wait for it lies in the loop.
template <int N>
__device__ __forceinline__ void mask_arrived(bf16x8 (&f)[N]) { attn_arrived(f); }
template <int N>
__device__ __forceinline__ void mask_arrived(f32x8 (&f)[N]) {
#pragma unroll
  for (int s = 0; s < N; ++s) asm volatile("" : "+v"(f[s]));
}

// Eight of a lane's accumulators as an operand.  bf16: probabilities and their gradients are rounded to 8 bits for the product, whose
// sum stays in fp32.
template <typename T>
__device__ __forceinline__ typename AttnType<T>::Frag mask_pack(const f32x16& s, int st) {
  if constexpr (sizeof(T) == 2) return attn_pack(s, st);
  else return f32x8{s[8 * st], s[8 * st + 1], s[8 * st + 2], s[8 * st + 3], s[8 * st + 4], s[8 * st + 5], s[8 * st + 6], s[8 * st + 7]};
}

// Whether eight elements hold something that is not finite.
__device__ __forceinline__ bool unfinite(const bf16x8& f) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  const uint4 u = __builtin_bit_cast(uint4, f);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  u16x2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
  return max(m[0], m[1]) >= 0x7f80;
}
__device__ __forceinline__ bool unfinite(const f32x8& f) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
  return m >= 0x7f800000u;
}
// A word of LDS that other waves write.
__device__ __forceinline__ uint32_t lds_word(const void* p) {
  typedef __attribute__((address_space(3))) const volatile uint32_t lds_u32;
  return *(lds_u32*)(const __attribute__((address_space(3))) char*)(const char*)p;
}
// What lies in a tile and is not finite must not meet the zero weight of a row that does not see it.  The wave that copied 1 KB of a tile looks it over
// once it is there, clears rows that hold such a value and writes down which; every wave gives the rows of its own that see one of them NaN.
// (Selecting in the products' operands instead, where a tile is masked, cost a tenth of the forward: a branch at every operand, or registers for two loops.)
template <typename T, int D, int NW = MASK_WAVES>
struct Spoilt {
  using S = MaskTile<T, D>;
  static constexpr int BYTES = 64;
  // Rows [0, 32) and [32, 64) of tile t at its place of four (with as many places as a ring of two has, a wave may write down those of the next tile before
  // they are cleared); the last word: whether there ever were any.
  uint32_t* words;
  __device__ __forceinline__ void init(char* lds) {
    words = reinterpret_cast<uint32_t*>(lds);
    if (threadIdx.x < 16) words[threadIdx.x] = 0;
    __syncthreads();
  }
  __device__ __forceinline__ static bool bad(const uint4& u) {
    if constexpr (sizeof(T) == 2) return unfinite(__builtin_bit_cast(bf16x8, u));
    else return ((u.x & 0x7f800000u) == 0x7f800000u) | ((u.y & 0x7f800000u) == 0x7f800000u) | ((u.z & 0x7f800000u) == 0x7f800000u) | ((u.w & 0x7f800000u) == 0x7f800000u);
  }
  __device__ __forceinline__ void look(char* tile, int t, int wave) const {
    constexpr int NC = S::G / NW;
    const int l = threadIdx.x & 63;
    uint4 u[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) u[i] = *reinterpret_cast<uint4*>(tile + (wave + i * NW) * 1024 + l * 16);
    bool some = false;
#pragma unroll
    for (int i = 0; i < NC; ++i) some |= bad(u[i]);
    if (!__any(some)) return;
#pragma unroll 1
    for (int i = 0; i < NC; ++i) {
      uint4* at = reinterpret_cast<uint4*>(tile + (wave + i * NW) * 1024 + l * 16);
      const uint64_t who = __ballot(bad(*at));
      const int in = l / S::G, row = (wave + i * NW) * (64 / S::G) + in;      // G lanes hold a row
      if (who >> (in * S::G) & ((1ull << S::G) - 1)) {
        *at = make_uint4(0, 0, 0, 0);
        if (l % S::G == 0) atomicOr(words + 2 * (t & 3) + (row >> 5), 1u << (row & 31));
        words[15] = 1;
      }
    }
  }
  // behind the barrier: the tile's rows; and room for those of the tile after the next, which nobody looks over before the next barrier.  (Read as LDS by its address space: through a generic
  // pointer the load counts as one of global memory too, and its wait is one for the copies just issued.)
  __device__ __forceinline__ bool any() const { return __builtin_amdgcn_readfirstlane(lds_word(words + 15)) != 0; }
  __device__ __forceinline__ uint64_t rows(int t) const { return (uint64_t)words[2 * (t & 3)] | (uint64_t)words[2 * (t & 3) + 1] << 32; }
  __device__ __forceinline__ void clear_after_next(int t) const {
    if (threadIdx.x < 2) words[2 * ((t + 2) & 3) + threadIdx.x] = 0;
  }
};

// tanh in fp32, of a = |x|, by one division: tanh(a) / a up to 0.8, by Lambert's continued fraction x / (1 + x^2 / (3 + x^2 / (5 + x^2 / (7 + x^2 / 9)))), relative error
// below 1e-8; past it what tanh lacks of 1, 2 / (1 + e^2a), which would lose the bits that x has below 1.
struct Tanh {
  bool near;
  float q;
  __device__ __forceinline__ explicit Tanh(float a) : near(a < 0.8f) {
    const float y = a * a, e = 1.f + __builtin_amdgcn_exp2f(a * (2.f * ATTN_LOG2E));
    q = (near ? fmaf(y, fmaf(y, 1.f, 105.f), 945.f) : 2.f) / (near ? fmaf(y, fmaf(y, 15.f, 420.f), 945.f) : e);
  }
};

// What the scores go through: nothing; a cap, a distance or both; the same with a cap past CAP_QUICK in bf16.  (A branch in one kernel takes 12 registers more, which cost the
// heads of 64 a wave of a SIMD, and dq of heads of 128 spills.)
enum { SCORES_PLAIN, SCORES_BENT, SCORES_FAR_CAP };
constexpr float CAP_QUICK = 256.f / ATTN_LOG2E;

// Scores as they come out of the product -> what 2^ is taken of, times `unit` (see below)
template <typename T, int BENT>
struct Scores {
  // k2 - 2 k2 / (1 + e^2x) for the capped score, with an error of 2 k2 2^-23: in bf16 with caps to CAP_QUICK, where that is a sixty-fourth of what a probability is
  // rounded by.  Otherwise the score itself times tanh(x) / x, whose error is relative however far the cap is.
  static constexpr bool QUICK = sizeof(T) == 2 && BENT == SCORES_BENT;
  float c;          // scale log2(e); without a cap the scores keep it out until they meet the maximum
  float k1, k2;     // with a cap: scale / cap (QUICK: 2 log2(e) times it), cap log2(e)
  float slope;      // times log2(e)
  bool cap, bias;
  __device__ __forceinline__ void init(float scale, float cap_, const float* slopes, int h) {
    cap = BENT && cap_ > 0.f; bias = BENT && slopes != nullptr;
    k1 = fminf(QUICK ? 2.f * ATTN_LOG2E * scale / cap_ : scale / cap_, 3e38f);      // (finite: a score of 0 stays 0 under the smallest caps)
    k2 = cap_ * ATTN_LOG2E;
    slope = bias ? slopes[h] * ATTN_LOG2E : 0.f;
    c = scale * ATTN_LOG2E;
  }
  // what is left to multiply by behind apply()
  __device__ __forceinline__ float unit() const { return BENT ? 1.f : c; }
  // the capped score times log2(e), and the derivative of the cap, 1 - tanh^2
  __device__ __forceinline__ float capped(float s, float& slope) const {
    if constexpr (QUICK) {
      const float t = fmaf(__builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s * k1)), -2.f, 1.f);      // to 2^-23
      slope = fmaf(-t, t, 1.f);
      return t * k2;
    } else {
      const float a = fabsf(s * k1);
      const Tanh t(a);
      const float lacks = t.near ? fmaf(-a, t.q, 1.f) : t.q;      // of 1, with all digits
      slope = lacks * (2.f - lacks);
      return t.near ? s * c * t.q : copysignf(fmaf(-k2, t.q, k2), s);
    }
  }
  // `first`: the place of the lane's element 0 minus the place of its own row
  __device__ __forceinline__ void apply(f32x16& s, int first) const {
    if constexpr (BENT == SCORES_PLAIN) return;
    if (cap) {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        float slope;
        if constexpr (QUICK) s[j] = fmaf(__builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s[j] * k1)), -2.f * k2, k2);
        else s[j] = capped(s[j], slope);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) s[j] *= c;
    }
    lower(s, first);
  }
  // the same, and the gradients dp (of what the softmax weighs) times the derivative of the cap
  __device__ __forceinline__ void apply(f32x16& s, f32x16& dp, int first) const {
    if constexpr (BENT == SCORES_PLAIN) return;
    if (cap) {
      // (in steps of four: one loop over both vectors leaves them in memory)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float by[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) s[4 * g + j] = capped(s[4 * g + j], by[j]);
#pragma unroll
        for (int j = 0; j < 4; ++j) dp[4 * g + j] *= by[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) s[j] *= c;
    }
    lower(s, first);
  }
  __device__ __forceinline__ void lower(f32x16& s, int first) const {
    if (!bias) return;
    const float f = (float)first;
#pragma unroll
    for (int j = 0; j < 16; ++j) s[j] = fmaf(fabsf(f + (float)(8 * (j / 4) + j % 4)), -slope, s[j]);
  }
};

// Waves of dk/dv that share 32 keys: heads of 128 in bf16 take two, one for the queries [0, 32) of every tile and one for [32, 64), whose sums are added at the
// end.  A wave's two accumulators (128 registers) and its own keys and values (64) leave too little of the 256 that two waves of a SIMD have each: here
// the values are read from LDS.  One wave with all of them in 400 registers: 148 us at 2 x 4096 tokens in documents, 12 heads.
// With a cap or a distance there are too many for that as well: 969 us as one wave, 1075 as two, the backward of 4 x 4096 tokens of 12 heads.
template <typename T, int D, int BENT> constexpr int mask_halves() { return sizeof(T) == 2 && D == 128 && !BENT ? 2 : 1; }
// 64-row tiles of both operands in LDS
template <typename T, int D> constexpr int mask_ring(bool keys) { return sizeof(T) == 4 || (D == 128 && !keys) ? 2 : 3; }
// stats: of dk/dv; groups of 32 rows; halves: waves that share them
template <typename T, int D>
constexpr int mask_lds_bytes(bool stats, int groups, int halves) {
  const int R = mask_ring<T, D>(stats);
  const int ring = R * 2 * MaskTile<T, D>::BYTES + (stats ? R * 512 + (halves - 1) * 2 * MaskTile<T, D>::BYTES : 0) + Spoilt<T, D>::BYTES;
  // what the rows are stored through, for splits in fp32, and what one half of the waves gives to the other
  const int store = groups * 32 * cmax((D + 16 / (int)sizeof(T)) * (int)sizeof(T), stats ? (D + 4) * 4 : 0);
  return cmax(cmax(ring, store), (halves - 1) * groups * 64 * ((stats ? 2 : 1) * D * 2 + 16));
}
// The second half's accumulators to the first, through LDS: a wave's [N][4][64 lanes] float4.
template <int N>
__device__ __forceinline__ void mask_give(float4* at, const f32x16 (&acc)[N]) {
#pragma unroll
  for (int dt = 0; dt < N; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) at[(dt * 4 + g) * 64] = make_float4(acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]);
}
template <int N>      // acc mine + theirs other
__device__ __forceinline__ void mask_take(const float4* at, f32x16 (&acc)[N], float mine, float theirs) {
#pragma unroll
  for (int dt = 0; dt < N; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float4 u = at[(dt * 4 + g) * 64];
      acc[dt][4 * g] = fmaf(acc[dt][4 * g], mine, u.x * theirs);
      acc[dt][4 * g + 1] = fmaf(acc[dt][4 * g + 1], mine, u.y * theirs);
      acc[dt][4 * g + 2] = fmaf(acc[dt][4 * g + 2], mine, u.z * theirs);
      acc[dt][4 * g + 3] = fmaf(acc[dt][4 * g + 3], mine, u.w * theirs);
    }
}

// Walks the tiles [0, n): issue(t) starts the copies of tile t, COPIES of a wave, RING - 1 tiles ahead; look(t) sees the wave's own when they are there;
// body(t, rows) uses the tile, `rows` of which are spoilt.
template <int COPIES, int RING, typename Sp, typename Issue, typename Look, typename Body>
__device__ __forceinline__ void mask_walk(int n, const Sp& spoilt, Issue issue, Look look, Body body) {
#pragma unroll
  for (int t = 0; t < RING - 1; ++t)
    if (t < n) issue(t);
  for (int t = 0; t < n; ++t) {
    if (RING == 3 && t + 1 < n) wait_vmcnt<COPIES>();
    else wait_vmcnt<0>();
    look(t);
    __syncthreads();      // tile t is there for every wave, and all are through with t - 1, whose place the next one takes
    if (t + RING - 1 < n) issue(t + RING - 1);
    uint64_t rows = 0;
    if (spoilt.any()) {
      rows = spoilt.rows(t);
      spoilt.clear_after_next(t);
    }
    body(t, rows);
  }
}

// A wave's [D][32] accumulator (rows = D, columns = its own rows), times `f`, to 32 rows of a tensor with rows ld apart.
template <typename T, int D>
__device__ __forceinline__ void mask_store_rows(char* lds, const f32x16 (&acc)[D / 32], float f, T* out, size_t ld, int row0, int L) {
  constexpr int E = 16 / (int)sizeof(T), LD = D + E, LPR = D / E;
  const int l = threadIdx.x & 63;
  T* t = reinterpret_cast<T*>(lds);
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      Elem<T>::store4(t + (l & 31) * LD + dt * 32 + 8 * g + 4 * (l >> 5), acc[dt][4 * g] * f, acc[dt][4 * g + 1] * f, acc[dt][4 * g + 2] * f, acc[dt][4 * g + 3] * f);
  wave_lds_fence();
#pragma unroll
  for (int i = 0; i < 32 * LPR / 64; ++i) {
    const int id = i * 64 + l, r = id / LPR, c = (id % LPR) * E;
    const uint4 u = *reinterpret_cast<const uint4*>(t + r * LD + c);
    if (row0 + r < L) *reinterpret_cast<uint4*>(out + (size_t)(row0 + r) * ld + c) = u;
  }
  wave_lds_fence();
}

// What rows see, over a wave.  Neither end of the intervals falls from one row to the next, but rows may see nothing, which have {INT_MAX, 0}.
struct Reach {
  int lo, hi;            // of all of them: no tile outside
  int full_lo, full_hi;  // of every one of them: no mask inside
  // `rows`: one row a lane, in order, in the first COUNT lanes
  template <int COUNT>
  __device__ __forceinline__ void init(int2 rows) {
    const uint64_t all = ~0ull >> (64 - COUNT), some = __ballot(rows.x < rows.y) & all;
    lo = full_lo = 0x7fffffff;
    hi = full_hi = 0;
    if (some) {
      lo = __builtin_amdgcn_readlane(rows.x, __builtin_ctzll(some));
      hi = __builtin_amdgcn_readlane(rows.y, 63 - __builtin_clzll(some));
    }
    if (some == all) {
      full_lo = __builtin_amdgcn_readlane(rows.x, COUNT - 1);
      full_hi = __builtin_amdgcn_readlane(rows.y, 0);
    }
  }
  __device__ __forceinline__ bool sees(int a, int n) const { return a < hi && a + n > lo; }
  __device__ __forceinline__ bool masked(int a, int n) const { return a < full_lo || a + n > full_hi; }
};

// Which of a lane's 16 elements of 32 tile rows lie in [lo, hi): element j is row 8 (j / 4) + j % 4, lo and hi count from the lane's first.  Two
// instructions an element to apply (a bit spread over a word, a select by it) where comparisons take four.
struct Seen {
  uint32_t bits;
  __device__ __forceinline__ Seen(int lo, int hi) {
    const uint32_t below = hi >= 32 ? 0xffffffffu : hi <= 0 ? 0u : (1u << hi) - 1u, under = lo >= 32 ? 0xffffffffu : lo <= 0 ? 0u : (1u << lo) - 1u;
    bits = below & ~under;
  }
  // whether a row among `rows` (of the 32) is one of them
  __device__ __forceinline__ bool any_of(uint32_t rows) const { return (bits & 0x0f0f0f0fu & rows >> (4 * ((threadIdx.x & 63) >> 5))) != 0; }
  // all ones or zero
  __device__ __forceinline__ uint32_t word(int j) const {
    uint32_t w;
    asm("v_bfe_i32 %0, %1, %2, 1" : "=v"(w) : "v"(bits), "n"(8 * (j / 4) + j % 4));
    return w;
  }
  __device__ __forceinline__ float or_nothing(float s, int j) const {      // s, or -infinity
    float r;
    asm("v_bfi_b32 %0, %1, %2, %3" : "=v"(r) : "v"(word(j)), "v"(s), "s"(0xff800000u));
    return r;
  }
  __device__ __forceinline__ float or_zero(float s, int j) const { return __uint_as_float(__float_as_uint(s) & word(j)); }
};
// One instruction; fmaxf quiets its operands first.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// Without a cap or a distance the maximum m of a row is rounded where the scores' maximum h is multiplied by c, the scores in fma are not: past 2^20 the difference would reach
// 2^(the rounding).  Such rows, far ones, subtract h ahead of the product.
constexpr float ATTN_FAR = 1048576.f;
__device__ __forceinline__ bool attn_far(float m) { return fabsf(m) > ATTN_FAR && m > ATTN_LOWEST; }
// How much more was taken off the scores of a row under (m, h) than under (n, i): exactly what either takes.
__device__ __forceinline__ float attn_above(float m, float h, float n, float i, float c) {
  if (attn_far(m)) return attn_far(n) ? (h - i) * c : fmaf(h, c, -n);
  return attn_far(n) ? fmaf(-i, c, m) : m - n;
}

// Outputs.  Bound by the vector instructions between the two products of a tile: for 64 scores of a wave some 70 cycles with a cap (two exponentials and a
// reciprocal at a quarter of the rate) beside 32 of matrix products at D = 128, which the other wave of the SIMD covers in part.  A prompt of 8191 tokens in
// a prefix, 32 heads of 128 over 8, cap 30: 746 us, 743 TFLOP/s, the vector units busy for 69 % of the time and the matrix units for 34 %; 2 x 4096 tokens in documents, 12 heads
// of 128, window 2048: 57 us.  (Where both apply, window_attention.h forms the scores a tile ahead: 4 x 4096 tokens, 12 heads of 128, window 2048, forward 180 / here 198 us.)
// HALVES: waves that share 32 queries, each with its half of every tile's keys; their sums are joined through LDS at the end.
template <typename T, int D, int BENT, int HALVES>
__global__ __launch_bounds__(64 * MASK_WAVES, sizeof(T) == 2 ? 2 : 1) void k_masked_attn_fwd(const MaskedAttnParams<T> p) {
  constexpr int NW = MASK_WAVES, KW = NW / HALVES, N = 2 / HALVES;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  using S = MaskTile<T, D>;
  using Copy = MaskCopy<T, D, NW>;
  using Frag = typename AttnType<T>::Frag;
  constexpr int STAGE = 2 * S::BYTES, RING = mask_ring<T, D>(false);
  prefetch_args<sizeof(p)>();
  int bx, z, b, h, hk;
  p.locate(bx, z);
  bx = (p.L - 1) / (32 * KW) - bx;      // the longest rows of a causal mask first
  p.query_head(z, b, h, hk);
  const int L = p.L;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int group = wave % KW, half = wave / KW;        // of rows; of a tile's keys
  const int blk0 = bx * 32 * KW, row0 = blk0 + group * 32, row = row0 + (lane & 31);
  Frag qf[D / 16];
  mask_own_rows<T, D>(qf, p.q + b * p.bsq + h * D, p.ldq, row, L);
  const int2 own = p.row_range(b, row);
  int first = 0x7fffffff, last = 0;
#pragma unroll
  for (int i = 0; i < KW / 2; ++i) {
    Reach part;
    part.init<64>(p.row_range(b, blk0 + i * 64 + lane));
    first = min(first, part.lo); last = max(last, part.hi);
  }
  Reach reach;
  reach.init<32>(own);
  Scores<T, BENT> sc;
  sc.init(p.scale, p.cap, p.slopes, h);
  MaskFrag<T, D> fr;
  fr.init();
  f32x16 o[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) o[i][j] = 0.f;
  const float c = sc.unit();
  float mc = ATTN_LOWEST, sum = 0.f;        // running row maximum (of what 2^ is taken of) and this lane's share of the row sum
  float high = ATTN_LOWEST;      // that maximum ahead of the product with c, for far rows (attn_far)
  bool far = false;
  first = min(first, L) / 64 * 64;
  const int tiles = last > first ? (last - first + 63) / 64 : 0;
  Copy ck, cv;
  ck.init(wave, p.k + b * p.bsk + hk * D, p.ldk, first, tiles, L);
  cv.init(wave, p.v + b * p.bsv + hk * D, p.ldv, first, tiles, L);
  const uint32_t lds0 = lds_addr(smem);
  Spoilt<T, D, NW> spoilt;
  spoilt.init(smem + RING * STAGE);
  mask_arrived(qf);
  mask_walk<2 * Copy::NC, RING>(tiles, spoilt,
    [&](int t) LACT_INLINE_LAMBDA {
      const uint32_t slot = lds0 + t % RING * STAGE;
      ck.issue(t, ck.base, slot, wave);
      cv.issue(t, cv.base, slot + S::BYTES, wave);
    },
    [&](int t) LACT_INLINE_LAMBDA { spoilt.look(smem + t % RING * STAGE + S::BYTES, t, wave); },
    [&](int t, uint64_t bad) LACT_INLINE_LAMBDA {
      const int k0 = first + t * 64 + 32 * half;
      if (!reach.sees(k0, 32 * N)) return;
      const char* kt = smem + t % RING * STAGE;
      const char* vt = kt + S::BYTES;
      f32x16 s[N];
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) s[i][j] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = mma32(fr.rows(kt, i + half, ks), qf[ks], s[i]);
      const int at = k0 + 4 * (lane >> 5);
#pragma unroll
      for (int i = 0; i < N; ++i) sc.apply(s[i], at + 32 * i - row);
      if (reach.masked(k0, 32 * N)) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const Seen seen(own.x - at - 32 * i, own.y - at - 32 * i);
#pragma unroll
          for (int j = 0; j < 16; ++j) s[i][j] = seen.or_nothing(s[i][j], j);
        }
      }
      if (bad) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (Seen(own.x - at - 32 * i, own.y - at - 32 * i).any_of((uint32_t)(bad >> (32 * (i + half))))) sum = __builtin_nanf("");
      }
      float mx;
      if constexpr (N == 2) {
        mx = max3(s[0][0], s[1][0], s[1][1]);
#pragma unroll
        for (int j = 1; j < 16; ++j) mx = max3(mx, s[0][j], s[N - 1][j]);
      } else {
        mx = max3(s[0][0], s[0][1], s[0][15]);
#pragma unroll
        for (int j = 1; j < 8; ++j) mx = max3(mx, s[0][2 * j], s[0][2 * j + 1]);
      }
      const float top = mx;
      mx *= c;
      // The maximum only has to keep exp2 in range: it follows the row when it is exceeded by more than 2^8 (its own row only: what a row
      // gives does not depend on the others).
      if (__any(mx > mc + 8.f)) {
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const bool moves = mx > mc + 8.f;
        const float nm = moves ? mx : mc;
        float f;
        if constexpr (BENT) {
          f = __builtin_amdgcn_exp2f(mc - nm);
        } else {
          const float was = high;
          high = moves ? fmaxf(top, __shfl_xor(top, 32, 64)) : high;
          f = __builtin_amdgcn_exp2f(attn_above(mc, was, nm, high, c));
          far = __any(attn_far(nm));
        }
        mc = nm;
        sum *= f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j) o[i][j] *= f;
      }
      float base = mc;
      if constexpr (!BENT)
        if (far) {
          const bool mine = attn_far(mc);
          base = mine ? 0.f : mc;
#pragma unroll
          for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) s[i][j] -= mine ? high : 0.f;
        }
      float part[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          s[i][j] = __builtin_amdgcn_exp2f(fmaf(s[i][j], c, -base));
          part[i] += s[i][j];
        }
      sum += part[0] + part[1];
#pragma unroll
      for (int st = 0; st < 2 * N; ++st) {
        const Frag pf = mask_pack<T>(s[st >> 1], st & 1);
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) o[dt] = mma32(fr.cols(vt, dt, st + 2 * half), pf, o[dt]);
      }
    });
  sum += __shfl_xor(sum, 32, 64);
  __syncthreads();
  if constexpr (HALVES == 2) {
    float4* theirs = reinterpret_cast<float4*>(smem) + group * (D / 32) * 256 + lane;
    float4* stats = reinterpret_cast<float4*>(smem + KW * D * 128) + group * 64 + lane;
    if (half == 1) {
      mask_give(theirs, o);
      *stats = make_float4(mc, sum, high, 0.f);
    }
    __syncthreads();
    if (half == 0) {
      const float4 u = *stats;
      float above = mc - u.x;
      if constexpr (!BENT) above = attn_above(mc, high, u.x, u.z, c);
      const float f = __builtin_amdgcn_exp2f(fminf(above, 0.f)), e = __builtin_amdgcn_exp2f(fminf(-above, 0.f));
      mask_take(theirs, o, f, e);
      mc = above < 0.f ? u.x : mc;
      sum = fmaf(sum, f, u.y * e);
    }
    __syncthreads();
    if (half == 1) return;
  }
  const bool empty = own.x >= own.y;
  if (lane < 32 && row < L) p.lse[(size_t)(b * p.H + h) * L + row] = empty ? 0.f : mc + __builtin_amdgcn_logf(sum);   // v_log_f32 is base 2
  mask_store_rows<T, D>(smem + group * 32 * (D + 16 / sizeof(T)) * sizeof(T), o, empty ? 0.f : 1.f / sum, p.out + ((size_t)b * L * p.H + h) * D, (size_t)p.H * D, row0, L);
}

// dq = scale * sum_keys ds k with ds = p (dp - delta) f', and delta itself, from the output as it is stored: what that was rounded by is in all of a row's ds
// (bf16, relative errors of dq: its own rounding 1.65e-3, with that of ds 2.37e-3, with the output's 2.46e-3; an output of 32 bits beside it would be written
// and read for the last).  The probabilities are formed again from lse: the scores are a product more, but nothing of length L^2 is in memory.  Bound as the
// outputs are; 2 x 4096 tokens in documents, 12 heads of 128, window 2048: 77 us.
template <typename T, int D, int BENT, int HALVES>
__global__ __launch_bounds__(64 * MASK_WAVES, sizeof(T) == 2 ? 2 : 1) void k_masked_attn_dq(const MaskedAttnParams<T> p) {
  constexpr int NW = MASK_WAVES, KW = NW / HALVES;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  using S = MaskTile<T, D>;
  using Copy = MaskCopy<T, D, NW>;
  using Frag = typename AttnType<T>::Frag;
  constexpr int STAGE = 2 * S::BYTES, RING = mask_ring<T, D>(false);
  prefetch_args<sizeof(p)>();
  int bx, z, b, h, hk;
  p.locate(bx, z);
  bx = (p.L - 1) / (32 * KW) - bx;
  p.query_head(z, b, h, hk);
  const int L = p.L;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int group = wave % KW, half = wave / KW;        // of rows; of a tile's keys
  const int blk0 = bx * 32 * KW, row0 = blk0 + group * 32, row = row0 + (lane & 31);
  Frag qf[D / 16], gf[D / 16];
  mask_own_rows<T, D>(gf, p.dout + b * p.bsdo + h * D, p.lddo, row, L);
  float delta = 0.f;
  {
    Frag of[D / 16];
    mask_own_rows<T, D>(of, p.o + ((size_t)b * L * p.H + h) * D, p.H * D, row, L);
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) delta += (float)gf[s][i] * (float)of[s][i];
    delta += __shfl_xor(delta, 32, 64);
  }
  const size_t stat = (size_t)(b * p.H + h) * L;
  if (half == 0 && lane < 32 && row < L) p.delta[stat + row] = delta;
  mask_own_rows<T, D>(qf, p.q + b * p.bsq + h * D, p.ldq, row, L);
  float lse = p.lse[stat + min(row, L - 1)];
  const int2 own = p.row_range(b, row);
  int first = 0x7fffffff, last = 0;
#pragma unroll
  for (int i = 0; i < KW / 2; ++i) {
    Reach part;
    part.init<64>(p.row_range(b, blk0 + i * 64 + lane));
    first = min(first, part.lo); last = max(last, part.hi);
  }
  Reach reach;
  reach.init<32>(own);
  Scores<T, BENT> sc;
  sc.init(p.scale, p.cap, p.slopes, h);
  MaskFrag<T, D> fr;
  fr.init();
  f32x16 o[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) o[i][j] = 0.f;
  const float c = sc.unit();
  first = min(first, L) / 64 * 64;
  const int tiles = last > first ? (last - first + 63) / 64 : 0;
  Copy ck, cv;
  ck.init(wave, p.k + b * p.bsk + hk * D, p.ldk, first, tiles, L);
  cv.init(wave, p.v + b * p.bsv + hk * D, p.ldv, first, tiles, L);
  const uint32_t lds0 = lds_addr(smem);
  mask_arrived(qf);
  mask_arrived(gf);
  asm volatile("" : "+v"(lse), "+v"(delta));
  Spoilt<T, D, NW> spoilt;
  spoilt.init(smem + RING * STAGE);
  float poison = 0.f;
  mask_walk<2 * Copy::NC, RING>(tiles, spoilt,
    [&](int t) LACT_INLINE_LAMBDA {
      const uint32_t slot = lds0 + t % RING * STAGE;
      ck.issue(t, ck.base, slot, wave);
      cv.issue(t, cv.base, slot + S::BYTES, wave);
    },
    [&](int t) LACT_INLINE_LAMBDA { spoilt.look(smem + t % RING * STAGE, t, wave); },
    [&](int t, uint64_t bad) LACT_INLINE_LAMBDA {
      const char* kt = smem + t % RING * STAGE;
      const char* vt = kt + S::BYTES;
#pragma unroll
      for (int part = 0; part < 2 / HALVES; ++part) {
        const int i = HALVES == 1 ? part : half, k0 = first + t * 64 + 32 * i;
        if (!reach.sees(k0, 32)) continue;
        f32x16 s, dp;
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = dp[j] = 0.f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          s = mma32(fr.rows(kt, i, ks), qf[ks], s);
          dp = mma32(fr.rows(vt, i, ks), gf[ks], dp);
        }
        const int at = k0 + 4 * (lane >> 5);
#pragma unroll
        for (int j = 0; j < 16; ++j) dp[j] -= delta;
        sc.apply(s, dp, at - row);
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = __builtin_amdgcn_exp2f(fmaf(s[j], c, -lse)) * dp[j];
        if (reach.masked(k0, 32)) {
          const Seen seen(own.x - at, own.y - at);
#pragma unroll
          for (int j = 0; j < 16; ++j) s[j] = seen.or_zero(s[j], j);
        }
        if (bad && Seen(own.x - at, own.y - at).any_of((uint32_t)(bad >> (32 * i)))) poison = __builtin_nanf("");
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          const Frag pf = mask_pack<T>(s, st);
#pragma unroll
          for (int dt = 0; dt < D / 32; ++dt) o[dt] = mma32(fr.cols(kt, dt, 2 * i + st), pf, o[dt]);
        }
      }
    });
  poison += __shfl_xor(poison, 32, 64);
  __syncthreads();
  if constexpr (HALVES == 2) {
    float4* theirs = reinterpret_cast<float4*>(smem) + group * (D / 32) * 256 + lane;
    float* spoils = reinterpret_cast<float*>(smem + KW * D * 128) + group * 64 + lane;
    if (half == 1) {
      mask_give(theirs, o);
      *spoils = poison;
    }
    __syncthreads();
    if (half == 0) {
      mask_take(theirs, o, 1.f, 1.f);
      poison += *spoils;
    }
    __syncthreads();
    if (half == 1) return;
  }
  mask_store_rows<T, D>(smem + group * 32 * (D + 16 / sizeof(T)) * sizeof(T), o, (p.alone(own) ? 0.f : p.scale) + poison, p.dq + ((size_t)b * L * p.H + h) * D, (size_t)p.H * D, row0, L);
}

// dv = sum_queries p dout, dk = scale * sum_queries ds q, over the queries of all heads that share the key head: a wave owns 32 keys and
// walks the queries that see them, head after head.  With few keys (blocks) the walk is cut into splits, whose sums k_attn_sum adds; all splits of the first
// keys, whose walks are the longest under a causal mask, come first.  (dq is not formed here as well: its sums over keys would be atomics, in no order.)
// 2 x 4096 tokens in documents, 12 heads of 128, window 2048: 117 us, bound as the outputs are and by LDS, which both operands are read from in both directions.  (bf16, heads of
// 128, without a cap or a distance: 256 registers and 12 more in memory.)
template <typename T, int D, int BENT>
__global__ __launch_bounds__((64 * MASK_WAVES * mask_halves<T, D, BENT>()), (sizeof(T) == 2 && (D == 64 || !BENT) ? 2 : 1)) void k_masked_attn_dkv(const MaskedAttnParams<T> p) {
  constexpr int KW = MASK_WAVES, HALVES = mask_halves<T, D, BENT>(), NW = KW * HALVES;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  using S = MaskTile<T, D>;
  using Copy = MaskCopy<T, D, NW>;
  using Frag = typename AttnType<T>::Frag;
  constexpr int STAGE = 2 * S::BYTES, RING = mask_ring<T, D>(true);
  prefetch_args<sizeof(p)>();
  int bx, z;
  p.locate(bx, z);
  const int split = p.by_kv.div(z);
  z -= split * (int)p.by_kv.d;
  const int b = z / p.HK, hk = z - b * p.HK, L = p.L;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int group = wave % KW, half = wave / KW;        // of keys; of a tile's queries
  const int blk0 = bx * 32 * KW, row0 = blk0 + group * 32, row = row0 + (lane & 31);
  Frag kf[D / 16], vf[HALVES == 1 ? D / 16 : 1];
  mask_own_rows<T, D>(kf, p.k + b * p.bsk + hk * D, p.ldk, row, L);
  char* values = smem + RING * (STAGE + 512) + Spoilt<T, D>::BYTES;      // of all of the block's keys, as two tiles
  if constexpr (HALVES == 1) {
    mask_own_rows<T, D>(vf, p.v + b * p.bsv + hk * D, p.ldv, row, L);
  } else {
    const int n = blk0 + 64 < L ? 2 : 1;      // (keys past the end have nothing in LDS, and nobody looks at their sums)
    Copy cv;
    cv.init(wave, p.v + b * p.bsv + hk * D, p.ldv, blk0, n, L);
    for (int i = 0; i < n; ++i) cv.issue(i, cv.base, lds_addr(values) + i * S::BYTES, wave);
  }
  const int2 own = p.col_range(b, row);
  const bool alone = p.alone(p.row_range(b, row));
  int first = 0x7fffffff, last = 0;
#pragma unroll
  for (int i = 0; i < KW / 2; ++i) {
    Reach part;
    part.init<64>(p.col_range(b, blk0 + i * 64 + lane));
    first = min(first, part.lo); last = max(last, part.hi);
  }
  Reach reach;
  reach.init<32>(own);
  MaskFrag<T, D> fr;
  fr.init();
  f32x16 ok[D / 32], ov[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) ok[i][j] = ov[i][j] = 0.f;
  first = min(first, L) / 64 * 64;
  const int tiles = last > first ? (last - first + 63) / 64 : 0, steps = tiles * p.group;
  const int splits = p.splits, from = (int)((long long)steps * split / splits), all = (int)((long long)steps * (split + 1) / splits) - from;
  const uint32_t lds0 = lds_addr(smem);
  const char* stats = smem + RING * STAGE;             // per ring slot: 64 lse, 64 delta
  const int h0 = hk * p.group;
  Copy cq, cg;
  cq.init(wave, p.q + b * p.bsq + h0 * D, p.ldq, first, tiles, L);
  cg.init(wave, p.dout + b * p.bsdo + h0 * D, p.lddo, first, tiles, L);
  // the even waves bring the slot's lse, the odd ones its delta: the same bytes from each, one copy per wave
  const float* st_src = (wave & 1 ? p.delta : p.lse) + (size_t)(b * p.H + h0) * L;
  int ih = tiles ? from / tiles : 0, it = from - ih * tiles, bh = ih, bt = it;      // head and tile of the next copies, and of the next use
  float poison = 0.f;
  Scores<T, BENT> sc;
  sc.init(p.scale, p.cap, p.slopes, h0);
  const float c = sc.unit();
  mask_arrived(kf);
  if constexpr (HALVES == 1) mask_arrived(vf);
  Spoilt<T, D, NW> spoilt;
  spoilt.init(smem + RING * (STAGE + 512));
  mask_walk<2 * Copy::NC + 1, RING>(all, spoilt,
    [&](int t) LACT_INLINE_LAMBDA {
      const uint32_t slot = t % RING;
      cq.issue(it, cq.base + ih * D, lds0 + slot * STAGE, wave);
      cg.issue(it, cg.base + ih * D, lds0 + slot * STAGE + S::BYTES, wave);
      const int q0 = first + it * 64;
      dma4(st_src + (size_t)ih * L + q0, (uint32_t)min(lane, L - 1 - q0) * 4, lds0 + RING * STAGE + slot * 512 + (wave & 1) * 256);
      if (++it == tiles) { it = 0; ++ih; }
    },
    [&](int t) LACT_INLINE_LAMBDA {
      spoilt.look(smem + t % RING * STAGE, t, wave);
      spoilt.look(smem + t % RING * STAGE + S::BYTES, t, wave);
    },
    [&](int t, uint64_t bad) LACT_INLINE_LAMBDA {
      const int slot = t % RING, t0 = first + bt * 64;
      if ((bt == 0 || t == 0) && p.slopes) sc.slope = p.slopes[h0 + bh] * ATTN_LOG2E;
      if (++bt == tiles) { bt = 0; ++bh; }
      const char* qt = smem + slot * STAGE;
      const char* gt = qt + S::BYTES;
#pragma unroll
      for (int part = 0; part < 2 / HALVES; ++part) {
        const int i = HALVES == 1 ? part : half, q0 = t0 + i * 32;
        if (!reach.sees(q0, 32)) continue;
        f32x16 s, ds;
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = ds[j] = 0.f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          s = mma32(fr.rows(qt, i, ks), kf[ks], s);
          ds = mma32(fr.rows(gt, i, ks), HALVES == 1 ? vf[HALVES == 1 ? ks : 0] : fr.rows(values + (group >> 1) * S::BYTES, group & 1, ks), ds);
        }
        const float* ls = reinterpret_cast<const float*>(stats + slot * 512) + i * 32 + 4 * (lane >> 5);
        const int at = q0 + 4 * (lane >> 5);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 d4 = *reinterpret_cast<const float4*>(ls + 64 + 8 * g);
          ds[4 * g] -= d4.x; ds[4 * g + 1] -= d4.y; ds[4 * g + 2] -= d4.z; ds[4 * g + 3] -= d4.w;
        }
        sc.apply(s, ds, at - row);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 l4 = *reinterpret_cast<const float4*>(ls + 8 * g);
          const float lv[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s[4 * g + j] = __builtin_amdgcn_exp2f(fmaf(s[4 * g + j], c, -lv[j]));
            ds[4 * g + j] *= s[4 * g + j];
          }
        }
        if (reach.masked(q0, 32)) {
          Seen seen(own.x - at, own.y - at);
#pragma unroll
          for (int j = 0; j < 16; ++j) s[j] = seen.or_zero(s[j], j);
          // (a query that sees its own key alone lies at an end of this key's interval, so that the tile is masked)
          if (alone && (uint32_t)(row - at) < 32) seen.bits &= ~(1u << (row - at));
#pragma unroll
          for (int j = 0; j < 16; ++j) ds[j] = seen.or_zero(ds[j], j);
        }
        if (bad && Seen(own.x - at, own.y - at).any_of((uint32_t)(bad >> (32 * i)))) poison = __builtin_nanf("");
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          const Frag pf = mask_pack<T>(s, st), df = mask_pack<T>(ds, st);
#pragma unroll
          for (int dt = 0; dt < D / 32; ++dt) {
            ov[dt] = mma32(fr.cols(gt, dt, 2 * i + st), pf, ov[dt]);
            ok[dt] = mma32(fr.cols(qt, dt, 2 * i + st), df, ok[dt]);
          }
        }
      }
    });
  poison += __shfl_xor(poison, 32, 64);
  if constexpr (HALVES == 2) wait_vmcnt<0>();      // the values', which a walk without tiles has not waited for
  __syncthreads();
  if constexpr (HALVES == 2) {      // the second half's sums to the first
    float4* theirs = reinterpret_cast<float4*>(smem) + group * 2 * (D / 32) * 256 + lane;
    float* spoils = reinterpret_cast<float*>(smem + 2 * KW * D * 128) + group * 64 + lane;
    if (half == 1) {
      mask_give(theirs, ok);
      mask_give(theirs + (D / 32) * 256, ov);
      *spoils = poison;
    }
    __syncthreads();
    if (half == 0) {
      mask_take(theirs, ok, 1.f, 1.f);
      mask_take(theirs + (D / 32) * 256, ov, 1.f, 1.f);
      poison += *spoils;
    }
    __syncthreads();
    if (half == 1) return;
  }
  const size_t o = ((size_t)b * L * p.HK + hk) * D, ld = (size_t)p.HK * D;
  if (splits > 1) {
    float* stage = reinterpret_cast<float*>(smem) + group * 32 * (D + 4);
    const size_t all_keys = (size_t)p.B * L * ld, at = split * all_keys + o;
    mask_store_rows<float, D>(reinterpret_cast<char*>(stage), ok, p.scale + poison, p.part + at, ld, row0, L);
    mask_store_rows<float, D>(reinterpret_cast<char*>(stage), ov, 1.f + poison, p.part + splits * all_keys + at, ld, row0, L);
    return;
  }
  char* stage = smem + group * 32 * (D + 16 / sizeof(T)) * sizeof(T);
  mask_store_rows<T, D>(stage, ok, p.scale + poison, p.dk + o, ld, row0, L);
  mask_store_rows<T, D>(stage, ov, 1.f + poison, p.dv + o, ld, row0, L);
}

// dk (blockIdx.y 0) and dv (1): the sums of their splits, four elements a thread, in the splits' order.  Bound by their way in: 31 MB, 6 us.
template <typename T>
__global__ __launch_bounds__(256) void k_attn_sum(long long n, int splits, const float* part, T* dk, T* dv) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const float* src = part + (blockIdx.y ? splits * n : 0) + i;
  float4 a = *reinterpret_cast<const float4*>(src);
#pragma unroll 4
  for (int s = 1; s < splits; ++s) {
    const float4 u = *reinterpret_cast<const float4*>(src + s * n);
    a.x += u.x; a.y += u.y; a.z += u.z; a.w += u.w;
  }
  Elem<T>::store4((blockIdx.y ? dv : dk) + i, a.x, a.y, a.z, a.w);
}

}  // namespace lact
