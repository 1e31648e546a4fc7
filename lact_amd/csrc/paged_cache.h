// A cache of keys and values in pages: [pages, HK, page size, D] each, bf16, fp32 or e4m3.  A sequence's place n lies in page table[b][n / size] at row n % size; what
// points outside the pages is no page.  A row of e4m3 has an exponent beside it (e8m0, [pages, HK, page size]): the smallest e with which the row's largest finite
// magnitude is at most 448 2^(e - 127).  The scale is a power of two, so that a number loses nothing but what lies under e4m3's three bits, and what is read back is exact in bf16
// where it is a multiple of bf16's smallest number, 2^-133, and below 2^128; with an exponent under 3 smaller ones are rounded.
//
// A head's rows of one page follow each other: what attention reads of a page is one piece, in 8 bits of 16 tokens 2 KB.
#pragma once
#include "common.h"

namespace lact {

struct Pages {
  int pages, size, wide, HK;        // wide: table entries of a sequence
  UDiv by_size;
  const int* table;                 // [B, wide]
  // from page to page, in elements
  long long k_page, v_page, ks_page, vs_page;
  void* k; void* v;
  uint8_t* ks; uint8_t* vs;
  // the page of a place, -1: none.  Nothing is read outside the table, and no other page comes back.
  __device__ __forceinline__ int page(int b, long long place) const {
    if (place < 0 || place >= (long long)wide * size) return -1;
    const int id = table[(size_t)b * wide + by_size.div((int)place)];
    return (unsigned)id < (unsigned)pages ? id : -1;
  }
  __device__ __forceinline__ int row(long long place) const { return (int)place - by_size.div((int)place) * size; }
  // rows in front of row `r` of a head in its page
  __device__ __forceinline__ int rows_before(int h, int r) const { return h * size + r; }
};

template <typename C> constexpr bool is_e4m3() { return sizeof(C) == 1; }

// 2^(e - 127) as fp32
__device__ __forceinline__ float e8m0(uint32_t e) { return __uint_as_float(e == 255 ? 0x7fc00000u : max(e << 23, 0x400000u)); }

// ---- tokens into their places, and back -------------------------------------------------------------
// A block has up to 16 places of one page, from a multiple of their number on, and some heads: a thread has 16 bytes of one token in each, at distances that are the same for all, and
// looks its page up once.  Its rows follow each other in the page and, head by head, in the tokens.
// Rows in the order of one head's tokens, each with a page of its own to look up and distances of its own, against this: 4 x 16384 tokens of 8 heads of 128 out of e4m3 93 -> 61 us
// (5.3 TB/s), 16381 into e4m3 26 -> 21 us, a ragged batch of 8 x 2048 of 12 heads in bf16 27 -> 17 us.
template <typename T, int D>
struct CacheTile {
  static constexpr int E = 16 / (int)sizeof(T), G = D / E, ROWS = 256 / G;      // elements of a thread, threads to a row, rows at once
  static constexpr int PLACES = ROWS < 16 ? ROWS : 16, ACROSS = ROWS / PLACES;   // of which heads
  static constexpr int TURNS = 4, HEADS = ACROSS * TURNS;                         // of a block
  // tiles that L places from anywhere touch
  static int tiles(int L) { return (L + 2 * PLACES - 2) / PLACES; }
  // With a quarter of these heads a thread's turns go along the sequence instead, each with a page of its own.  bf16 into e4m3 and back, pages of 64: 53 sequences of 16336 tokens, 2 heads of 64
  // 286 us for 348, 8 of 16336, one head of 128 40 for 53; with half of them it is worse: 8 x 16336, 2 heads of 128 92 for 84, 53 x 16336, 4 heads of 64 572 for 521.
  static bool along(int HK, int L) { return 4 * HK <= HEADS && L >= 4 * PLACES; }
};
struct CacheRows {
  int B, L, HK;
  UDiv by_tiles, by_groups;      // tiles of a sequence, blocks with some of the heads
  const int* starts;             // [B], null: 0
};
// What a thread has in turn i: a head of a token (which may lie outside) and its place; keys or values.
template <typename T, int D, bool ALONG>
struct CacheRow {
  using A = CacheTile<T, D>;
  int b, h;
  long long start, first;
  bool values;
  const CacheRows& r;
  __device__ __forceinline__ explicit CacheRow(const CacheRows& r_) : r(r_) {
    const int row = threadIdx.x / A::G, half = r.by_groups.div(blockIdx.y);
    b = r.by_tiles.div(blockIdx.x);
    values = half != 0;
    h = (blockIdx.y - half * (int)r.by_groups.d) * (ALONG ? A::ACROSS : A::HEADS) + row / A::PLACES;
    start = r.starts ? r.starts[b] : 0;
    first = start - (start & (A::PLACES - 1)) + (long long)(blockIdx.x - b * (int)r.by_tiles.d) * (ALONG ? A::TURNS * A::PLACES : A::PLACES) + row % A::PLACES;
  }
  __device__ __forceinline__ int head(int i) const { return ALONG ? h : h + i * A::ACROSS; }
  __device__ __forceinline__ long long place(int i) const { return ALONG ? first + i * A::PLACES : first; }
  __device__ __forceinline__ int token(int i) const {      // -1: none
    const long long t = place(i) - start;
    return t < 0 || t >= r.L || head(i) >= r.HK ? -1 : (int)t;
  }
};

// k, v: [B, L, HK, D] of T.  Token t of sequence b goes to place starts[b] + t if t < counts[b].
template <typename T>
struct CacheWriteParams {
  Pages to;
  CacheRows rows;
  const T* k; const T* v;
  long long ldk, bsk, ldv, bsv;
  const int* counts;          // null: L
};

template <typename T, typename C, int D, bool ALONG>
__global__ __launch_bounds__(256) void k_cache_write(const CacheWriteParams<T> p) {
  using A = CacheTile<T, D>;
  constexpr int E = A::E, G = A::G, LOOKUPS = ALONG ? A::TURNS : 1;
  const CacheRow<T, D, ALONG> r(p.rows);
  const int lane = threadIdx.x % G, count = p.counts ? p.counts[r.b] : 0x7fffffff;
  int page[LOOKUPS], row[LOOKUPS];
#pragma unroll
  for (int i = 0; i < LOOKUPS; ++i) {
    const int t = r.token(i);
    page[i] = t >= 0 && t < count ? p.to.page(r.b, r.place(i)) : -1;
    row[i] = page[i] >= 0 ? p.to.row(r.place(i)) : 0;
  }
  const T* from = (r.values ? p.v : p.k) + r.b * (r.values ? p.bsv : p.bsk) + lane * E;
  const long long ld = r.values ? p.ldv : p.ldk;
  uint4 u[A::TURNS];
#pragma unroll
  for (int i = 0; i < A::TURNS; ++i) {
    u[i] = make_uint4(0, 0, 0, 0);
    if (page[i % LOOKUPS] >= 0 && r.token(i) >= 0) u[i] = *reinterpret_cast<const uint4*>(from + r.token(i) * ld + r.head(i) * D);
  }
  C* pages = static_cast<C*>(r.values ? p.to.v : p.to.k);
  uint8_t* exponents = r.values ? p.to.vs : p.to.ks;
  const long long stride = r.values ? p.to.v_page : p.to.k_page, estride = r.values ? p.to.vs_page : p.to.ks_page;
#pragma unroll
  for (int i = 0; i < A::TURNS; ++i) {
    const bool there = page[i % LOOKUPS] >= 0 && r.token(i) >= 0;
    const long long rows = p.to.rows_before(r.head(i), row[i % LOOKUPS]);
    C* to = pages + page[i % LOOKUPS] * stride + rows * D + lane * E;
    if constexpr (!is_e4m3<C>()) {
      if (there) *reinterpret_cast<uint4*>(to) = u[i];
    } else {
      float x[E];
      if constexpr (E == 8) {
        Elem<T>::unpack4(make_uint2(u[i].x, u[i].y), x);
        Elem<T>::unpack4(make_uint2(u[i].z, u[i].w), x + 4);
      } else {
        Elem<T>::unpack4(__builtin_bit_cast(float4, u[i]), x);
      }
      uint32_t top = 0;      // the largest finite magnitude
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const uint32_t m = __float_as_uint(x[j]) & 0x7fffffffu;
        if (m >= 0x7f800000u) x[j] = __uint_as_float(0x7fc00000u);
        else top = max(top, m);
      }
#pragma unroll
      for (int o = 1; o < G; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
      // 448 is 1.75 * 2^8
      const int e = max(0, (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0));
      const float f = __uint_as_float((uint32_t)(254 - e) << 23);      // e is at most 247
      uint32_t c[E / 4];
#pragma unroll
      for (int j = 0; j < E / 4; ++j) {
        const int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j] * f, x[4 * j + 1] * f, 0, false);
        c[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j + 2] * f, x[4 * j + 3] * f, w, true);
      }
      if (there) {
        if constexpr (E == 8) *reinterpret_cast<uint2*>(to) = make_uint2(c[0], c[1]);
        else *reinterpret_cast<uint32_t*>(to) = c[0];
        if (lane == 0) exponents[page[i % LOOKUPS] * estride + rows] = (uint8_t)e;
      }
    }
  }
}

// k, v: [B, L, HK, D] of T, contiguous: place starts[b] + t of sequence b, zeros from place lengths[b] on and where there is no page.
template <typename T>
struct CacheReadParams {
  Pages from;
  CacheRows rows;
  T* k; T* v;
  const int* lengths;
};

template <typename T, typename C, int D, bool ALONG>
__global__ __launch_bounds__(256) void k_cache_read(const CacheReadParams<T> p) {
  using A = CacheTile<T, D>;
  constexpr int E = A::E, G = A::G, LOOKUPS = ALONG ? A::TURNS : 1;
  const CacheRow<T, D, ALONG> r(p.rows);
  const int lane = threadIdx.x % G, length = p.lengths[r.b];
  int page[LOOKUPS], row[LOOKUPS];
#pragma unroll
  for (int i = 0; i < LOOKUPS; ++i) {
    page[i] = r.token(i) >= 0 && r.place(i) < length ? p.from.page(r.b, r.place(i)) : -1;
    row[i] = page[i] >= 0 ? p.from.row(r.place(i)) : 0;
  }
  const C* pages = static_cast<const C*>(r.values ? p.from.v : p.from.k);
  const uint8_t* exponents = r.values ? p.from.vs : p.from.ks;
  const long long stride = r.values ? p.from.v_page : p.from.k_page, estride = r.values ? p.from.vs_page : p.from.ks_page;
  T* to = (r.values ? p.v : p.k) + (long long)r.b * p.rows.L * p.rows.HK * D + lane * E;
  using Raw = typename std::conditional<!is_e4m3<C>(), uint4, typename std::conditional<E == 8, uint2, uint32_t>::type>::type;
  Raw u[A::TURNS];
  uint32_t e[A::TURNS];
#pragma unroll
  for (int i = 0; i < A::TURNS; ++i) {
    u[i] = Raw{};
    e[i] = 127;
    if (page[i % LOOKUPS] >= 0 && r.token(i) >= 0) {
      const long long rows = p.from.rows_before(r.head(i), row[i % LOOKUPS]);
      u[i] = *reinterpret_cast<const Raw*>(pages + page[i % LOOKUPS] * stride + rows * D + lane * E);
      if constexpr (is_e4m3<C>()) e[i] = exponents[page[i % LOOKUPS] * estride + rows];
    }
  }
#pragma unroll
  for (int i = 0; i < A::TURNS; ++i) {
    uint4 w;
    if constexpr (!is_e4m3<C>()) {
      w = u[i];
    } else if constexpr (E == 8) {
      const float s = e8m0(e[i]);
      auto two = [&](uint32_t c, auto high) LACT_INLINE_LAMBDA { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, s, decltype(high)::value)); };
      w = make_uint4(two(u[i].x, std::false_type()), two(u[i].x, std::true_type()), two(u[i].y, std::false_type()), two(u[i].y, std::true_type()));
    } else {
      const float s = e8m0(e[i]);
      const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[i], true);
      w = make_uint4(__float_as_uint(a[0] * s), __float_as_uint(a[1] * s), __float_as_uint(b[0] * s), __float_as_uint(b[1] * s));
    }
    if (r.token(i) >= 0) *reinterpret_cast<uint4*>(to + ((long long)r.token(i) * p.rows.HK + r.head(i)) * D) = w;
  }
}

}  // namespace lact
