// A cache of keys and values in pages: [pages, HK, page size, D] each, bf16, fp32 or e4m3.  A sequence's place n lies in page table[b][n / size] at row n % size; what
// points outside the pages is no page.  A row of e4m3 has an exponent beside it (e8m0, [pages, HK, page size]): the smallest e with which the row's largest finite
// magnitude is at most 448 2^(e - 127).  The scale is a power of two, so that a number loses nothing but what lies under e4m3's three bits, and what is read back is exact in bf16.
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

// ---- tokens into their places -----------------------------------------------------------------------
// k, v: [B, L, HK, D] of T.  Token t of sequence b goes to place starts[b] + t if t < counts[b].
template <typename T>
struct CacheWriteParams {
  Pages to;
  int B, L;
  UDiv by_l, by_heads;
  const T* k; const T* v;
  long long ldk, bsk, ldv, bsv;
  const int* starts;          // null: 0
  const int* counts;          // null: L
};

constexpr int CACHE_ROWS = 4;      // of a group of lanes, their loads in flight together

// A row is 16 bytes of T a lane; groups of lanes take rows of consecutive tokens of one head, which lie next to each other in their page, and whose exponents do.
template <typename T, typename C, int D>
__global__ __launch_bounds__(256) void k_cache_write(const CacheWriteParams<T> p) {
  constexpr int E = 16 / (int)sizeof(T), G = D / E, PER = 256 / G;
  const bool values = blockIdx.y != 0;
  const int lane = threadIdx.x % G, n = p.B * p.to.HK * p.L;
  const T* from = values ? p.v : p.k;
  const long long ld = values ? p.ldv : p.ldk, bs = values ? p.bsv : p.bsk;
  uint4 u[CACHE_ROWS];
  int page[CACHE_ROWS], row[CACHE_ROWS];
#pragma unroll
  for (int i = 0; i < CACHE_ROWS; ++i) {
    const long long r = ((long long)blockIdx.x * CACHE_ROWS + i) * PER + threadIdx.x / G;
    page[i] = -1;
    row[i] = 0;
    u[i] = make_uint4(0, 0, 0, 0);
    if (r >= n) continue;
    const int bh = p.by_l.div((int)r), t = (int)r - bh * p.L, b = p.by_heads.div(bh), h = bh - b * p.to.HK;
    if (p.counts && t >= p.counts[b]) continue;
    const long long place = (long long)(p.starts ? p.starts[b] : 0) + t;
    page[i] = p.to.page(b, place);
    if (page[i] < 0) continue;
    row[i] = p.to.rows_before(h, p.to.row(place));
    u[i] = *reinterpret_cast<const uint4*>(from + b * bs + t * ld + h * D + lane * E);
  }
  C* to = static_cast<C*>(values ? p.to.v : p.to.k);
  const long long stride = values ? p.to.v_page : p.to.k_page;
#pragma unroll
  for (int i = 0; i < CACHE_ROWS; ++i) {
    C* at = to + page[i] * stride + (long long)row[i] * D + lane * E;
    if constexpr (!is_e4m3<C>()) {
      if (page[i] >= 0) *reinterpret_cast<uint4*>(at) = u[i];
    } else {
      float x[E];
#pragma unroll
      for (int j = 0; j < E / 4; ++j) {
        if constexpr (E == 8) Elem<T>::unpack4(j ? make_uint2(u[i].z, u[i].w) : make_uint2(u[i].x, u[i].y), x + 4 * j);
        else Elem<T>::unpack4(__builtin_bit_cast(float4, u[i]), x);
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
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j] * f, x[4 * j + 1] * f, 0, false);
        c[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j + 2] * f, x[4 * j + 3] * f, w, true);
      }
      if (page[i] >= 0) {
        if constexpr (E == 8) *reinterpret_cast<uint2*>(at) = make_uint2(c[0], c[1]);
        else *reinterpret_cast<uint32_t*>(at) = c[0];
        if (lane == 0) (values ? p.to.vs : p.to.ks)[page[i] * (values ? p.to.vs_page : p.to.ks_page) + row[i]] = (uint8_t)e;
      }
    }
  }
}

// ---- and back -----------------------------------------------------------------------------------------
// k, v: [B, L, HK, D] of T, contiguous: place starts[b] + t of sequence b, zeros from place lengths[b] on and where there is no page.
template <typename T>
struct CacheReadParams {
  Pages from;
  int B, L;
  UDiv by_l, by_heads;
  T* k; T* v;
  const int* starts;          // null: 0
  const int* lengths;
};

template <typename T, typename C, int D>
__global__ __launch_bounds__(256) void k_cache_read(const CacheReadParams<T> p) {
  constexpr int E = 16 / (int)sizeof(T), G = D / E, PER = 256 / G;
  const bool values = blockIdx.y != 0;
  const int lane = threadIdx.x % G, n = p.B * p.from.HK * p.L;
  const C* from = static_cast<const C*>(values ? p.from.v : p.from.k);
  const uint8_t* exponents = values ? p.from.vs : p.from.ks;
  const long long stride = values ? p.from.v_page : p.from.k_page, estride = values ? p.from.vs_page : p.from.ks_page;
  T* to = values ? p.v : p.k;
  using Raw = typename std::conditional<!is_e4m3<C>(), uint4, typename std::conditional<E == 8, uint2, uint32_t>::type>::type;
  Raw u[CACHE_ROWS];
  uint32_t e[CACHE_ROWS];
  long long at[CACHE_ROWS];      // in the output, -1: no row
#pragma unroll
  for (int i = 0; i < CACHE_ROWS; ++i) {
    const long long r = ((long long)blockIdx.x * CACHE_ROWS + i) * PER + threadIdx.x / G;
    at[i] = -1;
    u[i] = Raw{};
    e[i] = 127;
    if (r >= n) continue;
    const int bh = p.by_l.div((int)r), t = (int)r - bh * p.L, b = p.by_heads.div(bh), h = bh - b * p.from.HK;
    at[i] = (((long long)b * p.L + t) * p.from.HK + h) * D + lane * E;
    const long long place = (long long)(p.starts ? p.starts[b] : 0) + t;
    const int page = place < p.lengths[b] ? p.from.page(b, place) : -1;
    if (page < 0) continue;
    const int row = p.from.rows_before(h, p.from.row(place));
    u[i] = *reinterpret_cast<const Raw*>(from + page * stride + (long long)row * D + lane * E);
    if constexpr (is_e4m3<C>()) e[i] = exponents[page * estride + row];
  }
#pragma unroll
  for (int i = 0; i < CACHE_ROWS; ++i) {
    if (at[i] < 0) continue;
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
    *reinterpret_cast<uint4*>(to + at[i]) = w;
  }
}

}  // namespace lact
