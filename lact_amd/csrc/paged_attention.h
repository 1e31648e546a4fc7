// Softmax attention of one new token of every sequence with keys and values in pages (paged_cache.h), head sizes 64 and 128; queries bf16 or fp32, pages of the
// same type or e4m3:
//
//   o_h = sum_j softmax_j(f(q_h . k_j / sqrt(D)) - slope_h (n - 1 - j)) v_j,   max(0, n - window) <= j < n,   f(x) = cap tanh(x / cap) or x
//
// over the places j that lie on a page; n = lengths[b], read on the device.  A sequence that sees nothing has output 0.
//
// The host does not know the lengths.  The work of all items, a key head of a sequence each (with up to 16 of its query heads, or 32 where it has more), in steps of 32
// places a wave, is cut into equal shares; what a block has of an item that it does not have as a whole, at most its first and its last, goes to the workspace
// unnormalised, and k_paged_join adds the parts in the blocks' order.  Where no sequence can have more than a few steps, a block has an item as a whole.
//
// A wave's step is 32 places from a multiple of 16 on: two pieces of 16 rows, each of which lies in one page, as page sizes are multiples of 16.  The wave looks up where
// the keys and the values of 32 pieces lie at once, a lane each, and copies a piece from where its lane says; one without a page is copied from zeros and masked.  In a
// piece that the window or the length ends in, the keys outside repeat one inside and the values outside are zeros (of 8 bits, which have no infinities, they repeat one too).
//
// e4m3: numbers become bf16 as they leave LDS, exactly down to multiples of 2^-133.  A key's exponent is applied in that conversion (a lane has one key's row), a value's to
// the weight that meets it.  fp32 queries and weights meet them in three bf16 parts of 8 bits.  (Products below 2^-126 count as 0: values under 2^-118.)
//
// Nothing is rounded to fewer bits in front of the output but the weights of bf16 queries, which meet the values in two bf16 parts: 2^-15 of each.  In one part (2^-8) outputs of 131072 places
// were off by 2.3e-3 of their norm where rounding them alone costs 1.7e-3; the second costs 1 % of a long case and 0.4-1.2 us of short ones (16 sequences of up to 1000: 12.4 -> 13.6).
//
// What bounds it is the one read of the keys and values.  131072 places of 8 heads of 128 with 4 queries each in bf16: 95 us and 6.5 for the join, 5.6 and 5.3 TB/s (a large copy
// reaches 5.0); 64 sequences of up to 16384 in e4m3, 5 queries each: 172 + 7 us, 5.3 TB/s; 32 of up to 8192 with a cap and a distance: 55 + 5 us, 4.6 TB/s: what lies between two
// items.  The pages' size and order make no difference (16 to 256 places: 2 %).  One block to a compute unit in 8 bits, with a ring twice as deep: 68 us instead of 61 in the last of
// these, 184 instead of 178 in the one before, with heads of 64 44 instead of 36.
#pragma once
#include "attention_step.h"
#include "paged_cache.h"

namespace lact {

template <typename T>
struct PagedStepParams {
  Pages kv;
  int B, N, H, HK, group, window;            // N: places of a sequence
  int columns, tiles;                        // query heads that a block works for at once, 16 or 32; how often a key head's
  int blocks, whole;                         // of the main kernel; whether each has one item, whose steps are few
  const T* q; long long bsq;
  const int* lengths;
  const float* slopes;
  float scale, cap;
  T* out;
  float* part;
  __device__ __forceinline__ int length(int b) const { return b < B ? min(max(lengths[b], 0), N) : 0; }
  __device__ __forceinline__ int first(int len) const { return max(0, len - window); }
  template <int KEYS>
  __device__ __forceinline__ int steps(int len) const { return (len - (first(len) & ~15) + KEYS - 1) / KEYS; }
  __device__ __forceinline__ int rows() const { return min(group, columns); }      // of a part
  __device__ __forceinline__ int first_head(int item) const { return item / tiles * group + item % tiles * columns; }
  // what a block left of the item that its share begins in, or of its last one
  template <int D>
  __device__ __forceinline__ float* part_of(int block, bool head) const { return part + (size_t)(2 * block + (head ? 0 : 1)) * rows() * (D + 2); }
  __device__ __forceinline__ static float mean(float sum, float weights) { return weights == 0.f ? 0.f : sum / weights; }
};

// of numbers that are not negative and the same for the whole wave
__device__ __forceinline__ long long quotient(long long a, long long b) { return same((a | b) >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b)); }

// inclusive sums over the wave
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);      // one lane up, two, four, eight, inside rows of 16
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);      // the last lane of a row to the next one, of the first two rows to the others
  return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
}

// What a new item costs a block, in steps: the ring runs empty, parts are joined, pages looked up, the ring fills.  In the row of all items 0 / 1 / 2 / 3 / 6 for it: 32 sequences of up to
// 8192 places, 8 heads of 128, e4m3 69 / 61 / 61 / 62 / 64 us, bf16 113 / 99 / 96 / 97 / 98; 64 of up to 16384, e4m3 178 / 178 / 179 / 177 / 182.
constexpr int PAGED_START = 2;

// The work of all items in a row: sequence by sequence, each of whose `items` costs the same, its steps and PAGED_START in front of them.  Shares differ by one at most.  Every
// wave computes it for itself, 64 sequences at a time, whose lengths stay with its lanes.
template <int KEYS, typename P>
struct PagedWork {
  const P& p;
  int items, blocks, more;           // blocks with a share: none is empty; the first `more` have one more
  long long total, per;
  int b0, len, sum;                  // the lanes' sequences from b0 on: lengths, and what one item of each up to and with them costs
  __device__ __forceinline__ explicit PagedWork(const P& p_) : p(p_), items(p_.HK * p_.tiles) {}
  __device__ __forceinline__ void load(int from) {
    b0 = from;
    len = p.length(b0 + (int)(threadIdx.x & 63));
    sum = wave_scan(cost(p.template steps<KEYS>(len)));
  }
  __device__ __forceinline__ static int cost(int steps) { return steps ? steps + PAGED_START : 0; }
  __device__ __forceinline__ int of_all() const { return __builtin_amdgcn_readlane(sum, 63); }
  __device__ __forceinline__ void init() {
    total = 0;
    for (int b = 0; b < p.B; b += 64) {
      load(b);
      total += of_all();
    }
    total *= items;
    blocks = (int)min((long long)p.blocks, total);
    per = blocks ? quotient(total, blocks) : 0;
    more = (int)(total - per * blocks);
  }
  __device__ __forceinline__ long long share(int block) const { return block * per + min(block, more); }
  __device__ __forceinline__ int block_of(long long s) const {
    const long long longer = (per + 1) * more;
    return s < longer ? (int)quotient(s, per + 1) : more + (int)quotient(s - longer, per);
  }
  __device__ __forceinline__ int length(int b) {
    if (b < b0 || b >= b0 + 64) load(b & ~63);
    return __builtin_amdgcn_readlane(len, b - b0);
  }
  // where place s < total of the row lies: sequence, item, place in the item, and how many steps its items have.  (Lengths that somebody changes meanwhile make no sense, but nothing here
  // leaves the batch, the heads or the workspace for it.)
  __device__ __forceinline__ void find(long long s, int& b, int& item, int& at, int& n) {
    const long long x = quotient(s, items);      // in a row of one item of each
    long long before = 0;
    if (p.B > 64) load(0);
    for (;;) {
      const uint64_t past = __ballot(x - before < sum);
      if (past || b0 + 64 >= p.B) {
        const int i = past ? __ffsll((unsigned long long)past) - 1 : p.B - 1 - b0;
        b = b0 + i;
        n = max(1, p.template steps<KEYS>(__builtin_amdgcn_readlane(len, i)));
        const long long in_b = max(0LL, s - (before + __builtin_amdgcn_readlane(sum, i) - cost(n)) * items);
        item = (int)min((long long)items - 1, quotient(in_b, cost(n)));
        at = (int)min((long long)cost(n) - 1, in_b - (long long)item * cost(n));
        return;
      }
      before += of_all();
      load(b0 + 64);
    }
  }
};

static __device__ const uint4 paged_zeros[512] = {};      // a piece of any type

// 32 keys or values as they lie in LDS: the 16-byte granule g of row r at slot g ^ key(r).  The keys spread over the banks what is read at once: a granule of 16 rows, and of the transposed
// reads four rows from a multiple of four on (two neighbouring granules each), with 8 bits these and the four 16 rows further on (one granule).
template <typename C, int D>
struct PagedTile {
  static constexpr int ROWB = D * (int)sizeof(C), G = ROWB / 16, BYTES = 32 * ROWB, COPIES = BYTES / 1024;
  __device__ static __forceinline__ int key(int r) {
    if constexpr (is_e4m3<C>()) return D == 128 ? ((r >> 1) & 7) ^ (r >> 4 << 2) : ((r >> 2) & 3) ^ (r >> 4 << 1);
    else if constexpr (sizeof(C) == 2) return AttnTile<D>::key(r);
    else return r & 15;
  }
};
template <typename T, typename C, int D>
struct PagedShape {
  using S = PagedTile<C, D>;
  static constexpr int NW = 4;                                               // waves, each with a ring of its own
  static constexpr int BLOCKS = sizeof(C) * D >= 256 ? 1 : 2;                // to a compute unit
  static constexpr int STAGE = 2 * S::BYTES;
  static constexpr int RING = 131072 / (BLOCKS * NW * STAGE);
  static constexpr int EXP = is_e4m3<C>() ? 1024 : 0;                        // exponents of 32 pieces of keys and of values, twice
  static constexpr int WAVE = RING * STAGE + 2 * EXP;
  static constexpr int KEYS = 32 * NW;                                       // of a step
  static constexpr int LDS = NW * WAVE;
  // A block has an item as a whole, and no second launch, where the longest has no more steps.  Against shares: 64 sequences of up to 1000 places, 8 heads of 128, e4m3 19.9 us for 22.6, bf16 32.8
  // for 32.7; 16 of up to 1000 in bf16 13.6 for 16.1, of up to 500 9.6 for 13.7; 4 steps of fp32, one sequence of 500, 12 heads of 64 10.8 for 13.0, 64 of up to 500 of 8 heads of 128 40.0 for
  // 41.4, but 8 steps 17.6 for 12.9 (its products take longer).
  static constexpr int WHOLE = sizeof(C) == 4 ? 4 : 8;
};

// Products of 16 x 16: a wave's 32 keys in two tiles as rows, QT tiles of 16 query heads as columns.  A lane has the keys 16 kt + 4 h + i (h = lane / 16) of column
// lane % 16, and what it has of them is the second operand of the next product as it lies: its k slots stand for the same keys on both sides.
__device__ __forceinline__ f32x4 mma16(const bf16x8& a, const bf16x8& b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma16(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
template <int QT> struct PagedScores { f32x4 s[QT][2]; };

// The leading bf16 part of eight numbers, which keep the rest.
__device__ __forceinline__ bf16x8 bf16_part(float (&x)[8]) {
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
    x[2 * i] -= bf16_lo(r[i]);
    x[2 * i + 1] -= bf16_hi(r[i]);
  }
  return __builtin_bit_cast(bf16x8, make_uint4(r[0], r[1], r[2], r[3]));
}
// All eight as parts, the leading one first.
template <int N>
__device__ __forceinline__ void bf16_parts(const f32x4 (&x)[2], bf16x8 (&p)[N]) {
  float y[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = x[j / 4][j % 4];
#pragma unroll
  for (int i = 0; i < N; ++i) p[i] = bf16_part(y);
}
// bf16 queries: a weight, which may be anything, in two parts of 8 bits, so that what is stored is the only rounding that shows (2^-15 of a weight against 2^-8).
constexpr int WEIGHT_PARTS = 2;
// The two for values that may be infinite: the leading part is cut below the weight, so that both are positive, and none of a weight that is not 0 is 0.
__device__ __forceinline__ void positive_parts(const f32x4 (&x)[2], bf16x8 (&p)[WEIGHT_PARTS]) {
  uint32_t lead[4], rest[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = x[i / 2][2 * i % 4], b = x[i / 2][2 * i % 4 + 1];
    const uint32_t c = __builtin_elementwise_sub_sat(__float_as_uint(a), 1u), d = __builtin_elementwise_sub_sat(__float_as_uint(b), 1u);
    lead[i] = __builtin_amdgcn_perm(d, c, 0x07060302u);      // their upper halves
    rest[i] = pack_bf16(a - __uint_as_float(c & 0xffff0000u), b - __uint_as_float(d & 0xffff0000u));
  }
  p[0] = __builtin_bit_cast(bf16x8, make_uint4(lead[0], lead[1], lead[2], lead[3]));
  p[1] = __builtin_bit_cast(bf16x8, make_uint4(rest[0], rest[1], rest[2], rest[3]));
}

template <typename T, typename C, int D, int QT> struct PagedMath;
template <int D, int QT>
struct PagedMath<uint16_t, uint16_t, D, QT> {
  using S = PagedTile<uint16_t, D>;
  bf16x8 q[QT][D / 32];
  uint32_t row, row_key, col[D / 16];
  __device__ __forceinline__ void init() {
    const int l = threadIdx.x & 63, h = l >> 4, r = 4 * h + ((l & 15) >> 2);
    row = (l & 15) * S::ROWB;
    row_key = (uint32_t)(S::key(l & 15) ^ h) << 4;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) col[dt] = r * S::ROWB + (((dt * 2 + ((l & 3) >> 1)) ^ S::key(r)) << 4) + (l & 1) * 8;
  }
  __device__ __forceinline__ void query(int t, const uint16_t* at) {
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks) q[t][ks] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(at + ks * 32 + 8 * ((threadIdx.x & 63) >> 4)));
  }
  __device__ __forceinline__ void arrived() {
#pragma unroll
    for (int t = 0; t < QT; ++t) attn_arrived(q[t]);
  }
  __device__ __forceinline__ void scores(PagedScores<QT>& x, const char* tile, const char*) const {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks) {
        // (rows 16 further on: the key is the same)
        const bf16x8 k = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(tile + kt * 16 * S::ROWB + row + ((uint32_t)(ks * 64) ^ row_key)));
#pragma unroll
        for (int t = 0; t < QT; ++t) x.s[t][kt] = mma16(k, q[t][ks], x.s[t][kt]);
      }
  }
  __device__ __forceinline__ uint2 value_exponents(const char*) const { return uint2{}; }
  __device__ __forceinline__ void weigh(PagedScores<QT>&, const uint2&) const {}
  __device__ __forceinline__ void add(f32x4 (&o)[QT][D / 16], const PagedScores<QT>& x, const char* tile) const {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    bf16x8 p[QT][WEIGHT_PARTS];
#pragma unroll
    for (int t = 0; t < QT; ++t) positive_parts(x.s[t], p[t]);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + col[dt]));
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + col[dt] + 16 * S::ROWB));
      const bf16x8 v = __builtin_bit_cast(bf16x8, (s16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}));
#pragma unroll
      for (int i = WEIGHT_PARTS - 1; i >= 0; --i)
#pragma unroll
        for (int t = 0; t < QT; ++t) o[t][dt] = mma16(v, p[t][i], o[t][dt]);
    }
  }
};
template <int D, int QT>
struct PagedMath<float, float, D, QT> {
  using S = PagedTile<float, D>;
  f32x4 q[QT][D / 16];
  uint32_t row, row_key, col[4];
  __device__ __forceinline__ void init() {
    const int l = threadIdx.x & 63, h = l >> 4;
    row = (l & 15) * S::ROWB;
    row_key = (uint32_t)(S::key(l & 15) ^ h) << 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) col[i] = (4 * h + i) * S::ROWB + (((((l & 15) >> 2) ^ S::key(4 * h + i)) << 4) | ((l & 3) << 2));
  }
  __device__ __forceinline__ void query(int t, const float* at) {
#pragma unroll
    for (int m = 0; m < D / 16; ++m) q[t][m] = *reinterpret_cast<const f32x4*>(at + m * 16 + 4 * ((threadIdx.x & 63) >> 4));
  }
  __device__ __forceinline__ void arrived() {
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int m = 0; m < D / 16; ++m) asm volatile("" : "+v"(q[t][m]));
  }
  __device__ __forceinline__ void scores(PagedScores<QT>& x, const char* tile, const char*) const {
#pragma unroll
    for (int m = 0; m < D / 16; ++m)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const f32x4 k = *reinterpret_cast<const f32x4*>(tile + kt * 16 * S::ROWB + row + ((uint32_t)(m * 64) ^ row_key));
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int t = 0; t < QT; ++t) x.s[t][kt] = mma16(k[j], q[t][m][j], x.s[t][kt]);
      }
  }
  __device__ __forceinline__ uint2 value_exponents(const char*) const { return uint2{}; }
  __device__ __forceinline__ void weigh(PagedScores<QT>&, const uint2&) const {}
  __device__ __forceinline__ void add(f32x4 (&o)[QT][D / 16], const PagedScores<QT>& x, const char* tile) const {
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = *reinterpret_cast<const float*>(tile + kt * 16 * S::ROWB + (dt / 4) * 256 + (col[i] ^ (uint32_t)((dt & 3) << 6)));
#pragma unroll
          for (int t = 0; t < QT; ++t) o[t][dt] = mma16(v, x.s[t][kt][i], o[t][dt]);
        }
  }
};
// e4m3.  Of every 64 columns a lane takes the 16 from 16 h on, eight for each of two products, in one read; the queries' fragments follow that.  fp32 queries and weights are
// three bf16 parts, 24 bits in all.
template <typename T, int D, int QT>
struct PagedMath<T, uint8_t, D, QT> {
  static constexpr int PARTS = sizeof(T) == 4 ? 3 : 1;
  using S = PagedTile<uint8_t, D>;
  bf16x8 q[QT][PARTS][D / 32];
  uint32_t row[2], col[D / 16];
  __device__ __forceinline__ void init() {
    const int l = threadIdx.x & 63, h = l >> 4, rr = (l & 15) >> 1, r = 16 * (rr >> 2) + 4 * h + (rr & 3);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) row[kt] = (kt * 16 + (l & 15)) * S::ROWB + ((S::key(kt * 16 + (l & 15)) ^ h) << 4);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) col[dt] = r * S::ROWB + ((dt ^ S::key(r)) << 4) + (l & 1) * 8;
  }
  __device__ __forceinline__ void query(int t, const T* base) {
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks) {
      const T* at = base + (ks >> 1) * 64 + 16 * ((threadIdx.x & 63) >> 4) + (ks & 1) * 8;
      if constexpr (PARTS == 1) {
        q[t][0][ks] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(at));
      } else {
        float x[8];
        Elem<T>::load4(at, x);
        Elem<T>::load4(at + 4, x + 4);
#pragma unroll
        for (int i = 0; i < PARTS; ++i) q[t][i][ks] = bf16_part(x);
      }
    }
  }
  __device__ __forceinline__ void arrived() {
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int i = 0; i < PARTS; ++i) attn_arrived(q[t][i]);
  }
  __device__ __forceinline__ static bf16x8 widen(uint32_t a, uint32_t b, float scale) {
    return __builtin_bit_cast(bf16x8, make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, false)),
                                                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, true)),
                                                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, false)),
                                                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, true))));
  }
  __device__ __forceinline__ void scores(PagedScores<QT>& x, const char* tile, const char* exps) const {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      // (the conversion takes its exponent bits alone)
      const float scale = __uint_as_float((uint32_t)*reinterpret_cast<const uint8_t*>(exps + kt * 16 + (threadIdx.x & 15)) << 23);
#pragma unroll
      for (int m = 0; m < D / 64; ++m) {
        const uint4 u = *reinterpret_cast<const uint4*>(tile + (row[kt] ^ (uint32_t)(m * 64)));
        const bf16x8 a = widen(u.x, u.y, scale), b = widen(u.z, u.w, scale);
#pragma unroll
        for (int i = PARTS - 1; i >= 0; --i)      // the smaller ones first
#pragma unroll
          for (int t = 0; t < QT; ++t) {
            x.s[t][kt] = mma16(a, q[t][i][2 * m], x.s[t][kt]);
            x.s[t][kt] = mma16(b, q[t][i][2 * m + 1], x.s[t][kt]);
          }
      }
    }
  }
  // of the lane's eight values, in the order of its weights
  __device__ __forceinline__ uint2 value_exponents(const char* exps) const {
    const uint32_t* e = reinterpret_cast<const uint32_t*>(exps + 512 + 4 * ((threadIdx.x & 63) >> 4));
    return make_uint2(e[0], e[4]);
  }
  __device__ __forceinline__ void weigh(PagedScores<QT>& x, const uint2& exps) const {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {      // an exponent of 255, which stands for NaN, is infinity here: what the weight's leading part leaves of it is NaN
        const uint32_t w = kt ? exps.y : exps.x, f = (i == 3 ? w >> 1 : w << (23 - 8 * i)) & 0x7f800000u;
#pragma unroll
        for (int t = 0; t < QT; ++t) x.s[t][kt][i] *= __uint_as_float(max(f, 0x400000u));
      }
  }
  __device__ __forceinline__ void add(f32x4 (&o)[QT][D / 16], const PagedScores<QT>& x, const char* tile) const {
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
    constexpr int WEIGHTS = PARTS == 1 ? WEIGHT_PARTS : PARTS;
    bf16x8 p[QT][WEIGHTS];
#pragma unroll
    for (int t = 0; t < QT; ++t) bf16_parts(x.s[t], p[t]);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
      const i32x2 c = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(tile + col[dt]));
      const bf16x8 v = widen((uint32_t)c[0], (uint32_t)c[1], 1.f);
#pragma unroll
      for (int i = WEIGHTS - 1; i >= 0; --i)
#pragma unroll
        for (int t = 0; t < QT; ++t) o[t][dt] = mma16(v, p[t][i], o[t][dt]);
    }
  }
};

// A lane's scores of one tile of queries as Scores has them, `first`: its first key's place minus its row's.
template <typename T, int BENT>
__device__ __forceinline__ void bend(const Scores<T, BENT>& sc, f32x4 (&s)[2], int first) {
  if constexpr (BENT == SCORES_PLAIN) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float x = s[j / 4][j % 4], slope;
    if (!sc.cap) x *= sc.c;
    else if constexpr (Scores<T, BENT>::QUICK) x = fmaf(__builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * sc.k1)), -2.f * sc.k2, sc.k2);
    else x = sc.capped(x, slope);
    s[j / 4][j % 4] = x;
  }
  if (!sc.bias) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) s[j / 4][j % 4] = fmaf(fabsf((float)first + (float)(16 * (j / 4) + j % 4)), -sc.slope, s[j / 4][j % 4]);
}

// 16 bytes per lane to LDS from where each lane says: lane i lands at lds_base + 16 * i
__device__ __forceinline__ void dma16_from(uint64_t at, uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\t" ::"s"(lds_base), "v"(at) : "memory", "m0");
}

template <typename T, typename C, int D, int QT, int BENT>
__global__ __launch_bounds__((64 * PagedShape<T, C, D>::NW), (sizeof(T) == 4 && D == 128 && QT == 2 ? 1 : 2)) void k_paged_step(const PagedStepParams<T> p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  using A = PagedShape<T, C, D>;
  using S = PagedTile<C, D>;
  constexpr int NW = A::NW, RING = A::RING, NC = S::COPIES, HALF = NC / 2, BATCH = 16;      // copies of a wave for 32 keys; tiles that it looks up at once
  static_assert(RING <= BATCH, "one batch holds what is on its way");
  prefetch_args<sizeof(p)>();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  PagedWork<A::KEYS, PagedStepParams<T>> work(p);
  const int items = work.items;
  // the block's share: from place `at` of this item of sequence b on
  int b, item, at, n;
  long long left;
  if (p.whole) {
    b = blockIdx.x / items;
    item = blockIdx.x - b * items;
    at = 0;
    work.load(b);
    n = p.template steps<A::KEYS>(__builtin_amdgcn_readlane(work.len, 0));
    left = work.cost(n);
    if (n == 0) {
      const int h0 = p.first_head(item), rows = min(16 * QT, (item / p.tiles + 1) * p.group - h0);
      for (int i = threadIdx.x; i < rows * D; i += 64 * NW) Elem<T>::store(p.out + ((size_t)b * p.H + h0) * D + i, 0.f);
      return;
    }
  } else {
    work.init();
    // sequences without a step: nobody else writes their outputs
    for (int i = blockIdx.x; i < p.B; i += gridDim.x)
      if (p.template steps<A::KEYS>(work.length(i)) == 0)
        for (int j = threadIdx.x; j < p.H * D; j += 64 * NW) Elem<T>::store(p.out + (size_t)i * p.H * D + j, 0.f);
    if ((int)blockIdx.x >= work.blocks) return;
    const long long s0 = work.share(blockIdx.x);
    left = work.share(blockIdx.x + 1) - s0;
    work.find(s0, b, item, at, n);
  }
  const uint32_t ring = lds_addr(smem) + wave * A::WAVE;
  const char* mine = smem + wave * A::WAVE;
  PagedMath<T, C, D, QT> math;
  math.init();
  int crow[NC];
  uint32_t ccol[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = i * 64 + lane, r = c / S::G;
    crow[i] = r & 15;
    ccol[i] = (uint32_t)((c % S::G) ^ S::key(r)) * 16;
  }
  bool head_of_share = true;
  while (left > 0) {
    const int end = (int)min((long long)work.cost(n), at + left), step0 = max(0, at - PAGED_START), step1 = end - PAGED_START;
    if (step1 <= step0) return;      // (the share ends in front of the item's first step)
    const int hk = item / p.tiles, h0 = p.first_head(item), rows = min(16 * QT, (hk + 1) * p.group - h0);
    const int len = work.length(b), lo = p.first(len), lo16 = lo & ~15;
    // the wave's tiles: 32 places from place(t) on
    auto place = [&](int t) LACT_INLINE_LAMBDA { return lo16 + ((step0 + t) * NW + wave) * 32; };
    const int tiles = min(step1 - step0, max(0, (len - lo16 - wave * 32 - step0 * A::KEYS + A::KEYS - 1) / A::KEYS));
    // Where the 32 pieces of 16 tiles from a multiple of 16 on lie, keys in the first half of the lanes, values in the second; which have a page, of this batch and the one
    // before it.
    uint32_t from_lo = 0, from_hi = 0, there = 0, there_before = 0;
    int batch = 0;      // the newest
    auto look_up = [&](int t) LACT_INLINE_LAMBDA {
      const int at = place(t + (lane & 31) / 2) + (lane & 1) * 16, page = at < len ? p.kv.page(b, at) : -1;
      const long long row = page >= 0 ? p.kv.rows_before(hk, p.kv.row(at)) : 0;
      const bool values = lane >= 32;
      const uint64_t zeros = reinterpret_cast<uint64_t>(paged_zeros);
      const uint64_t from = page < 0 ? zeros
                                     : reinterpret_cast<uint64_t>(values ? p.kv.v : p.kv.k) + (page * (values ? p.kv.v_page : p.kv.k_page) + row * D) * (long long)sizeof(C);
      if constexpr (A::EXP)
        dma16_from(page < 0 ? zeros : reinterpret_cast<uint64_t>(values ? p.kv.vs : p.kv.ks) + page * (values ? p.kv.vs_page : p.kv.ks_page) + row,
                   ring + RING * A::STAGE + (t / BATCH & 1) * A::EXP);
      from_lo = (uint32_t)from;
      from_hi = (uint32_t)(from >> 32);
      there_before = there;
      there = (uint32_t)__ballot(page >= 0);
    };
    auto copy = [&](int t, int half, uint32_t to) LACT_INLINE_LAMBDA {
      const int k0 = place(t);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int at = half + 2 * (t % BATCH) + x, first = lo - (k0 + 16 * x), last = max(0, len - 1 - (k0 + 16 * x));
        uint64_t address = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(from_lo, at) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane(from_hi, at) << 32;
        asm volatile("s_nop 4" : "+s"(address));      // between a scalar register's write by a vector instruction and its use as an address, which the compiler does not see
        const void* from = reinterpret_cast<const void*>(address);
        if (!A::EXP && half && (first > 0 || last < 15)) {      // values: zeros, as 0 times an infinity that is seen is NaN (8 bits have none)
#pragma unroll
          for (int i = x * HALF; i < (x + 1) * HALF; ++i)
            dma16_from((crow[i] < first || crow[i] > last ? reinterpret_cast<uint64_t>(paged_zeros) : address + (uint32_t)crow[i] * S::ROWB) + ccol[i], to + i * 1024);
        } else {
#pragma unroll
          for (int i = x * HALF; i < (x + 1) * HALF; ++i) dma16<false>(from, (uint32_t)min(max(crow[i], first), last) * S::ROWB + ccol[i], to + i * 1024);
        }
      }
    };
    auto keys = [&](int t) LACT_INLINE_LAMBDA { copy(t, 0, ring + t % RING * A::STAGE); };
    auto values = [&](int t) LACT_INLINE_LAMBDA { copy(t, 32, ring + t % RING * A::STAGE + S::BYTES); };
    Scores<T, BENT> sc[QT];
#pragma unroll
    for (int x = 0; x < QT; ++x) {
      const int h = h0 + min(x * 16 + (lane & 15), rows - 1);
      math.query(x, p.q + b * p.bsq + (long long)h * D);
      sc[x].init(p.scale, p.cap, p.slopes, h);
    }
    const float c = sc[0].unit();
    // no barrier: nobody else uses the wave's ring
    if (tiles > 0) look_up(0);
#pragma unroll
    for (int t = 0; t < RING; ++t)
      if (t < tiles) {
        keys(t);
        values(t);
      }
    math.arrived();
    f32x4 o[QT][D / 16];
    float mc[QT], sum[QT];
#pragma unroll
    for (int x = 0; x < QT; ++x) {
      mc[x] = ATTN_LOWEST;
      sum[x] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[x][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int t = 0; t < tiles; ++t) {
      const bool more = t + RING < tiles, full = t + RING <= tiles;
      if (full) wait_vmcnt<(2 * RING - 1) * NC>();
      else wait_vmcnt<0>();
      const char* kt = mine + t % RING * A::STAGE;
      const char* vt = kt + S::BYTES;
      const char* et = mine + RING * A::STAGE + (t / BATCH & 1) * A::EXP + t % BATCH * 32;
      const int k0 = place(t), mine0 = k0 + 4 * (lane >> 4);      // the lane's first key
      const int on_pages = (t / BATCH == batch ? there : there_before) >> (2 * (t % BATCH)) & 3;      // of the two pieces
      const bool masked = k0 < lo || k0 + 32 > len || on_pages != 3;
      PagedScores<QT> s;
#pragma unroll
      for (int x = 0; x < 2 * QT; ++x) s.s[x / 2][x % 2] = f32x4{0.f, 0.f, 0.f, 0.f};
      math.scores(s, kt, et);
      const auto exps = math.value_exponents(et);
      wave_reads_done();
      if (more) {
        if ((t + RING) % BATCH == 0) {
          look_up(t + RING);
          ++batch;
        }
        keys(t + RING);
      }
      auto mask = [&](float nothing) LACT_INLINE_LAMBDA {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = mine0 + 16 * kt + i;
            const bool seen = key >= lo && key < len && (on_pages >> kt & 1);
#pragma unroll
            for (int x = 0; x < QT; ++x) s.s[x][kt][i] = seen ? s.s[x][kt][i] : nothing;
          }
      };
#pragma unroll
      for (int x = 0; x < QT; ++x) bend(sc[x], s.s[x], mine0 - (len - 1));
      if (masked) mask(-__builtin_inff());
#pragma unroll
      for (int x = 0; x < QT; ++x) {
        f32x4(&a)[2] = s.s[x];
        float mx = max3(max3(a[0][0], a[0][1], a[0][2]), max3(a[0][3], a[1][0], a[1][1]), max3(a[1][2], a[1][3], a[1][3])) * c;
        // The maximum only has to keep the powers in range: it follows the row when it is exceeded by more than 2^8.
        if (__any(mx > mc[x] + 8.f)) {
          mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
          mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
          const float nm = mx > mc[x] + 8.f ? mx : mc[x], f = __builtin_amdgcn_exp2f(mc[x] - nm);
          mc[x] = nm;
          sum[x] *= f;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) o[x][i] *= f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          a[j / 4][j % 4] = __builtin_amdgcn_exp2f(fmaf(a[j / 4][j % 4], c, -mc[x]));
          sum[x] += a[j / 4][j % 4];
        }
      }
      if constexpr (A::EXP) {
        math.weigh(s, exps);
        if (masked) mask(0.f);      // (whatever exponent lies beside a row that nobody sees)
      }
      if (more) wait_vmcnt<(2 * RING - 1) * NC>();
      else wait_vmcnt<0>();
      math.add(o, s, vt);
      wave_reads_done();
      if (more) values(t + RING);
    }
    const bool whole = step0 == 0 && step1 == n;
    // The waves' parts together: sums at their place in each one's ring, [row][D + 4], maximum and row sum behind them.
    constexpr int LD = D + 4, WSTRIDE = A::WAVE / 4;
    static_assert(16 * QT * LD * 4 <= A::WAVE, "a wave's part fits its memory");
    float* w = reinterpret_cast<float*>(smem + wave * A::WAVE);
#pragma unroll
    for (int x = 0; x < QT; ++x) {
      sum[x] += __shfl_xor(sum[x], 16, 64);
      sum[x] += __shfl_xor(sum[x], 32, 64);
      const int r = x * 16 + (lane & 15);
      if (r < rows) {
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) Elem<float>::store4(w + r * LD + dt * 16 + 4 * (lane >> 4), o[x][dt][0], o[x][dt][1], o[x][dt][2], o[x][dt][3]);
        if (lane < 16) {
          w[r * LD + D] = mc[x];
          w[r * LD + D + 1] = sum[x];
        }
      }
    }
    __syncthreads();
    T* out = p.out + ((size_t)b * p.H + h0) * D;
    float* part = p.template part_of<D>(blockIdx.x, head_of_share);
    for (int i = threadIdx.x; i < rows * D; i += 64 * NW) {
      const int r = i / D, d = i % D;
      const float* src = reinterpret_cast<const float*>(smem) + r * LD;
      float m = src[D];
#pragma unroll
      for (int x = 1; x < NW; ++x) m = fmaxf(m, src[x * WSTRIDE + D]);
      float acc = 0.f, total = 0.f;
#pragma unroll
      for (int x = 0; x < NW; ++x) {
        const float f = __builtin_amdgcn_exp2f(src[x * WSTRIDE + D] - m);
        acc += src[x * WSTRIDE + d] * f;
        total += src[x * WSTRIDE + D + 1] * f;
      }
      if (whole) {
        Elem<T>::store(out + (size_t)r * D + d, p.mean(acc, total));
      } else {
        part[r * (D + 2) + d] = acc;
        if (d == 0) {
          part[r * (D + 2) + D] = m;
          part[r * (D + 2) + D + 1] = total;
        }
      }
    }
    __syncthreads();      // the rings are free again
    head_of_share = false;
    left -= end - at;
    at = 0;
    if (++item == items) {
      item = 0;
      do {
        if (++b >= p.B) return;
      } while ((n = p.template steps<A::KEYS>(work.length(b))) == 0);
    }
  }
}

// Joins what blocks left of an item that they share.  A block (x, y): row y of the item that share x + 1 begins inside, behind its first step, if share x does not as well.
// THREADS: 512 where items have many parts, so that each reads few (256 parts of one sequence: 7 us, bound by the launch and the way to them), else 128.
template <typename T, int D, int KEYS, int THREADS>
__global__ __launch_bounds__(THREADS) void k_paged_join(const PagedStepParams<T> p) {
  constexpr int GROUPS = THREADS / D;
  __shared__ float acc_s[GROUPS][D], sum_s[GROUPS], max_s[GROUPS];
  PagedWork<KEYS, PagedStepParams<T>> work(p);
  work.init();
  const int first = blockIdx.x;
  if (first + 1 >= work.blocks) return;
  const long long next = work.share(first + 1);
  int b, item, at, n;
  work.find(next, b, item, at, n);
  const long long begin = next - at;
  if (at <= PAGED_START || work.share(first) > begin + PAGED_START) return;
  const int h = p.first_head(item) + (int)blockIdx.y;
  if (h >= (item / p.tiles + 1) * p.group) return;
  const int last = min(work.blocks - 1, work.block_of(begin + work.cost(n) - 1));
  auto part = [&](int i) { return p.template part_of<D>(i, i != first || work.share(i) >= begin) + blockIdx.y * (D + 2); };
  // each group of D threads goes through its parts once, with a maximum of its own
  const int grp = threadIdx.x / D, d = threadIdx.x % D;
  float m = ATTN_LOWEST, acc = 0.f, total = 0.f;
#pragma unroll 4
  for (int i = first + grp; i <= last; i += GROUPS) {
    const float* x = part(i);
    const float nm = fmaxf(m, x[D]), f = __builtin_amdgcn_exp2f(m - nm), w = __builtin_amdgcn_exp2f(x[D] - nm);
    acc = fmaf(acc, f, x[d] * w);
    total = fmaf(total, f, x[D + 1] * w);
    m = nm;
  }
  if constexpr (GROUPS > 1) {
    acc_s[grp][d] = acc;
    if (d == 0) {
      max_s[grp] = m;
      sum_s[grp] = total;
    }
    __syncthreads();
    if (grp != 0) return;
    float nm = m;
#pragma unroll
    for (int i = 1; i < GROUPS; ++i) nm = fmaxf(nm, max_s[i]);
    const float f = __builtin_amdgcn_exp2f(m - nm);
    acc *= f;
    total *= f;
#pragma unroll
    for (int i = 1; i < GROUPS; ++i) {
      const float w = __builtin_amdgcn_exp2f(max_s[i] - nm);
      acc = fmaf(acc_s[i][d], w, acc);
      total = fmaf(sum_s[i], w, total);
    }
  }
  Elem<T>::store(p.out + ((size_t)b * p.H + h) * D + d, p.mean(acc, total));
}

}  // namespace lact
