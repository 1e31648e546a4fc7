// Softmax attention of one new token of every sequence with keys and values in pages (paged_cache.h), head sizes 64 and 128; queries bf16 or fp32, pages of the
// same type or e4m3:
//
//   o_h = sum_j softmax_j(f(q_h . k_j / sqrt(D)) - slope_h (n - 1 - j)) v_j,   max(0, n - window) <= j < n,   f(x) = cap tanh(x / cap) or x
//
// over the places j that lie on a page; n = lengths[b], read on the device.  A sequence that sees nothing has output 0.
//
// Work is split, and parts are joined, as in attention_step.h, unless a block has a key head of a sequence as a whole (PagedStepParams::whole).  A wave's step is 32
// places from a multiple of 16 on: two pieces of 16 rows, each of which lies in one page, as page sizes are multiples of 16.  The wave looks up where the
// keys and the values of 32 pieces lie at once, a lane each, and copies a piece from where its lane says; one without a page is copied from zeros and masked.  In a piece
// that the window or the length ends in, the rows outside repeat one inside.
//
// e4m3: numbers become bf16 exactly as they leave LDS.  A key's exponent is applied in that conversion (a lane has one key's row), a value's to the weight
// that meets it, both exactly.  fp32 queries and weights meet them in three bf16 parts of 8 bits.
#pragma once
#include "attention_step.h"
#include "paged_cache.h"

namespace lact {

template <typename T>
struct PagedStepParams {
  Pages kv;
  int B, N, H, HK, group, tiles, window;     // N: places of a sequence; tiles: of 32 query heads to a key head
  int blocks, whole;                         // of the main kernel; whether each has one item, whose steps are few
  const T* q; long long bsq;
  const int* lengths;
  const float* slopes;
  float scale, cap;
  T* out;
  float* part;
  __device__ __forceinline__ int length(int b) const { return min(max(lengths[b], 0), N); }
  __device__ __forceinline__ int first(int b) const { return max(0, length(b) - window); }
  __device__ __forceinline__ int span(int b) const { return length(b) - (first(b) & ~15); }
  __device__ __forceinline__ static float mean(float sum, float weights) { return weights == 0.f ? 0.f : sum / weights; }
};

static __device__ const uint4 paged_zeros[512] = {};      // a piece of any type

// 32 keys or values as they lie in LDS: the 16-byte granule g of row r at slot g ^ key(r)
template <typename C, int D>
struct PagedTile {
  static constexpr int ROWB = D * (int)sizeof(C), G = ROWB / 16, BYTES = 32 * ROWB, COPIES = BYTES / 1024;
  __device__ static __forceinline__ int key(int r) {
    if constexpr (is_e4m3<C>()) return D == 128 ? (r >> 1) & 7 : (r >> 2) & 3;
    else return MaskTile<C, D>::key(r);
  }
};
template <typename T, typename C, int D>
struct PagedShape {
  using S = PagedTile<C, D>;
  static constexpr int NW = sizeof(C) == 4 && D == 128 ? 2 : 4;             // waves, each with a ring of its own
  // To a compute unit.  8 bits take as much work for half the bytes: two waves of a SIMD.  (fp32 queries of 128 in three parts: no registers for that.)
  static constexpr int BLOCKS = is_e4m3<C>() && !(sizeof(T) == 4 && D == 128) ? 2 : 1;
  static constexpr int SIMD = sizeof(T) == 2 ? 2 : BLOCKS;                   // waves that registers are kept for: with those of two, sums stay where they are worked on
  static constexpr int STAGE = 2 * S::BYTES;
  static constexpr int RING = 131072 / (BLOCKS * NW * STAGE);
  static constexpr int EXP = is_e4m3<C>() ? 1024 : 0;                        // exponents of 32 pieces of keys and of values, twice
  static constexpr int WAVE = RING * STAGE + 2 * EXP;
  static constexpr int KEYS = 32 * NW;                                       // of a step
  static constexpr int LDS = NW * WAVE;
};

// bf16 parts of an fp32 operand, 24 bits in all; one of bf16
template <typename T, typename C> constexpr int paged_parts() { return sizeof(T) == 4 && is_e4m3<C>() ? 3 : 1; }

template <typename C, int D>
struct PagedFrag {      // the type of the queries, which the pages have as well
  using Frag = typename AttnType<C>::Frag;
  MaskFrag<C, D> fr;
  Frag q[1][D / 16];
  __device__ __forceinline__ void init() { fr.init(); }
  template <typename T>
  __device__ __forceinline__ void queries(const T* base, int h) {
    mask_own_rows<T, D>(q[0], base, D, h, h + 1);
  }
  __device__ __forceinline__ void arrived() { mask_arrived(q[0]); }
  __device__ __forceinline__ f32x16 scores(const char* tile, const char*) const {
    f32x16 s;
#pragma unroll
    for (int j = 0; j < 16; ++j) s[j] = 0.f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) s = mma32(fr.rows(tile, 0, ks), q[0][ks], s);
    return s;
  }
  __device__ __forceinline__ uint4 value_exponents(const char*) const { return uint4{}; }
  __device__ __forceinline__ void weigh(f32x16&, const uint4&) const {}
  __device__ __forceinline__ void add(f32x16 (&o)[D / 32], const f32x16& s, const char* tile) const {
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const Frag pf = mask_pack<C>(s, st);
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) o[dt] = mma32(fr.cols(tile, dt, st), pf, o[dt]);
    }
  }
};
// e4m3.  Of every 32 columns lane half h takes the 16 from 16 h on, eight for each of two products, in one read; the queries' fragments follow that.
template <typename T, int D>
struct PagedFrag8 {
  static constexpr int PARTS = paged_parts<T, uint8_t>();
  using S = PagedTile<uint8_t, D>;
  bf16x8 q[PARTS][D / 16];
  uint32_t row_base, row_key, tr_off[D / 32];
  __device__ __forceinline__ void init() {
    const int l = threadIdx.x & 63, h = l >> 5, r = (l & 15) >> 1, row = 8 * (r >> 2) + 4 * h + (r & 3);
    row_base = (l & 31) * S::ROWB;
    row_key = (uint32_t)(S::key(l & 31) ^ h) << 4;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) tr_off[dt] = row * S::ROWB + (((dt * 2 + ((l >> 4) & 1)) ^ S::key(row)) << 4) + (l & 1) * 8;
  }
  __device__ __forceinline__ void queries(const T* base, int head) {
    const T* p = base + (size_t)head * D + 16 * ((threadIdx.x & 63) >> 5);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const T* at = p + (ks >> 1) * 32 + (ks & 1) * 8;
      if constexpr (PARTS == 1) {
        q[0][ks] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(at));
      } else {
        float x[8];
        Elem<T>::load4(at, x);
        Elem<T>::load4(at + 4, x + 4);
#pragma unroll
        for (int i = 0; i < PARTS; ++i) q[i][ks] = next_part(x);
      }
    }
  }
  __device__ __forceinline__ void arrived() {
#pragma unroll
    for (int i = 0; i < PARTS; ++i) mask_arrived(q[i]);
  }
  // the leading bf16 part of eight numbers, which keep the rest
  __device__ __forceinline__ static bf16x8 next_part(float (&x)[8]) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
      x[2 * i] -= bf16_lo(r[i]);
      x[2 * i + 1] -= bf16_hi(r[i]);
    }
    return __builtin_bit_cast(bf16x8, make_uint4(r[0], r[1], r[2], r[3]));
  }
  __device__ __forceinline__ static bf16x8 widen(uint32_t a, uint32_t b, float scale) {
    return __builtin_bit_cast(bf16x8, make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, false)),
                                                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, true)),
                                                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, false)),
                                                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, true))));
  }
  __device__ __forceinline__ f32x16 scores(const char* tile, const char* exps) const {
    f32x16 s;
#pragma unroll
    for (int j = 0; j < 16; ++j) s[j] = 0.f;
    const float scale = __uint_as_float((uint32_t)*reinterpret_cast<const uint8_t*>(exps + (threadIdx.x & 31)) << 23);      // (the conversion takes its exponent bits alone)
#pragma unroll
    for (int m = 0; m < D / 32; ++m) {
      const uint4 u = *reinterpret_cast<const uint4*>(tile + row_base + ((uint32_t)(m * 32) ^ row_key));
      const bf16x8 a = widen(u.x, u.y, scale), b = widen(u.z, u.w, scale);
#pragma unroll
      for (int i = PARTS - 1; i >= 0; --i) {      // the smaller ones first
        s = mma32(a, q[i][2 * m], s);
        s = mma32(b, q[i][2 * m + 1], s);
      }
    }
    return s;
  }
  // of the lane's 16 values, in the order of its weights
  __device__ __forceinline__ uint4 value_exponents(const char* exps) const {
    const uint32_t* e = reinterpret_cast<const uint32_t*>(exps + 512 + 4 * ((threadIdx.x & 63) >> 5));
    return make_uint4(e[0], e[2], e[4], e[6]);
  }
  __device__ __forceinline__ void weigh(f32x16& s, const uint4& exps) const {
    const uint32_t e[4] = {exps.x, exps.y, exps.z, exps.w};
#pragma unroll
    for (int j = 0; j < 16; ++j) {      // an exponent of 255 is infinity here
      const uint32_t w = e[j / 4], f = (j % 4 == 3 ? w >> 1 : w << (23 - 8 * (j % 4))) & 0x7f800000u;
      s[j] *= __uint_as_float(max(f, 0x400000u));
    }
  }
  __device__ __forceinline__ void add(f32x16 (&o)[D / 32], const f32x16& s, const char* tile) const {
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = s[8 * st + j];
      bf16x8 pf[PARTS];
#pragma unroll
      for (int i = 0; i < PARTS; ++i) pf[i] = next_part(x);
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) {
        const i32x2 c = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(tile + tr_off[dt] + st * 16 * S::ROWB));
        const bf16x8 v = widen((uint32_t)c[0], (uint32_t)c[1], 1.f);
#pragma unroll
        for (int i = PARTS - 1; i >= 0; --i) o[dt] = mma32(v, pf[i], o[dt]);
      }
    }
  }
};
template <typename T, typename C, int D>
using PagedMath = typename std::conditional<is_e4m3<C>(), PagedFrag8<T, D>, PagedFrag<T, D>>::type;

// 16 bytes per lane to LDS from where each lane says: lane i lands at lds_base + 16 * i
__device__ __forceinline__ void dma16_from(uint64_t at, uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\t" ::"s"(lds_base), "v"(at) : "memory", "m0");
}

template <typename T, typename C, int D, int BENT>
__global__ __launch_bounds__((64 * PagedShape<T, C, D>::NW), (PagedShape<T, C, D>::SIMD)) void k_paged_step(const PagedStepParams<T> p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  using A = PagedShape<T, C, D>;
  using S = PagedTile<C, D>;
  constexpr int NW = A::NW, RING = A::RING, NC = S::COPIES, HALF = NC / 2, BATCH = 16;      // copies of a wave for 32 keys; tiles that it looks up at once
  static_assert(RING <= BATCH, "one batch holds what is on its way");
  prefetch_args<sizeof(p)>();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, items = p.HK * p.tiles;
  // the block's steps: from step0 of this item of sequence b on
  int b, item, step0;
  long long left;
  if (p.whole) {
    b = blockIdx.x / items;
    item = blockIdx.x - b * items;
    step0 = 0;
    left = same(StepWork::steps<A::KEYS>(p, b));
    if (left == 0) {
      const int h0 = item / p.tiles * p.group + item % p.tiles * 32, rows = min(32, (item / p.tiles + 1) * p.group - h0);
      for (int i = threadIdx.x; i < rows * D; i += 64 * NW) Elem<T>::store(p.out + ((size_t)b * p.H + h0) * D + i, 0.f);
      return;
    }
  } else {
    StepWork work;
    work.init<A::KEYS>(p);
    if ((int)blockIdx.x >= work.blocks) return;
    const long long s0 = work.share(blockIdx.x);
    long long begin;
    left = work.share(blockIdx.x + 1) - s0;
    b = work.find<A::KEYS>(p, s0, begin);
    if (b >= p.B) return;
    const int n = same(StepWork::steps<A::KEYS>(p, b));
    item = (int)((s0 - begin) / n);
    step0 = (int)(s0 - begin - (long long)item * n);
  }
  const uint32_t ring = lds_addr(smem) + wave * A::WAVE;
  const char* mine = smem + wave * A::WAVE;
  PagedMath<T, C, D> math;
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
    const int n = same(StepWork::steps<A::KEYS>(p, b));
    if (n == 0) {
      if (++b >= p.B) return;                                   // (the shares end with the last sequence)
      continue;
    }
    const int step1 = (int)min((long long)n, step0 + left);
    const int hk = item / p.tiles, h0 = hk * p.group + (item - hk * p.tiles) * 32;
    const int rows = min(32, (hk + 1) * p.group - h0), h = h0 + min(lane & 31, rows - 1);
    const int len = same(p.length(b)), lo = same(p.first(b)), lo16 = lo & ~15;
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
#pragma unroll
        for (int i = x * HALF; i < (x + 1) * HALF; ++i) dma16<false>(from, (uint32_t)min(max(crow[i], first), last) * S::ROWB + ccol[i], to + i * 1024);
      }
    };
    auto keys = [&](int t) LACT_INLINE_LAMBDA { copy(t, 0, ring + t % RING * A::STAGE); };
    auto values = [&](int t) LACT_INLINE_LAMBDA { copy(t, 32, ring + t % RING * A::STAGE + S::BYTES); };
    math.queries(p.q + b * p.bsq, h);
    Scores<T, BENT> sc;
    sc.init(p.scale, p.cap, p.slopes, h);
    const float c = sc.unit();
    // no barrier: nobody else uses the wave's ring
    if (tiles > 0) look_up(0);
#pragma unroll
    for (int t = 0; t < RING; ++t)
      if (t < tiles) {
        keys(t);
        values(t);
      }
    math.arrived();
    f32x16 o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) o[i][j] = 0.f;
    float mc = ATTN_LOWEST, sum = 0.f;
    for (int t = 0; t < tiles; ++t) {
      const bool more = t + RING < tiles, full = t + RING <= tiles;
      if (full) wait_vmcnt<(2 * RING - 1) * NC>();
      else wait_vmcnt<0>();
      const char* kt = mine + t % RING * A::STAGE;
      const char* vt = kt + S::BYTES;
      const char* et = mine + RING * A::STAGE + (t / BATCH & 1) * A::EXP + t % BATCH * 32;
      const int k0 = place(t), at = k0 + 4 * (lane >> 5);
      const int on_pages = (t / BATCH == batch ? there : there_before) >> (2 * (t % BATCH)) & 3;      // of the two pieces
      const bool masked = k0 < lo || k0 + 32 > len || on_pages != 3;
      f32x16 s = math.scores(kt, et);
      const auto exps = math.value_exponents(et);
      wave_reads_done();
      if (more) {
        if ((t + RING) % BATCH == 0) {
          look_up(t + RING);
          ++batch;
        }
        keys(t + RING);
      }
      sc.apply(s, at - (len - 1));
      auto mask = [&](float nothing) LACT_INLINE_LAMBDA {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int key = at + 8 * (j / 4) + j % 4;
          s[j] = key >= lo && key < len && (on_pages >> (j / 8) & 1) ? s[j] : nothing;
        }
      };
      if (masked) mask(-__builtin_inff());
      float mx = max3(s[0], s[1], s[15]);
#pragma unroll
      for (int j = 1; j < 8; ++j) mx = max3(mx, s[2 * j], s[2 * j + 1]);
      mx *= c;
      if (__any(mx > mc + 8.f)) {
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float nm = mx > mc + 8.f ? mx : mc, f = __builtin_amdgcn_exp2f(mc - nm);
        mc = nm;
        sum *= f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j) o[i][j] *= f;
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        s[j] = __builtin_amdgcn_exp2f(fmaf(s[j], c, -mc));
        sum += s[j];
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
    const int stride = min(p.group, 32);
    attn_step_leave<T, D, NW, A::WAVE>(p, smem, o, mc, sum, rows, whole ? p.out + ((size_t)b * p.H + h0) * D : nullptr,
                                       p.part + (size_t)(2 * blockIdx.x + (head_of_share ? 0 : 1)) * stride * (D + 2));
    __syncthreads();      // the rings are free again
    head_of_share = false;
    left -= step1 - step0;
    step0 = 0;
    if (++item == items) {
      item = 0;
      if (++b >= p.B) return;
    }
  }
}

}  // namespace lact
