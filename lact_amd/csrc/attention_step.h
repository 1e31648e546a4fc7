// Softmax attention of one new token of every sequence with that sequence's cache of keys and values, bf16 and fp32, head sizes 64 and 128:
//
//   o_h = sum_j softmax_j(f(q_h . k_j / sqrt(D)) - slope_h (n - 1 - j)) v_j,   max(0, n - window) <= j < n,   f(x) = cap tanh(x / cap) or x
//
// q, out: [B, H, D]; k, v: [B, N, HK, D] with any token, head and batch strides; n = lengths[b], read on the device.  n = 0: output 0.
//
// The keys are read once for all query heads that share a key head: those are the columns (32, the rest unused) of 32x32 products over 32 keys.  What
// bounds it is that one read; the products take a fifth of its time.  131072 keys and values, 8 heads of 128 with 4 queries each: 103 us, 5.2 TB/s (a
// large copy reaches 4.9); 32 sequences of up to 8192: 117 us, 4.3 TB/s.
//
// Sequences differ in length, and the host does not know them.  The work of all (sequence, key head) items, in steps of 32 keys a wave, is cut
// into equal shares for one block per compute unit: a share may end inside an item and begin inside another.  What a block has of an item
// that it does not have as a whole, at most its first and its last, goes to the workspace unnormalised, and k_attn_step_join adds the parts
// in the blocks' order.
#pragma once
#include "masked_attention.h"

namespace lact {

template <typename T>
struct AttnStepParams {
  int B, N, H, HK, group, tiles, window;     // tiles: of 32 query heads to a key head
  int blocks;                                // of the main kernel
  const T* q; long long bsq;                 // heads follow each other
  const T* k; const T* v;
  long long ldk, bsk, hsk, ldv, bsv, hsv;    // elements between tokens, batch entries, heads
  const int* lengths;                        // [B]
  const float* slopes;                       // [H] or null
  float scale, cap;
  T* out;                                    // [B, H, D]
  float* part;                               // [2 * blocks][rows][D + 2]: sums, then row maximum and row sum; rows = min(group, 32)
  __device__ __forceinline__ int length(int b) const { return min(max(lengths[b], 0), N); }
};

// What the wave has read of LDS is in registers: the next copies may overwrite it.
__device__ __forceinline__ void wave_reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// What is the same for the whole wave, in scalar registers.
__device__ __forceinline__ int same(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ long long same(long long v) {
  return (long long)((uint64_t)(uint32_t)same((int)v) | (uint64_t)(uint32_t)same((int)(v >> 32)) << 32);
}

template <typename T, int D>
struct AttnStepShape {
  static constexpr int NW = sizeof(T) == 4 && D == 128 ? 2 : 4;             // waves, each with a ring of its own
  static constexpr int TILE = 32 * D * (int)sizeof(T);                      // 32 keys
  static constexpr int RING = 131072 / (NW * 2 * TILE);                     // 2, bf16 of 64: 4
  static constexpr int KEYS = 32 * NW;                                      // of a step
  static constexpr int LDS = NW * RING * 2 * TILE;
};

// Where the steps of the sequences lie in the row of all of them.  Every wave computes it for itself, 64 sequences at a time.
struct StepWork {
  long long total;
  int blocks;        // with a share: none is empty
  template <int KEYS, typename P>
  __device__ __forceinline__ static int steps(const P& p, int b) {
    return b < p.B ? (min(p.length(b), p.window) + KEYS - 1) / KEYS : 0;
  }
  __device__ __forceinline__ static long long scan(long long v) {           // inclusive, over the wave
    const int l = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const long long u = __shfl_up(v, o, 64);
      if (l >= o) v += u;
    }
    return v;
  }
  template <int KEYS, typename P>
  __device__ __forceinline__ void init(const P& p) {
    total = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) total += __shfl(scan(steps<KEYS>(p, b0 + (threadIdx.x & 63))), 63, 64);
    total = same(total * (p.HK * p.tiles));
    blocks = (int)min((long long)p.blocks, total);
  }
  // the sequence that step s < total belongs to, and the step that it begins with
  template <int KEYS, typename P>
  __device__ __forceinline__ int find(const P& p, long long s, long long& begin) const {
    const int per = p.HK * p.tiles;
    long long before = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
      const int n = steps<KEYS>(p, b0 + (threadIdx.x & 63));
      const long long end = (before + scan(n)) * per;
      const uint64_t past = __ballot(s < end);
      if (past) {
        const int i = __ffsll((unsigned long long)past) - 1;
        begin = same(__shfl(end - (long long)n * per, i, 64));
        return same(b0 + i);
      }
      before = __shfl(end, 63, 64) / per;
    }
    begin = 0;
    return p.B;
  }
  // the steps in front of sequence b
  template <int KEYS, typename P>
  __device__ __forceinline__ long long begin(const P& p, int b) const {
    long long before = 0;
    for (int b0 = 0; b0 < b; b0 += 64) {
      const int i = b0 + (threadIdx.x & 63);
      before += __shfl(scan(i < b ? steps<KEYS>(p, i) : 0), 63, 64);
    }
    return before * p.HK * p.tiles;
  }
  __device__ __forceinline__ long long share(int block) const { return block * total / blocks; }
  __device__ __forceinline__ int block_of(long long s) const { return (int)(((s + 1) * blocks - 1) / total); }
};

template <typename T, int D, int BENT>
__global__ __launch_bounds__((64 * AttnStepShape<T, D>::NW), 1) void k_attn_step(const AttnStepParams<T> p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  using A = AttnStepShape<T, D>;
  using S = MaskTile<T, D>;
  using Frag = typename AttnType<T>::Frag;
  constexpr int NW = A::NW, RING = A::RING, NC = A::TILE / 1024;      // copies of a wave for 32 keys
  prefetch_args<sizeof(p)>();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  StepWork work;
  work.init<A::KEYS>(p);
  if ((int)blockIdx.x >= work.blocks) return;
  long long s0 = work.share(blockIdx.x);
  const long long s1 = work.share(blockIdx.x + 1);
  long long begin;
  int b = work.find<A::KEYS>(p, s0, begin);
  const uint32_t ring = lds_addr(smem) + wave * RING * 2 * A::TILE;
  char* mine = smem + wave * RING * 2 * A::TILE;
  MaskFrag<T, D> fr;
  fr.init();
  int crow[NC];
  uint32_t ccol[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = i * 64 + lane;
    crow[i] = c / S::G;
    ccol[i] = (uint32_t)((c % S::G) ^ S::key(crow[i])) * 16;
  }
  bool head_of_share = true;
  while (s0 < s1) {
    int n = 0;
    while (b < p.B && (n = same(StepWork::steps<A::KEYS>(p, b))) == 0) ++b;
    if (b >= p.B) return;                                       // (the shares end with the last sequence)
    const long long in_b = s0 - begin;
    const int item = (int)(in_b / n), step0 = (int)(in_b - (long long)item * n);
    const int step1 = (int)min((long long)n, step0 + (s1 - s0));
    const int hk = item / p.tiles, h0 = hk * p.group + (item - hk * p.tiles) * 32;
    const int rows = min(32, (hk + 1) * p.group - h0), h = h0 + min(lane & 31, rows - 1);
    const int len = same(p.length(b)), lo = max(0, len - p.window);
    const T* K = p.k + b * p.bsk + hk * p.hsk;
    const T* V = p.v + b * p.bsv + hk * p.hsv;
    Frag qf[D / 16];
    mask_own_rows<T, D>(qf, p.q + b * p.bsq, D, h, p.H);
    Scores<T, BENT> sc;
    sc.init(p.scale, p.cap, p.slopes, h);
    const float c = sc.unit();
    f32x16 o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) o[i][j] = 0.f;
    float mc = ATTN_LOWEST, sum = 0.f;
    mask_arrived(qf);
    // the wave's tiles: 32 keys from lo + (step * NW + wave) * 32 on
    const int tiles = min(step1 - step0, max(0, (len - lo - wave * 32 - step0 * A::KEYS + A::KEYS - 1) / A::KEYS));
    auto copy = [&](const T* base, long long ld, int t, uint32_t to) LACT_INLINE_LAMBDA {
      const int k0 = lo + ((step0 + t) * NW + wave) * 32;
      const T* from = uniform(base + (long long)k0 * ld);
#pragma unroll
      for (int i = 0; i < NC; ++i) dma16<false>(from, (uint32_t)min(crow[i], len - 1 - k0) * (uint32_t)ld * (uint32_t)sizeof(T) + ccol[i], to + i * 1024);
    };
    auto keys = [&](int t) LACT_INLINE_LAMBDA { copy(K, p.ldk, t, ring + t % RING * 2 * A::TILE); };
    auto values = [&](int t) LACT_INLINE_LAMBDA { copy(V, p.ldv, t, ring + t % RING * 2 * A::TILE + A::TILE); };
    // no barrier: nobody else uses the wave's ring
#pragma unroll
    for (int t = 0; t < RING; ++t)
      if (t < tiles) {
        keys(t);
        values(t);
      }
    for (int t = 0; t < tiles; ++t) {
      const bool more = t + RING < tiles, full = t + RING <= tiles;
      if (full) wait_vmcnt<(2 * RING - 1) * NC>();
      else wait_vmcnt<0>();
      const char* kt = mine + t % RING * 2 * A::TILE;
      const char* vt = kt + A::TILE;
      const int k0 = lo + ((step0 + t) * NW + wave) * 32, at = k0 + 4 * (lane >> 5);
      f32x16 s;
#pragma unroll
      for (int j = 0; j < 16; ++j) s[j] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) s = mma32(fr.rows(kt, 0, ks), qf[ks], s);
      wave_reads_done();
      if (more) keys(t + RING);
      sc.apply(s, at - (len - 1));
      if (k0 + 32 > len) {
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = Seen(0, len - at).or_nothing(s[j], j);
      }
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
      if (more) wait_vmcnt<(2 * RING - 1) * NC>();
      else wait_vmcnt<0>();
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const Frag pf = mask_pack<T>(s, st);
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) o[dt] = mma32(fr.cols(vt, dt, st), pf, o[dt]);
      }
      wave_reads_done();
      if (more) values(t + RING);
    }
    // The waves' parts together: sums at their place in each one's ring, [row][D + 4], maximum and row sum behind them.
    constexpr int LD = D + 4;
    sum += __shfl_xor(sum, 32, 64);
    float* w = reinterpret_cast<float*>(mine);
    if ((lane & 31) < rows) {
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          Elem<float>::store4(w + (lane & 31) * LD + dt * 32 + 8 * g + 4 * (lane >> 5), o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]);
      if (lane < 32) {
        w[lane * LD + D] = mc;
        w[lane * LD + D + 1] = sum;
      }
    }
    __syncthreads();
    const bool whole = step0 == 0 && step1 == n;
    const int stride = min(p.group, 32);
    float* part = p.part + (size_t)(2 * blockIdx.x + (head_of_share ? 0 : 1)) * stride * (D + 2);
    constexpr int WSTRIDE = RING * 2 * A::TILE / 4;
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
        Elem<T>::store(p.out + ((size_t)b * p.H + h0 + r) * D + d, acc / total);
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
    s0 += step1 - step0;
    if (step1 == n && item + 1 == p.HK * p.tiles) {
      begin += (long long)n * p.HK * p.tiles;
      ++b;
    }
  }
}

// (7 us for 256 parts of one sequence, bound by the launch and the way to them: 512 threads, so that each reads few.)
// One block of 512 threads per (sequence, query head): the sum of the parts that blocks left of it, and zeros for a sequence without tokens.
template <typename T, int D>
__global__ __launch_bounds__(512) void k_attn_step_join(const AttnStepParams<T> p) {
  constexpr int GROUPS = 512 / D;
  __shared__ float acc_s[GROUPS][D], sum_s[GROUPS], max_s[8];
  const int b = blockIdx.x / p.H, h = blockIdx.x - b * p.H;
  constexpr int KEYS = AttnStepShape<T, D>::KEYS;
  const int n = StepWork::steps<KEYS>(p, b);
  T* out = p.out + ((size_t)b * p.H + h) * D;
  if (n == 0) {
    if (threadIdx.x < D) Elem<T>::store(out + threadIdx.x, 0.f);
    return;
  }
  StepWork work;
  work.init<KEYS>(p);
  const int hk = h / p.group, g = h - hk * p.group;
  const long long first = work.begin<KEYS>(p, b) + (long long)(hk * p.tiles + g / 32) * n;
  const int f = work.block_of(first), e = work.block_of(first + n - 1);
  if (f == e) return;
  const int stride = min(p.group, 32);
  auto part = [&](int i) { return p.part + ((size_t)(2 * i + (work.share(i) >= first ? 0 : 1)) * stride + (g & 31)) * (D + 2); };
  float m = -INFINITY;
  for (int i = f + (int)threadIdx.x; i <= e; i += 512) m = fmaxf(m, part(i)[D]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  if ((threadIdx.x & 63) == 0) max_s[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, max_s[i]);
  const int grp = threadIdx.x / D, d = threadIdx.x % D;
  float acc = 0.f, total = 0.f;
#pragma unroll 4
  for (int i = f + grp; i <= e; i += GROUPS) {
    const float* x = part(i);
    const float w = __builtin_amdgcn_exp2f(x[D] - m);
    acc += x[d] * w;
    total += x[D + 1] * w;
  }
  acc_s[grp][d] = acc;
  if (d == 0) sum_s[grp] = total;
  __syncthreads();
  if (grp == 0) {
#pragma unroll
    for (int i = 1; i < GROUPS; ++i) {
      acc += acc_s[i][d];
      total += sum_s[i];
    }
    Elem<T>::store(out + d, acc / total);
  }
}

}  // namespace lact
