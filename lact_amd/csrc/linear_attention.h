// Linear attention with a decay, bf16 and fp32, key and value sizes 64 and 128:
//
//   S_t = e^(g_t) S_(t-1) + k_t v_t^T,   o_t = scale S_t^T q_t
//
// q, k: [B, L, H, DK], v: [B, L, H, DV] with token and batch strides, heads next to each other; g: log decays, fp32, [B, L, H] or one per
// head; S: [B, H, DK, DV] fp32.
//
// In chunks of 64 tokens, with G the sum of g from the chunk's start to a token, itself included:
//
//   o_i = scale (sum_(j <= i) e^(G_i - G_j) (q_i . k_j) v_j + e^(G_i) S^T q_i),   S <- e^(G_last) S + sum_j e^(G_last - G_j) k_j v_j^T
//
// Only differences of later and earlier sums are exponentiated, so no decay overflows; the sums are formed in fp64 and kept in two floats.
// The gradients are the same recurrence with other operands: of q with (dout, v, k) and the transposed state; of k with (v, dout, q) and of v with (k, q, dout)
// backwards in time from the gradient of the last state.  One function, lin_walk, is all four.
//
// A block walks the chunks of a segment of one head (lin_walk); a wave owns a quarter of the state's columns, in accumulators, from where they are
// packed as the next product's operand where they lie (an accumulator's rows are k slots there; which row of the state an accumulator row
// holds is chosen so that the queries' operand is 8 neighbours).  Segments start from states that k_lin_segments and k_lin_scan form first, where heads
// and batch alone do not fill the chip.
//
// 4 x 4096 tokens, 12 heads of 128 x 128, decays per token, us: weights 5, segments 30 and scan 11 (the two of them also for the gradients, backwards), outputs
// 57, gradients 217, decays' gradient 17.  The segments, the scan and the decays are bound by memory: 100 MB at 3.4 TB/s, 62 MB at 5.8 (out of the cache),
// 63 MB at 3.7.  The walks are bound by the way from one dependent product to the next: a chunk's pairs, the state's share, the update and the outputs follow each
// other, two waves of a SIMD cover what they can (gradients: the matrix units are busy for 17 % of the time, the vector units for 27 %, and waves wait for 38 % of theirs).  Eight
// waves to a block with half of the columns each (255 us for the gradients) read the shared operands from LDS twice as often, and have too few registers.  In fp32 the
// gradients of 128 x 128 keep 66 registers in memory with the decays' gradient, 13 without.
//
// The state is held, and added to, in fp32: what is added is a product of bf16 inputs with a weight, which goes into the matrix product
// as three bf16 parts (24 bits).  Where only rounded results depend on the state (dk, and dq without the decays' gradient) it is added to in one part, and as an operand it
// is one part there and in the outputs; pairs are rounded to bf16 as well.
//
// A gradient of the decays adds what crosses a token (k_lin_decay_grad): pairs M_ij = e^(G_i - G_j) (q_i . k_j)(dout_i . v_j) scale of a source in front and an
// output behind it, and the states' shares.
#pragma once
#include <type_traits>

#include "masked_attention.h"

namespace lact {

constexpr int LIN_CHUNK = 64;
constexpr int LIN_STRETCH = 8;             // chunks over which the decays' gradient carries a sum, see k_lin_decay_grad
constexpr float LIN_MIN_LOG = -200.f;      // e^-200 is 0 in fp32: a log decay of -infinity forgets everything, and its sums stay finite

struct LinDecay {
  const float* g;         // [B, L, H] or [H]
  int per_token;
  __device__ __forceinline__ float at(int b, int t, int h, int L, int H) const {
    if (t >= L) return 0.f;
    const float x = per_token ? g[((size_t)b * L + t) * H + h] : g[h];
    return x < LIN_MIN_LOG ? LIN_MIN_LOG : x;
  }
};

template <typename T>
struct LinRows {          // [B, L, H, D]
  const T* p;
  int ld;
  long long bs;
};

template <typename T>
struct LinParams {
  int B, L, H, segments, seg_chunks;     // chunks of a segment
  LinRows<T> x, y, z, w;                 // out_i = sum_j (x_i . y_j) z_j + x_i S, S += y_j z_j^T; w: see lin_walk
  const float* weights;                  // [B * H][chunks][4][64], see k_lin_weights
  float pair_scale, state_scale, source_scale;
  T* out;                                // [B, L, H, DZ]
  const float* states;                   // [segments][B * H][DX * DZ] (or transposed): where each segment starts, null: from zero
  const float* state0;                   // [B * H][..]: the same for a single segment
  int transposed;                        // the states in memory are [DZ][DX]
  float* last;                           // [B * H][..]: state behind the walk's last chunk, nullable
  float* dots;                           // [B * H][L] fp32, forwards two of them, for the gradient of the decays
  float* between;                        // [segments][stretches - 1][B * H][DX * DZ] (or transposed): states between a segment's stretches, null: it has one
  int stretches;                         // of LIN_STRETCH chunks in a segment
  UDiv by_heads;                         // H
};

// ---- operands of 16x16 products with 32 k slots: lane l holds row (or column) l & 15, slots 8 * (l >> 4) + j
__device__ __forceinline__ f32x4 mma16(const bf16x8& a, const bf16x8& b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma16(const f32x8& a, const f32x8& b, f32x4 c) {
#pragma unroll
  for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
  return c;
}
__device__ __forceinline__ void lin_zero(f32x4& v) { v = f32x4{0.f, 0.f, 0.f, 0.f}; }

__device__ __forceinline__ bf16x8 lin_pack(const float (&v)[8], uint16_t) {
  return __builtin_bit_cast(bf16x8, make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])));
}
__device__ __forceinline__ f32x8 lin_pack(const float (&v)[8], float) { return f32x8{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]}; }
// Sum over 16 neighbouring lanes, without a way through LDS
__device__ __forceinline__ float sum16(float v) {
  auto turned = [](float x, auto by) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x120 + decltype(by)::value, 0xf, 0xf, false));      // row_ror
  };
  v += turned(v, std::integral_constant<int, 8>());
  v += turned(v, std::integral_constant<int, 4>());
  v += turned(v, std::integral_constant<int, 2>());
  v += turned(v, std::integral_constant<int, 1>());
  return v;
}
// Eight floats as PARTS operands whose sum they are, largest first; fp32 needs one.
template <typename T, int PARTS>
__device__ __forceinline__ void lin_split(float (&v)[8], typename AttnType<T>::Frag (&f)[PARTS]) {
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    f[p] = lin_pack(v, T());
    if (p + 1 < PARTS)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] -= (float)f[p][i];
  }
}
template <typename T> constexpr int lin_parts() { return sizeof(T) == 2 ? 3 : 1; }

// Reads of a 64 x D tile laid out as MaskTile.
template <typename T, int D> struct LinFrag {
  using S = MaskTile<T, D>;
  using Frag = typename AttnType<T>::Frag;
  // rows [16 * rt, +16), columns 32 * u + 8 * (l >> 4) + j
  __device__ static __forceinline__ Frag rows(const char* tile, int rt, int u) {
    const int l = threadIdx.x & 63, r = rt * 16 + (l & 15), c = l >> 4;
    const char* p = tile + r * S::ROWB;
    if constexpr (sizeof(T) == 2) {
      return __builtin_bit_cast(Frag, *reinterpret_cast<const uint4*>(p + (((4 * u + c) ^ S::key(r)) << 4)));
    } else {
      const float4 a = *reinterpret_cast<const float4*>(p + (((8 * u + 2 * c) ^ S::key(r)) << 4));
      const float4 b = *reinterpret_cast<const float4*>(p + (((8 * u + 2 * c + 1) ^ S::key(r)) << 4));
      return Frag{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    }
  }
  // Transposed: lane l holds column `col(l & 15)`, slot j tile row 32 * v + 8 * (l >> 4) + j.  col(i) = c0 + cs * (i >> 2) + (i & 3).
  template <int CS>
  __device__ static __forceinline__ Frag cols(const char* tile, int c0, int v) {
    const int l = threadIdx.x & 63, c = l >> 4;
    if constexpr (sizeof(T) == 2) {
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      typedef short s16x8 __attribute__((ext_vector_type(8)));
      // inside 16 lanes, lane i receives element i & 3 of the 8 bytes that lanes 4 j + (i >> 2) address, j = 0 .. 3
      const int r = 32 * v + 8 * c + ((l >> 2) & 3), col = c0 + CS * (l & 3);
      const uint32_t in = (col & 7) * 2;
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + r * S::ROWB + (((col >> 3) ^ S::key(r)) << 4) + in));
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + (r + 4) * S::ROWB + (((col >> 3) ^ S::key(r + 4)) << 4) + in));
      const s16x8 x = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
      return __builtin_bit_cast(Frag, x);
    } else {
      const int col = c0 + CS * ((l & 15) >> 2) + (l & 3);
      Frag x;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int r = 32 * v + 8 * c + j;
        x[j] = *reinterpret_cast<const float*>(tile + r * S::ROWB + (((col >> 2) ^ S::key(r)) << 4) + (col & 3) * 4);
      }
      return x;
    }
  }
  __device__ static __forceinline__ const char* at(const char* tile, int r, int col) {
    constexpr int E = 16 / (int)sizeof(T);
    return tile + r * S::ROWB + (((col / E) ^ S::key(r)) << 4) + (col % E) * (int)sizeof(T);
  }
};

// What the tokens of a chunk weigh, for every walk over it, 64 of each: the sum of log2 decays from the chunk's start in two floats, 2 to it (the weight of the
// state in front in the token's output, forwards) and 2 to the rest of the chunk (the weight of the token in the state behind); both weights 0 past the
// sequence's end.  One wave per chunk and head.
enum { LIN_HI = 0, LIN_LO = 64, LIN_FRONT = 128, LIN_BEHIND = 192 };
__global__ __launch_bounds__(256) void k_lin_weights(int B, int L, int H, LinDecay decay, float* weights) {
  const int chunks = (L + 63) / 64, lane = threadIdx.x & 63;
  const long long id = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (id >= (long long)B * H * chunks) return;
  const int bh = (int)(id / chunks), t = (int)(id - (long long)bh * chunks) * 64 + lane, b = bh / H, h = bh - b * H;
  double s = (double)decay.at(b, t, h, L, H) * 1.4426950408889634;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double u = __shfl_up(s, o, 64);
    if (lane >= o) s += u;
  }
  const double end = __shfl(s, 63, 64);
  const float hi = (float)s, lo = (float)(s - (double)hi);
  float* to = weights + id * 256 + lane;
  to[LIN_HI] = hi;
  to[LIN_LO] = lo;
  to[LIN_FRONT] = t < L ? __builtin_amdgcn_exp2f(hi) : 0.f;
  to[LIN_BEHIND] = t < L ? __builtin_amdgcn_exp2f((float)(end - s)) : 0.f;
}

// 2^(later - earlier) of the sums of two tokens
__device__ __forceinline__ float lin_between(float later_hi, float later_lo, float earlier_hi, float earlier_lo) {
  return __builtin_amdgcn_exp2f((later_hi - earlier_hi) + (later_lo - earlier_lo));
}

template <typename T, int DX, int DZ, bool GATE>
struct LinShape {
  static constexpr int X = MaskTile<T, DX>::BYTES, Z = MaskTile<T, DZ>::BYTES;
  static constexpr int STAGE = 2 * X + (GATE ? 2 : 1) * Z + 1024;         // x, y, z (, w), weights
  static constexpr int PAIRS = MaskTile<T, 64>::BYTES;
  static constexpr int SUMS = GATE ? 4 * 64 * 4 * 2 : 0;                  // per wave: what its columns, and its pairs, add to the dots
  // two chunks where two blocks of them fit a compute unit
  static constexpr int BUFFERS = 2 * STAGE + PAIRS + SUMS + 16 <= 80 * 1024 ? 2 : 1;
  static constexpr int LDS = BUFFERS * STAGE + PAIRS + SUMS + 16;
  static_assert(LDS <= 160 * 1024, "LDS");
};

template <typename T, int DX, int DZ>
struct LinState {        // columns [wave * DZ / 4, + DZ / 4): accumulator a, row 4 c + r holds state row 32 (a / 2) + 8 c + 4 (a % 2) + r
  static constexpr int NT = DZ / 64, AT = DX / 16;
  f32x4 s[AT][NT];
  __device__ static __forceinline__ int row(int a, int l) { return 32 * (a >> 1) + 8 * ((l & 63) >> 4) + 4 * (a & 1); }
  __device__ static __forceinline__ int col(int wave, int nt, int l) { return wave * (DZ / 4) + nt * 16 + (l & 15); }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int a = 0; a < AT; ++a)
#pragma unroll
      for (int n = 0; n < NT; ++n) lin_zero(s[a][n]);
  }
  __device__ __forceinline__ void load(const float* m, bool transposed, int wave) {
    const int l = threadIdx.x;
#pragma unroll
    for (int a = 0; a < AT; ++a)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (transposed) {
          const float4 v = *reinterpret_cast<const float4*>(m + (size_t)col(wave, n, l) * DX + row(a, l));
          s[a][n] = f32x4{v.x, v.y, v.z, v.w};
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) s[a][n][r] = m[(size_t)(row(a, l) + r) * DZ + col(wave, n, l)];
        }
      }
  }
  __device__ __forceinline__ void store(float* m, bool transposed, int wave) const {
    int l = threadIdx.x;
    asm volatile("" : "+v"(l));      // (places are computed here, not held in registers through the walk)
#pragma unroll
    for (int a = 0; a < AT; ++a)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (transposed) {
          *reinterpret_cast<float4*>(m + (size_t)col(wave, n, l) * DX + row(a, l)) = make_float4(s[a][n][0], s[a][n][1], s[a][n][2], s[a][n][3]);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) m[(size_t)(row(a, l) + r) * DZ + col(wave, n, l)] = s[a][n][r];
        }
      }
  }
  // decays by `whole` and adds y^T (weight z); zf: the wave's columns of z
  template <bool REV, int PARTS, typename Frag>
  __device__ __forceinline__ void update(const char* y, const Frag (&zf)[2][NT], const float* w, float source_scale) {
    const float whole = __builtin_amdgcn_exp2f(w[LIN_HI + 63] + w[LIN_LO + 63]);
#pragma unroll
    for (int a = 0; a < AT; ++a)
#pragma unroll
      for (int n = 0; n < NT; ++n) s[a][n] *= whole;
    const int c = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      __builtin_amdgcn_sched_barrier(0);
      Frag zw[NT][PARTS];
      float weight[8];
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        const float4 u = *reinterpret_cast<const float4*>(w + (REV ? LIN_FRONT : LIN_BEHIND) + 32 * v + 8 * c + j);
        weight[j] = u.x * source_scale; weight[j + 1] = u.y * source_scale; weight[j + 2] = u.z * source_scale; weight[j + 3] = u.w * source_scale;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (float)zf[v][n][j] * weight[j];
        lin_split<T, PARTS>(x, zw[n]);
      }
      auto rows = [&](int a) LACT_INLINE_LAMBDA { return LinFrag<T, DX>::template cols<8>(y, 32 * (a >> 1) + 4 * (a & 1), v); };
      Frag yf[3];
      yf[0] = rows(0);
      yf[1] = rows(1);
#pragma unroll
      for (int a = 0; a < AT; ++a) {
        if (a + 2 < AT) yf[(a + 2) % 3] = rows(a + 2);
#pragma unroll
        for (int p = 0; p < PARTS; ++p)      // (products of one sum after another wait for each other)
#pragma unroll
          for (int n = 0; n < NT; ++n) s[a][n] = mma16(yf[a % 3], zw[n][p], s[a][n]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
};

// A chunk's rows of one operand, 64 from token t on; rows past the end repeat the last one.
template <typename T, int D>
__device__ __forceinline__ void lin_copy(const LinRows<T>& m, int b, int h, int t, int L, uint32_t lds, int wave) {
  using S = MaskTile<T, D>;
  const T* from = uniform(m.p + b * m.bs + (long long)t * m.ld + (long long)h * D);
#pragma unroll
  for (int i = 0; i < S::G / 4; ++i) {
    const int c = (wave + i * 4) * 64 + (threadIdx.x & 63), r = c / S::G, slot = c % S::G;
    dma16<false>(from, (uint32_t)min(r, L - 1 - t) * (uint32_t)m.ld * (uint32_t)sizeof(T) + (uint32_t)((slot ^ S::key(r)) << 4), lds + (wave + i * 4) * 1024);
  }
}

// The walk over a segment.  REV: from its end to its beginning, sources are the later tokens.
// GATE: also dots[t], for the gradient of the decays.  Forwards (x, y, z, w = dout, v, k, q): the state's share in q_t . dq_t, and row sum minus column sum
// of M at t; backwards (x, y, z, w = k, q, dout, v): the state's share in v_t . dv_t.
// ROUNDED: only rounded outputs depend on the state, which then is added to in products of one part.
template <typename T, int DX, int DZ, bool REV, bool GATE, bool ROUNDED>
__device__ __forceinline__ void lin_walk(const LinParams<T>& p, int item, char* smem) {
  using Sh = LinShape<T, DX, DZ, GATE>;
  using St = LinState<T, DX, DZ>;
  using Frag = typename AttnType<T>::Frag;
  using FX = LinFrag<T, DX>;
  using FZ = LinFrag<T, DZ>;
  using FP = LinFrag<T, 64>;
  constexpr int NT = St::NT, UX = DX / 32, UZ = DZ / 32, SP = GATE ? lin_parts<T>() : 1;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane >> 4, li = lane & 15;
  const int seg = item % p.segments, bh = item / p.segments, b = p.by_heads.div(bh), h = bh - b * p.H;
  const int L = p.L, chunks = (L + 63) / 64, first = seg * p.seg_chunks, n = min(p.seg_chunks, chunks - first);
  char* pairs = smem + Sh::BUFFERS * Sh::STAGE;
  float* sums = reinterpret_cast<float*>(pairs + Sh::PAIRS);
  int* spoilt = reinterpret_cast<int*>(pairs + Sh::PAIRS + Sh::SUMS);
  if (threadIdx.x == 0) *spoilt = 0;
  const float* weights = uniform(p.weights + (size_t)bh * chunks * 256);
  const uint32_t lds0 = lds_addr(smem);
  auto token = [&](int i) { return (first + (REV ? n - 1 - i : i)) * 64; };
  auto issue = [&](int i) LACT_INLINE_LAMBDA {
    const int t = token(i);
    const uint32_t to = lds0 + i % Sh::BUFFERS * Sh::STAGE;
    lin_copy<T, DX>(p.x, b, h, t, L, to, wave);
    lin_copy<T, DX>(p.y, b, h, t, L, to + Sh::X, wave);
    lin_copy<T, DZ>(p.z, b, h, t, L, to + 2 * Sh::X, wave);
    if (GATE) lin_copy<T, DZ>(p.w, b, h, t, L, to + 2 * Sh::X + Sh::Z, wave);
    if (wave == 0) dma16<false>(weights + (long long)t * 4, lane * 16, to + Sh::STAGE - 1024);
  };
  St st;
  const float* start = p.states ? p.states + ((size_t)seg * p.B * p.H + bh) * (DX * DZ) : p.state0 ? p.state0 + (size_t)bh * (DX * DZ) : nullptr;
  if (start) st.load(start, p.transposed, wave);
  else st.zero();
  const bool final = p.last && seg == (REV ? 0 : p.segments - 1);
  issue(0);
  for (int i = 0; i < n; ++i) {
    const int t0 = token(i);
    if constexpr (GATE) {
      const int at = REV ? n - i : i;      // chunks of the segment on the earlier side of here
      if (p.between && i > 0 && at % LIN_STRETCH == 0)
        st.store(p.between + (((size_t)seg * (p.stretches - 1) + at / LIN_STRETCH - 1) * p.B * p.H + bh) * (DX * DZ), p.transposed, wave);
    }
    if (i == 0) wait_vmcnt<0>();
    __syncthreads();      // the chunk is there, and every wave is through with the pairs of the one before
    if (Sh::BUFFERS == 2 && i + 1 < n) issue(i + 1);
    const char* x = smem + i % Sh::BUFFERS * Sh::STAGE;
    const char* y = x + Sh::X;
    const char* z = y + Sh::X;
    const char* w = z + Sh::Z;
    const float* lw = reinterpret_cast<const float*>(x + Sh::STAGE - 1024);
    // Pairs of outputs [16 wave, +16) with their sources, [output][source] in LDS
    {
      constexpr bool PAIRED = GATE && !REV;
      const float my_hi = lw[LIN_HI + 16 * wave + li], my_lo = lw[LIN_LO + 16 * wave + li];
      float rowsum = 0.f;
      Frag xr[UX], wr[PAIRED ? UZ : 1];
#pragma unroll
      for (int u = 0; u < UX; ++u) xr[u] = FX::rows(x, wave, u);
      if constexpr (PAIRED)
#pragma unroll
        for (int u = 0; u < UZ; ++u) wr[u] = FZ::rows(w, wave, u);
#pragma unroll
      for (int jt = 0; jt < 4; ++jt) {
        const bool none = REV ? jt < wave : jt > wave;
        if (none && (jt >> 1) != (wave >> 1)) continue;      // no product reads it
        float v[4] = {0.f, 0.f, 0.f, 0.f}, m[4] = {0.f, 0.f, 0.f, 0.f};
        if (!none) {
          f32x4 acc, other;
          lin_zero(acc);
          lin_zero(other);
          Frag yf[UX], zr[PAIRED ? UZ : 1];
#pragma unroll
          for (int u = 0; u < UX; ++u) yf[u] = FX::rows(y, jt, u);
          if constexpr (PAIRED)
#pragma unroll
            for (int u = 0; u < UZ; ++u) zr[u] = FZ::rows(z, jt, u);
#pragma unroll
          for (int u = 0; u < UX; ++u) acc = mma16(yf[u], xr[u], acc);
          if constexpr (PAIRED)
#pragma unroll
            for (int u = 0; u < UZ; ++u) other = mma16(zr[u], wr[u], other);
          const float4 h4 = *reinterpret_cast<const float4*>(lw + LIN_HI + 16 * jt + 4 * c), l4 = *reinterpret_cast<const float4*>(lw + LIN_LO + 16 * jt + 4 * c);
          const float hi[4] = {h4.x, h4.y, h4.z, h4.w}, lo[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = 16 * jt + 4 * c + r, o = 16 * wave + li;
            const float e = REV ? lin_between(hi[r], lo[r], my_hi, my_lo) : lin_between(my_hi, my_lo, hi[r], lo[r]);
            const bool on = (REV ? j >= o : j <= o) && t0 + max(j, o) < L;
            v[r] = on ? acc[r] * e * p.pair_scale : 0.f;
            if constexpr (GATE && !REV) {
              m[r] = on && j != o ? v[r] * other[r] : 0.f;
              rowsum += m[r];
            }
          }
        }
        Elem<T>::store4(reinterpret_cast<T*>(const_cast<char*>(FP::at(pairs, 16 * wave + li, 16 * jt + 4 * c))), v[0], v[1], v[2], v[3]);
        if constexpr (GATE && !REV) {      // columns of M over the wave's outputs
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            m[r] = sum16(m[r]);
            if (li == 0) sums[256 + wave * 64 + 16 * jt + 4 * c + r] = m[r];
          }
        }
      }
      if constexpr (GATE && !REV) {
        rowsum += __shfl_xor(rowsum, 16, 64);
        rowsum += __shfl_xor(rowsum, 32, 64);
        // (tiles that were passed over hold nothing)
#pragma unroll
        for (int jt = 0; jt < 4; ++jt)
          if (jt > wave && (jt >> 1) != (wave >> 1) && li == 0)
#pragma unroll
            for (int r = 0; r < 4; ++r) sums[256 + wave * 64 + 16 * jt + 4 * c + r] = 0.f;
        wave_lds_fence();
        if (lane < 16) sums[256 + wave * 64 + 16 * wave + li] -= rowsum;
      }
    }
    // The state's share: columns of the output are tokens
    f32x4 o[4][NT];
#pragma unroll
    for (int it = 0; it < 4; ++it)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) lin_zero(o[it][nt]);
    {
      // operands two steps ahead of the products: a wave waits for LDS longer than for them
      Frag xf[3], sf[NT][SP];
      xf[0] = FX::rows(x, 0, 0);
      xf[1] = FX::rows(x, 1, 0);
#pragma unroll
      for (int e = 0; e < 4 * UX; ++e) {
        const int u = e / 4, it = e % 4;
        if (e + 2 < 4 * UX) xf[(e + 2) % 3] = FX::rows(x, (e + 2) % 4, (e + 2) / 4);
        if (it == 0) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = st.s[2 * u + (j >> 2)][nt][j & 3];
            lin_split<T, SP>(v, sf[nt]);
          }
        }
#pragma unroll
        for (int q = 0; q < SP; ++q)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) o[it][nt] = mma16(sf[nt][q], xf[e % 3], o[it][nt]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const float e = lw[(REV ? LIN_BEHIND : LIN_FRONT) + 16 * it + li] * p.state_scale;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) o[it][nt] *= e;
      if constexpr (GATE) {
        float d = 0.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float v[4];
          Elem<T>::load4(reinterpret_cast<const T*>(FZ::at(w, 16 * it + li, wave * (DZ / 4) + nt * 16 + 4 * c)), v);
#pragma unroll
          for (int r = 0; r < 4; ++r) d = fmaf(v[r], o[it][nt][r], d);
        }
        d += __shfl_xor(d, 16, 64);
        d += __shfl_xor(d, 32, 64);
        if (lane < 16) sums[wave * 64 + 16 * it + li] = d;
      }
    }
    Frag zf[2][NT];
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) zf[v][nt] = FZ::template cols<4>(z, wave * (DZ / 4) + nt * 16, v);
    bool bad = false;
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) bad |= unfinite(zf[v][nt]);
    if (__any(bad)) *spoilt = 1;
    if (i + 1 < n || final) st.template update<REV, ROUNDED ? 1 : lin_parts<T>()>(y, zf, lw, p.source_scale);
    __syncthreads();      // the pairs of all waves; nobody reads the chunk any more
    if constexpr (GATE)
      if (wave == 0 && t0 + lane < L) {
        float* to = p.dots + (size_t)bh * L + t0 + lane;
        *to = (sums[lane] + sums[64 + lane]) + (sums[128 + lane] + sums[192 + lane]);
        if constexpr (!REV) to[(size_t)p.B * p.H * L] = -((sums[256 + lane] + sums[320 + lane]) + (sums[384 + lane] + sums[448 + lane]));
      }
    // A value that is not finite must not reach the outputs that do not see its token (0 * inf): those chunks are summed term by term.
    if (__builtin_amdgcn_readfirstlane(lds_word(spoilt))) {
      for (int j = 0; j < 64; ++j) {
        if (t0 + j >= L) break;
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const int out = 16 * it + li;
          const float pr = Elem<T>::load(reinterpret_cast<const T*>(FP::at(pairs, out, j)));
          const bool sees = REV ? j >= out : j <= out;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float zv = Elem<T>::load(reinterpret_cast<const T*>(FZ::at(z, j, wave * (DZ / 4) + nt * 16 + 4 * c + r)));
              o[it][nt][r] = sees ? fmaf(pr, zv, o[it][nt][r]) : o[it][nt][r];
            }
        }
      }
      __syncthreads();
      if (threadIdx.x == 0) *spoilt = 0;
      if (Sh::BUFFERS == 1 && i + 1 < n) issue(i + 1);
    } else {
      if (Sh::BUFFERS == 1 && i + 1 < n) issue(i + 1);
#pragma unroll
      for (int it = 0; it < 4; ++it)
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          if (REV ? v < (it >> 1) : v > (it >> 1)) continue;
          const Frag pf = FP::rows(pairs, it, v);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) o[it][nt] = mma16(zf[v][nt], pf, o[it][nt]);
        }
    }
    wait_vmcnt<0>();      // for the next chunk, here and not behind the stores
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const int t = t0 + 16 * it + li;
      if (t < L)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          Elem<T>::store4(p.out + (((size_t)b * L + t) * p.H + h) * DZ + wave * (DZ / 4) + nt * 16 + 4 * c, o[it][nt][0], o[it][nt][1], o[it][nt][2], o[it][nt][3]);
    }
  }
  if (final) st.store(p.last + (size_t)bh * (DX * DZ), p.transposed, wave);
}

template <typename T> constexpr int lin_waves() { return sizeof(T) == 2 ? 2 : 1; }      // a SIMD's
template <typename T, int DK, int DV>
__global__ __launch_bounds__(256, lin_waves<T>()) void k_lin_forward(const LinParams<T> p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  prefetch_args<sizeof(p)>();
  lin_walk<T, DK, DV, false, false, false>(p, blockIdx.x, smem);
}
// All three gradients in one launch: the blocks of an item (segment and head) for dq, dv and dk lie eight apart, on one die and at about the same time, so
// that the inputs of the three come through its L2 once.
template <typename T>
struct LinBackward {
  LinParams<T> dq, dv, dk;
  int items;
};
template <typename T, int DK, int DV, bool GATE>
__global__ __launch_bounds__(256, lin_waves<T>()) void k_lin_backward(const LinBackward<T> p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  prefetch_args<sizeof(p)>();
  const int what = blockIdx.x / 8 % 3, item = blockIdx.x / 24 * 8 + blockIdx.x % 8;
  if (item >= p.items) return;
  if (what == 0) lin_walk<T, DV, DK, false, GATE, !GATE>(p.dq, item, smem);
  else if (what == 1) lin_walk<T, DK, DV, true, GATE, false>(p.dv, item, smem);
  else lin_walk<T, DV, DK, true, false, true>(p.dk, item, smem);
}

// What the tokens of a segment add to the state, into entry `seg + 1` (REV: `seg - 1`) of states, and the segment's sum of log2 decays.
template <typename T, int DX, int DZ, bool REV>
__global__ __launch_bounds__(256, lin_waves<T>()) void k_lin_segments(const LinParams<T> p, float* states, float* sums) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  using St = LinState<T, DX, DZ>;
  using Frag = typename AttnType<T>::Frag;
  constexpr int NT = St::NT, STAGE = MaskTile<T, DX>::BYTES + MaskTile<T, DZ>::BYTES + 1024;
  prefetch_args<sizeof(p)>();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int count = p.segments - 1, seg = blockIdx.x % count + (REV ? 1 : 0), bh = blockIdx.x / count, b = p.by_heads.div(bh), h = bh - b * p.H;
  const int L = p.L, chunks = (L + 63) / 64, first = seg * p.seg_chunks, n = min(p.seg_chunks, chunks - first);
  const float* weights = uniform(p.weights + (size_t)bh * chunks * 256);
  const uint32_t lds0 = lds_addr(smem);
  auto token = [&](int i) { return (first + (REV ? n - 1 - i : i)) * 64; };
  auto issue = [&](int i) LACT_INLINE_LAMBDA {
    const uint32_t to = lds0 + i % 2 * STAGE;
    lin_copy<T, DX>(p.y, b, h, token(i), L, to, wave);
    lin_copy<T, DZ>(p.z, b, h, token(i), L, to + MaskTile<T, DX>::BYTES, wave);
    if (wave == 0) dma16<false>(weights + (long long)token(i) * 4, lane * 16, to + STAGE - 1024);
  };
  St st;
  st.zero();
  double total = 0.0;
  issue(0);
  for (int i = 0; i < n; ++i) {
    wait_vmcnt<0>();
    __syncthreads();
    if (i + 1 < n) issue(i + 1);
    const char* y = smem + i % 2 * STAGE;
    const char* z = y + MaskTile<T, DX>::BYTES;
    const float* lw = reinterpret_cast<const float*>(y + STAGE - 1024);
    Frag zf[2][NT];
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) zf[v][nt] = LinFrag<T, DZ>::template cols<4>(z, wave * (DZ / 4) + nt * 16, v);
    st.template update<REV, lin_parts<T>()>(y, zf, lw, p.source_scale);
    total += (double)lw[LIN_HI + 63] + (double)lw[LIN_LO + 63];
  }
  st.store(states + ((size_t)(seg + (REV ? -1 : 1)) * p.B * p.H + bh) * (DX * DZ), p.transposed, wave);
  if (threadIdx.x == 0) sums[(size_t)seg * p.B * p.H + bh] = (float)total;
}

// entry[s + 1] += 2^sums[s] entry[s] from entry[0] = initial on, or (reverse) entry[s - 1] += 2^sums[s] entry[s] from the last on; a
// thread has four elements of one matrix, and reads eight entries ahead: nothing but the sum depends on the one before (32
// entries of 16 matrices of 64 x 128: 13.6 / 8.4 us).
__global__ __launch_bounds__(256) void k_lin_scan(int segments, long long matrices, int elems, int reverse, const float* initial, const float* sums, float* states) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4, n = matrices * elems;
  if (i >= n) return;
  const long long m = i / elems;
  float4 s = initial ? *reinterpret_cast<const float4*>(initial + i) : make_float4(0.f, 0.f, 0.f, 0.f);
  auto entry = [&](int k) { return reinterpret_cast<float4*>(states + (size_t)(reverse ? segments - 1 - k : k) * n + i); };
  *entry(0) = s;
  for (int k0 = 1; k0 < segments; k0 += 8) {
    float4 a[8];
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k0 + j < segments) {
        a[j] = *entry(k0 + j);
        f[j] = sums[(size_t)(reverse ? segments - k0 - j : k0 + j - 1) * matrices + m];
      }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k0 + j < segments) {
        const float w = __builtin_amdgcn_exp2f(f[j]);
        s = make_float4(fmaf(w, s.x, a[j].x), fmaf(w, s.y, a[j].y), fmaf(w, s.z, a[j].z), fmaf(w, s.w, a[j].w));
        *entry(k0 + j) = s;
      }
  }
}

// The gradient of a decay is what crosses its token.  In a chunk with the state S in front, the state's gradient dS behind, the state's shares a_i of its
// outputs (in q . dq) and b_j of its tokens (in v . dv):
//   dg_t = sum_(i >= t > j) M_ij + sum_(i >= t) a_i + sum_(j < t) b_j + e^G <dS, S>;
// the last term is X - sum b with X the crossing at the chunk's end, or nothing where the whole chunk's decay G leaves less than 2^-30: no rounding of a large
// crossing is then carried to tokens that it does not reach.  X of the chunk before is the last term + sum a; of a stretch's last chunk, <dS, S> there.
// A decay wears a crossing off, but not the roundings of a and b that its sum has gathered: hence stretches of eight chunks, between which the walks leave S and
// dS.  (16384 tokens, 260 heads of 64, a decay per head, fp32: the gradients' relative error 6e-6, with one sum for all of a sequence 3e-4.  20 x 2048 tokens, 16 heads of
// 128 in bf16, the whole step: 922 us, without stretches 888.)
// M's part is summed as rows minus columns from t on.  0 where the decay forgets everything, and where there is nothing in front to forget.
// Where the decay is the head's, the stretch's sum instead, into part [segment, stretch][B * H].  states [segments][n]: the state in front of each segment; ends: the
// gradient behind each (null with one segment); last, dlast: behind the last one (either null: no crossing); between, dbetween: between stretches.  One block
// per stretch and head, two chunks to a wave.
__global__ __launch_bounds__(256) void k_lin_decay_grad(int B, int L, int H, int segments, int seg_chunks, int stretches, int elems, const float* weights, const float* up,
                                                        const float* down, const float* states, const float* ends, const float* last, const float* dlast,
                                                        const float* between, const float* dbetween, LinDecay decay, int from_zero, float* dg, double* part) {
  constexpr int N = LIN_STRETCH / 4;
  __shared__ double tail[LIN_STRETCH], source[LIN_STRETCH], sums[4];
  __shared__ int cut[LIN_STRETCH];
  const int count = segments * stretches, at = blockIdx.x % count, seg = at / stretches, str = at - seg * stretches, bh = blockIdx.x / count;
  const int b = bh / H, h = bh - b * H, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const size_t n = (size_t)B * H * elems, own = (size_t)bh * elems;
  const int chunks = (L + 63) / 64, first = seg * seg_chunks + str * LIN_STRETCH, seg_end = min(chunks, (seg + 1) * seg_chunks);
  const int end = min(seg_end, first + LIN_STRETCH);      // (the last segment may have fewer stretches: nothing is left for the others)
  const float *a, *d;
  if (end < seg_end) {
    const size_t entry = ((size_t)seg * (stretches - 1) + str) * n + own;
    a = between + entry;
    d = dbetween + entry;
  } else if (seg + 1 < segments) {
    a = states + (seg + 1) * n + own;
    d = ends + seg * n + own;
  } else {
    a = last ? last + own : nullptr;
    d = dlast ? dlast + own : nullptr;
  }
  double crossing = 0.0;
  if (a && d && first < end)
#pragma unroll 4
    for (int i = threadIdx.x * 4; i < elems; i += 1024) {
      const float4 u = *reinterpret_cast<const float4*>(a + i), v = *reinterpret_cast<const float4*>(d + i);
      crossing += (double)u.x * v.x + (double)u.y * v.y + (double)u.z * v.z + (double)u.w * v.w;
    }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) crossing += __shfl_xor(crossing, o, 64);
  if (lane == 0) sums[wave] = crossing;
  // the latest chunk first; lane 0 holds a chunk's latest token
  const float* ends_of = weights + ((size_t)bh * chunks) * 256 + 63;
  double v[N], from[N], pairs[N];      // a - b, b, M
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int c = end - 1 - wave * N - k, t = c * 64 + 63 - lane;
    const size_t i = (size_t)bh * L + t;
    const bool on = c >= first && t < L;
    from[k] = on ? (double)down[i] : 0.0;
    v[k] = on ? (double)up[i] - from[k] : 0.0;
    pairs[k] = on ? (double)up[i + (size_t)B * H * L] : 0.0;
    if (lane == 0 && c >= first) cut[wave * N + k] = ends_of[(size_t)c * 256 + LIN_HI] + ends_of[(size_t)c * 256 + LIN_LO] < -30.f;
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double u = __shfl_up(v[k], o, 64), w = __shfl_up(pairs[k], o, 64);
      if (lane >= o) {
        v[k] += u;
        pairs[k] += w;
      }
      from[k] += __shfl_xor(from[k], o, 64);
    }
    if (lane == 63) {
      tail[wave * N + k] = v[k];
      source[wave * N + k] = from[k];
    }
  }
  __syncthreads();
  double run = (sums[0] + sums[1]) + (sums[2] + sums[3]), sum = 0.0, base[N];
#pragma unroll
  for (int k = 0; k < LIN_STRETCH; ++k)
    if (end - 1 - k >= first) {
      const double x = cut[k] ? source[k] : run;
      if (k / N == wave) base[k % N] = x;
      run = x + tail[k];
    }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int c = end - 1 - wave * N - k, t = c * 64 + 63 - lane;
    if (c >= first && t < L) {
      const double x = decay.at(b, t, h, L, H) <= LIN_MIN_LOG || (from_zero && t == 0) ? 0.0 : base[k] + v[k] + pairs[k];
      if (decay.per_token) dg[((size_t)b * L + t) * H + h] = (float)x;
      else sum += x;
    }
  }
  if (!decay.per_token) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    __syncthreads();      // (the crossing's sums have been read)
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) part[(size_t)at * B * H + bh] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  }
}
// One wave per head: the sum of part [rows][H].
__global__ __launch_bounds__(64) void k_lin_decay_sum(int rows, int H, const double* part, float* dg) {
  double s = 0.0;
  for (int r = threadIdx.x; r < rows; r += 64) s += part[(size_t)r * H + blockIdx.x];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if (threadIdx.x == 0) dg[blockIdx.x] = (float)s;
}

// ---- one token: S' = e^g S + k v^T, o = scale S'^T q.  Bound by the state's way in and out: 1024 states of 128 x 128, 135 MB, 21.6 us, 6.2 TB/s (in part from
// the cache).  A block has 32 columns of one head's state: 8 lanes of four columns,
// 32 rows at a time.
template <typename T>
struct LinStepParams {
  int H, DK, DV, per_token;            // g: [B, H] or [H]
  const T* q; const T* k; const T* v;  // [B, H, D], batch strides
  long long bsq, bsk, bsv;
  const float* g;
  const float* state;
  float* state_out;                    // may be `state`
  float scale;
  T* out;                              // [B, H, DV]
};
template <typename T>
__global__ __launch_bounds__(256) void k_lin_step(const LinStepParams<T> p) {
  __shared__ float4 red[4][8];
  const int parts = p.DV / 32, bh = blockIdx.x / parts, col = (blockIdx.x - bh * parts) * 32 + (threadIdx.x & 7) * 4, b = bh / p.H, h = bh - b * p.H;
  const int row = threadIdx.x >> 3;
  const float decay = __expf(p.g[p.per_token ? bh : h]);
  const T* q = p.q + b * p.bsq + h * p.DK;
  const T* k = p.k + b * p.bsk + h * p.DK;
  float v[4];
  Elem<T>::load4(p.v + b * p.bsv + h * p.DV + col, v);
  const float* s = p.state + (size_t)bh * p.DK * p.DV + col;
  float* s_out = p.state_out + (size_t)bh * p.DK * p.DV + col;
  float4 x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (row + 32 * i < p.DK) x[i] = *reinterpret_cast<const float4*>(s + (size_t)(row + 32 * i) * p.DV);
  float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = row + 32 * i;
    if (r >= p.DK) break;
    const float kr = Elem<T>::load(k + r), qr = Elem<T>::load(q + r);
    const float4 y = make_float4(fmaf(decay, x[i].x, kr * v[0]), fmaf(decay, x[i].y, kr * v[1]), fmaf(decay, x[i].z, kr * v[2]), fmaf(decay, x[i].w, kr * v[3]));
    *reinterpret_cast<float4*>(s_out + (size_t)r * p.DV) = y;
    o[0] = fmaf(qr, y.x, o[0]); o[1] = fmaf(qr, y.y, o[1]); o[2] = fmaf(qr, y.z, o[2]); o[3] = fmaf(qr, y.w, o[3]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int m = 8; m < 64; m <<= 1) o[i] += __shfl_xor(o[i], m, 64);
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) < 8) red[wave][threadIdx.x & 7] = make_float4(o[0], o[1], o[2], o[3]);
  __syncthreads();
  if (threadIdx.x < 8) {
    float4 a = red[0][threadIdx.x];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const float4 u = red[w][threadIdx.x];
      a.x += u.x; a.y += u.y; a.z += u.z; a.w += u.w;
    }
    Elem<T>::store4(p.out + (size_t)bh * p.DV + col, a.x * p.scale, a.y * p.scale, a.z * p.scale, a.w * p.scale);
  }
}

}  // namespace lact
