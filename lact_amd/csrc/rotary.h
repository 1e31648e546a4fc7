// Rotary positions with several axes: the channels of a head in pairs, pair p turned by the angle of its axis' position times its frequency:
//
//   (x, y) -> (x cos a - y sin a, x sin a + y cos a),   a = positions[.., axis p] f_p
//
// for the queries' and the keys' heads in one launch.  The gradient is the same with -a.  Channels behind the last pair go through as they are.
//
// An angle is formed once for all heads of a token, in quarter turns in fp64 (a far position times a frequency in fp32 would have lost its place in the turn), of
// which the whole ones are taken off before the rest is rounded to fp32: what is left is at most half a quarter, and its sine and cosine are the first terms of their series.
// Bound by memory: every channel is read once and written once.  24960 tokens of a video, 12 + 12 heads of 128 in bf16, training step (forward and gradients): neighbouring pairs 122 us,
// in halves 139 (5.0 and 4.4 TB/s; a large copy reaches 5.0).  One head on its way at a time: 136 and 155.  A block has four of a token's heads at once, each of which forms the angles: two
// at once 127 and 142, eight 152 and 153.  With few heads fewer: 147285 tokens, 6 + 3 heads of 128, in halves, half of each head turned, forward, one / two / four at once 158 / 198 / 316 us;
// 24960 tokens, 8 + 8 heads, neighbouring pairs 43 / 39 / 43.  Tried: blocks that walk several tokens, with positions on their way ahead (registers: the forward alone 68 us
// for 59), 32 bytes a lane for neighbouring pairs.
#pragma once
#include "common.h"

namespace lact {

constexpr int ROTARY_PAIRS = 128;      // at most, of heads of at most twice as many channels

struct RotaryOperand {
  const void* x; void* y;                     // y: [B, L, heads, D] contiguous
  long long bs, ls, hs;                       // of x, in elements
  int heads;
};
struct RotaryParams {
  RotaryOperand op[2];
  int B, L, D, pairs;
  int per;                                    // heads of a block
  int units, across, tokens;                  // lanes to a head, heads of a token at once, tokens of a block
  UDiv by_units, by_across, by_l;
  const void* positions;
  int position_type;                          // 0: int32, 1: int64, 2: fp32
  long long pos_bs, pos_ls;
  float sign;                                 // -1: backward
  double frequency[ROTARY_PAIRS];             // in quarter turns
  uint8_t axis[ROTARY_PAIRS];
};

struct Turn { float c, s; };
// cos and sin of `quarters` quarter turns.  x = r pi / 2 is at most pi / 4; the first terms left out are x^11 / 11! < 2e-9 and x^12 / 12! < 2e-10.
__device__ __forceinline__ Turn turn_of(double quarters, float sign) {
  const double whole = __builtin_rint(quarters);
  const float x = (float)(quarters - whole) * 1.57079632679489662f, y = x * x;
  const int q = (int)(whole - 4.0 * __builtin_floor(whole * 0.25));
  float s = fmaf(y, fmaf(y, fmaf(y, fmaf(y, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), 1.f) * x;
  float c = fmaf(y, fmaf(y, fmaf(y, fmaf(y, fmaf(y, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f), 1.f);
  const float a = q & 1 ? -s : c, b = q & 1 ? c : s;
  const bool flip = q & 2;
  return Turn{flip ? -a : a, (flip ? -b : b) * sign};
}
__device__ __forceinline__ double position_of(const RotaryParams& p, int b, int t, int axis) {
  const long long at = b * p.pos_bs + t * p.pos_ls + axis;
  if (p.position_type == 0) return (double)static_cast<const int*>(p.positions)[at];
  if (p.position_type == 1) return (double)static_cast<const long long*>(p.positions)[at];
  return (double)static_cast<const float*>(p.positions)[at];
}

// One pair, whose bits stay as they are where nothing is turned (an infinity times a sine of 0 is NaN).
__device__ __forceinline__ void turn_pair(const Turn& w, float x, float y, float& c, float& d) {
  c = fmaf(x, w.c, -(y * w.s));
  d = fmaf(x, w.s, y * w.c);
}

// V elements as they lie in memory: 16 bytes in words, or one or two elements wherever they lie.
template <typename T, int V>
struct RotaryFew {
  T v[V];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = p[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = v[i];
  }
  __device__ __forceinline__ void unpack(float (&f)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = Elem<T>::load(v + i);
  }
  __device__ __forceinline__ void pack(const float (&f)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) Elem<T>::store(v + i, f[i]);
  }
  // pair j of neighbours as `from` has it
  __device__ __forceinline__ void take(const RotaryFew& from, int j) {
    v[2 * j] = from.v[2 * j];
    v[2 * j + 1] = from.v[2 * j + 1];
  }
};
template <typename T>
struct RotaryWide {
  static constexpr int V = 16 / sizeof(T);
  uint32_t w[4];
  __device__ __forceinline__ void load(const T* p) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]); }
  __device__ __forceinline__ void unpack(float (&f)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = sizeof(T) == 4 ? __uint_as_float(w[i & 3]) : i & 1 ? bf16_hi(w[i / 2]) : bf16_lo(w[i / 2]);
  }
  __device__ __forceinline__ void pack(const float (&f)[V]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = sizeof(T) == 4 ? __float_as_uint(f[i]) : pack_bf16(f[2 * i % V], f[(2 * i + 1) % V]);
  }
  __device__ __forceinline__ void take(const RotaryWide& from, int j) {
    constexpr int WORDS = sizeof(T) / 2;
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[WORDS * j + i] = from.w[WORDS * j + i];
  }
};

// A lane has V channels of a token's heads, and with halves apart (pairs p and p + pairs) V others.  V = 16 bytes where all sizes, strides and addresses allow
// it, else 1 (2 where pairs lie side by side).  Four heads are on their way at once.
template <typename T, int V, bool SIDE>
__global__ __launch_bounds__(256) void k_rotary(const RotaryParams p) {
  using Vec = typename std::conditional<V * sizeof(T) == 16, RotaryWide<T>, RotaryFew<T, V>>::type;
  const int slot = p.by_units.div(threadIdx.x), unit = threadIdx.x - slot * p.units, place = p.by_across.div(slot);
  const long long token = (long long)blockIdx.x * p.tokens + place;
  if (place >= p.tokens || token >= (long long)p.B * p.L) return;
  const int b = p.by_l.div((int)token), t = (int)token - b * p.L;
  constexpr int N = SIDE ? V / 2 : V, AHEAD = 4;
  const int turning = SIDE ? (2 * p.pairs + V - 1) / V : p.pairs / V;      // units with a pair
  const bool turns = unit < turning;
  const int first = SIDE || turns ? unit * V : 2 * p.pairs + (unit - turning) * V;
  Turn w[N];
  bool still[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int pair = (SIDE ? unit * N : unit * V) + j;
    still[j] = !turns || pair >= p.pairs;
    w[j] = still[j] ? Turn{1.f, 0.f} : turn_of(position_of(p, b, t, p.axis[pair]) * p.frequency[pair], p.sign);
  }
  // the lane's heads in turn, first the queries', then the keys'
  const int g0 = blockIdx.y * p.per + slot - place * p.across;
  const int end = min((int)(blockIdx.y + 1) * p.per, p.op[0].heads + p.op[1].heads);
#pragma unroll
  for (int op = 0; op < 2; ++op) {
    const RotaryOperand& o = p.op[op];
    const int before = op ? p.op[0].heads : 0, last = min(end, before + o.heads);
    int g = g0 + p.by_across.div(max(0, before - g0) + p.across - 1) * p.across;      // the first one from there on
    const T* x = static_cast<const T*>(o.x) + b * o.bs + t * o.ls + (g - before) * o.hs + first;
    T* y = static_cast<T*>(o.y) + (token * o.heads + g - before) * p.D + first;
    const long long xs = p.across * o.hs;
    const int ys = p.across * p.D;
    for (; g < last; g += AHEAD * p.across, x += AHEAD * xs, y += AHEAD * ys) {
      Vec u[AHEAD], u2[SIDE ? 1 : AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (g + i * p.across < last) {
          u[i].load(x + i * xs);
          if constexpr (!SIDE)
            if (turns) u2[i].load(x + i * xs + p.pairs);
        }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (g + i * p.across < last) {
          float f[V];
          u[i].unpack(f);
          if constexpr (SIDE) {
            Vec r;
#pragma unroll
            for (int j = 0; j < N; ++j) turn_pair(w[j], f[2 * j], f[2 * j + 1], f[2 * j], f[2 * j + 1]);
            r.pack(f);
#pragma unroll
            for (int j = 0; j < N; ++j)
              if (still[j]) r.take(u[i], j);
            r.store(y + i * ys);
          } else if (turns) {
            float f2[V];
            u2[i].unpack(f2);
#pragma unroll
            for (int j = 0; j < N; ++j) turn_pair(w[j], f[j], f2[j], f[j], f2[j]);
            u[i].pack(f);
            u2[i].pack(f2);
            u[i].store(y + i * ys);
            u2[i].store(y + i * ys + p.pairs);
          } else {
            u[i].store(y + i * ys);
          }
        }
    }
  }
}

}  // namespace lact
