// Rotary positions with several axes: the channels of a head in pairs, pair p turned by the angle of its axis' position times its frequency:
//
//   (x, y) -> (x cos a - y sin a, x sin a + y cos a),   a = positions[.., axis p] f_p
//
// for the queries' and the keys' heads in one launch.  The gradient is the same with -a.  Channels behind the last pair go through as they are.
//
// An angle is formed once for all heads of a token, in quarter turns in fp64 (a far position times a frequency in fp32 would have lost its place in the turn), of
// which the whole ones are taken off before the rest is rounded to fp32: what is left is at most half a quarter, and its sine and cosine are the first terms of their series.
// Bound by memory: every channel is read once and written once.
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
  int B, L, D, pairs, axes;
  int per;                                    // heads of a block
  int units, tokens;                          // lanes to a token, tokens of a block
  UDiv by_units, by_l;
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
__device__ __forceinline__ Turn turn_of_pair(const RotaryParams& p, int b, int t, int pair) {
  if (pair >= p.pairs) return Turn{1.f, 0.f};
  return turn_of(position_of(p, b, t, p.axis[pair]) * p.frequency[pair], p.sign);
}

// One pair, of which what is not turned keeps its bits (an infinity times a sine of 0 is NaN).
template <typename T>
__device__ __forceinline__ void turn_pair(const Turn& w, T a, T b, T& c, T& d) {
  const float x = Elem<T>::load(&a), y = Elem<T>::load(&b);
  Elem<T>::store(&c, fmaf(x, w.c, -(y * w.s)));
  Elem<T>::store(&d, fmaf(x, w.s, y * w.c));
}

template <typename T, int N> struct alignas(sizeof(T) * N < 16 ? sizeof(T) : 16) RotaryVec { T v[N]; };

// A lane has V channels of a token's heads, and with halves apart (pairs p and p + pairs) V others.  V = 16 bytes where all sizes, strides and addresses allow
// it, else 1 (2 where pairs lie side by side).
template <typename T, int V, bool SIDE>
__global__ __launch_bounds__(256) void k_rotary(const RotaryParams p) {
  using Vec = RotaryVec<T, V>;
  const int slot = p.by_units.div(threadIdx.x), unit = threadIdx.x - slot * p.units;
  const long long token = (long long)blockIdx.x * p.tokens + slot;
  if (slot >= p.tokens || token >= (long long)p.B * p.L) return;
  const int b = p.by_l.div((int)token), t = (int)token - b * p.L;
  constexpr int N = SIDE ? V / 2 : V;
  const int turning = SIDE ? (2 * p.pairs + V - 1) / V : p.pairs / V;      // units with a pair
  const bool turns = unit < turning;
  const int first = SIDE || turns ? unit * V : 2 * p.pairs + (unit - turning) * V;
  Turn w[N];
  bool still[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int pair = SIDE ? unit * N + j : unit * V + j;
    still[j] = !turns || pair >= p.pairs;
    w[j] = still[j] ? Turn{1.f, 0.f} : turn_of_pair(p, b, t, pair);
  }
  const int h0 = blockIdx.y * p.per, h1 = min(h0 + p.per, p.op[0].heads + p.op[1].heads);
#pragma unroll 4
  for (int g = h0; g < h1; ++g) {
    const RotaryOperand& o = p.op[g >= p.op[0].heads];
    const int h = g >= p.op[0].heads ? g - p.op[0].heads : g;
    const T* x = static_cast<const T*>(o.x) + b * o.bs + t * o.ls + h * o.hs;
    T* y = static_cast<T*>(o.y) + (token * o.heads + h) * p.D;
    Vec u = *reinterpret_cast<const Vec*>(x + first), r = u;
    if constexpr (SIDE) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (!still[j]) turn_pair<T>(w[j], u.v[2 * j], u.v[2 * j + 1], r.v[2 * j], r.v[2 * j + 1]);
    } else if (turns) {
      Vec u2 = *reinterpret_cast<const Vec*>(x + first + p.pairs), r2;
#pragma unroll
      for (int j = 0; j < N; ++j) turn_pair<T>(w[j], u.v[j], u2.v[j], r.v[j], r2.v[j]);
      *reinterpret_cast<Vec*>(y + first + p.pairs) = r2;
    }
    *reinterpret_cast<Vec*>(y + first) = r;
  }
}

}  // namespace lact
