// rotary.cuh -- angles of rotary positions.
//
// Pair i of a row at position p turns by p * f_i radians.  f_i / 2 pi is held as a
// 64-bit fraction of a turn, so that p * f_i modulo a turn is one integer product
// whose upper bits fall away: the angle of position 2^31 is as good as that of
// position 1 (2^-64 of a turn a position, 2^-33 in all), where 32-bit floats have
// lost it past 2^20.
#pragma once

#include "common.cuh"

namespace grm_b200 {

struct Turn {
  float cos, sin;
};

// cos and sin of `position` (not negative) times `turns` 2^-64 turns.  The eighth of
// a turn next to the angle is taken off in integers; what is left, x within an
// eighth, goes into the Taylor series of sin and cos (the first terms left out are
// (pi/4)^11 / 11! = 2e-9 and (pi/4)^12 / 12! = 1e-10).  About 25 instructions.
__device__ __forceinline__ Turn turn_of(int position, uint64_t turns) {
  const uint64_t at = (uint64_t)(uint32_t)position * turns + ((uint64_t)1 << 61);
  const unsigned quarter = (unsigned)(at >> 62);
  // the rest in 2^-34 turns, within 2^31
  const int rest = (int)((int64_t)((at & (((uint64_t)1 << 62) - 1)) - ((uint64_t)1 << 61)) >> 30);
  const float x = __int2float_rn(rest) * (6.28318530717958648f * 0x1p-34f);
  const float y = x * x;
  float s = fmaf(y, 1.0f / 362880.0f, -1.0f / 5040.0f);
  s = fmaf(y, s, 1.0f / 120.0f);
  s = fmaf(y, s, -1.0f / 6.0f);
  s = fmaf(x * y, s, x);
  float c = fmaf(y, -1.0f / 3628800.0f, 1.0f / 40320.0f);
  c = fmaf(y, c, -1.0f / 720.0f);
  c = fmaf(y, c, 1.0f / 24.0f);
  c = fmaf(y, c, -0.5f);
  c = fmaf(y, c, 1.0f);
  const float a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;  // |cos|, |sin|
  Turn t;
  t.cos = quarter == 1 || quarter == 2 ? -a : a;
  t.sin = quarter >= 2 ? -b : b;
  return t;
}

// Where the pairs of a row lie, and how they turn.  The two members of pair i of
// `dim` values are at i and i + dim / 2 (GRM_B200_ROTARY_HALF), at 2 i and 2 i + 1
// (_INTERLEAVED), or taken from 2 i and 2 i + 1 and put to i and i + dim / 2
// (_PAIR_SWAP; taken off the other way round).
struct RotaryParams {
  const uint64_t* turns;  // [dim / 2]
  int dim, offset, layout;
  float amplitude;
};

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T round_to(float v);
template <>
__device__ __forceinline__ float round_to<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half round_to<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
// Two 16-bit values in a word.
template <typename T>
__device__ __forceinline__ float2 unpack(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
__device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t repack(float a, float b);
template <>
__device__ __forceinline__ uint32_t repack<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t repack<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// V values of one load or store: 8 (16-bit ones two to a word, which half the
// registers hold), or 1.
template <typename T, int V>
struct Values;
template <typename T>
struct Values<T, 1> {
  T v;
  __device__ __forceinline__ void get(float (&x)[1]) const { x[0] = to_float(v); }
  __device__ __forceinline__ void put(const float (&x)[1]) { v = round_to<T>(x[0]); }
};
template <typename T>
struct alignas(16) Values<T, 8> {
  uint32_t w[4];
  __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 u = unpack<T>(w[i]);
      x[2 * i] = u.x;
      x[2 * i + 1] = u.y;
    }
  }
  __device__ __forceinline__ void put(const float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = repack<T>(x[2 * i], x[2 * i + 1]);
  }
};
template <>
struct alignas(16) Values<float, 8> {
  float v[8];
  __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = v[i];
  }
  __device__ __forceinline__ void put(const float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x[i];
  }
};

// V pairs by their cos and sin.  IN, OUT: a pair's members lie side by side (in a and
// b one after another), else in a and b.
template <typename T, int V, bool IN, bool OUT>
__device__ __forceinline__ void turn_values(const float2 (&angle)[V], const Values<T, V>& a,
                                            const Values<T, V>& b, Values<T, V>* c,
                                            Values<T, V>* d) {
  float x[V], y[V], u[V], v[V];
  a.get(x);
  b.get(y);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float x1 = IN ? (2 * i < V ? x[2 * i % V] : y[2 * i % V]) : x[i];
    const float x2 = IN ? (2 * i + 1 < V ? x[(2 * i + 1) % V] : y[(2 * i + 1) % V]) : y[i];
    const float y1 = x1 * angle[i].x - x2 * angle[i].y, y2 = x2 * angle[i].x + x1 * angle[i].y;
    (OUT && 2 * i >= V ? v[2 * i % V] : u[OUT ? 2 * i % V : i]) = y1;
    (OUT && 2 * i + 1 < V ? u[(2 * i + 1) % V] : v[OUT ? (2 * i + 1) % V : i]) = y2;
  }
  c->put(u);
  d->put(v);
}

// The same of one head of 2 * half values, c the first pair.
template <typename T, int V, bool IN, bool OUT>
__device__ __forceinline__ void turn_pairs(int half, const float2 (&angle)[V], int c, const T* x,
                                           T* out) {
  using W = Values<T, V>;
  const W a = *reinterpret_cast<const W*>(x + (IN ? 2 * c : c));
  const W b = *reinterpret_cast<const W*>(x + (IN ? 2 * c + V : half + c));
  W y0, y1;
  turn_values<T, V, IN, OUT>(angle, a, b, &y0, &y1);
  *reinterpret_cast<W*>(out + (OUT ? 2 * c : c)) = y0;
  *reinterpret_cast<W*>(out + (OUT ? 2 * c + V : half + c)) = y1;
}

int check_rotary(const char* what, const grm_b200_rotary* r);
inline RotaryParams rotary_params(const grm_b200_rotary& r) {
  return {r.turns, r.dim, r.offset, r.layout, r.amplitude};
}

}  // namespace grm_b200
