// Rotary positions: what turning rows of heads (rotary.hip) and turning them on their way
// into a paged cache (rotary_append.hip) share.
//
// Frequency i of n turns a pair (a, b) of a row's first 2 n dims by angle = p f_i:
//   a' = a cos - b sin,  b' = b cos + a sin
// with the pair (i, i + n), or (2 i, 2 i + 1) where neighbours are turned (interleaved).
#pragma once

#include "common.h"

namespace la {

constexpr int RO_NT = 256;

// (cos, sin) of p f.  The turns p f / 2 pi are counted in 64 bits, in which a product of a
// 31-bit position and a 24-bit frequency rounds by 2^-53 of itself: position 2^31 - 1 at
// frequency 1 is off by 5e-7, a million by 2e-10.  What is left of a quarter turn fits
// 32 bits: Taylor series, whose first terms left out are 2e-9 (sin) and 2e-10 (cos) at pi / 4.
__device__ __forceinline__ float2 ro_turn(double p, float f) {
  const double t = p * (double)f * 0.15915494309189533577;
  double r = t - __builtin_rint(t);
  const double quarter = __builtin_rint(4.0 * r);
  r = __builtin_fma(-0.25, quarter, r);
  const float y = (float)(r * 6.283185307179586477), y2 = y * y;
  float s = __builtin_fmaf(y2, 2.7557319e-6f, -1.9841270e-4f);
  s = __builtin_fmaf(y2, s, 8.3333333e-3f);
  s = __builtin_fmaf(y2, s, -1.6666667e-1f);
  s = __builtin_fmaf(y2 * y, s, y);
  float c = __builtin_fmaf(y2, -2.7557319e-7f, 2.4801587e-5f);
  c = __builtin_fmaf(y2, c, -1.3888889e-3f);
  c = __builtin_fmaf(y2, c, 4.1666667e-2f);
  c = __builtin_fmaf(y2, c, -0.5f);
  c = __builtin_fmaf(y2, c, 1.f);
  const int q = (int)quarter & 3;  // (-2 .. 2)
  const float c1 = q & 1 ? s : c, s1 = q & 1 ? c : s;
  return float2{q == 1 || q == 2 ? -c1 : c1, q >= 2 ? -s1 : s1};
}

// Positions of tokens (b, t) on axis a, and the frequencies.
struct RoAngles {
  const int32_t *pos, *axes;
  const float *freq;
  int64_t p_sa, p_sb, p_st;
  int32_t n, A, interleaved, inverse;

  __device__ __forceinline__ int axis(int f) const { return axes ? min(max(axes[f], 0), A - 1) : 0; }
  __device__ __forceinline__ float2 turn(double p, int f) const {
    float2 cs = ro_turn(p, freq[f]);
    if (inverse) cs.y = -cs.y;
    return cs;
  }
};

// A row in units of two chunks of V values: the chunks that hold both halves of V pairs, then
// what is not turned, two chunks at a time (of the last there may be one).
template <class E, int V>
struct RoUnit {
  typedef E vec __attribute__((ext_vector_type(V)));
  int oa, ob, f0;  // where the chunks begin (ob < 0: none); the first pair's frequency (< 0: not turned)

  static __host__ __device__ __forceinline__ int count(int D, int n) { return n / V + ((D - 2 * n) / V + 1) / 2; }

  __device__ __forceinline__ RoUnit(int u, int D, int n, bool interleaved) {
    const int turned = n / V;
    f0 = u < turned ? V * u : -1;
    if (u >= turned) {
      oa = 2 * n + 2 * V * (u - turned);
      ob = oa + V < D ? oa + V : -1;
    } else {
      oa = interleaved ? 2 * V * u : V * u;
      ob = interleaved ? oa + V : n + oa;
    }
  }
  __device__ __forceinline__ void load(const E *row, vec &a, vec &b) const {
    a = *(const vec *)(row + oa);
    b = *(const vec *)(row + (ob < 0 ? oa : ob));
  }
  __device__ __forceinline__ void store(E *row, const float (&x)[2 * V]) const {
    vec a, b;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      a[i] = (E)x[i];
      b[i] = (E)x[V + i];
    }
    *(vec *)(row + oa) = a;
    if (ob >= 0) *(vec *)(row + ob) = b;
  }
  static __device__ __forceinline__ void widen(const vec &a, const vec &b, float (&x)[2 * V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x[i] = (float)a[i];
      x[V + i] = (float)b[i];
    }
  }
};

// The V turns of a unit, of the angles' table of its token in LDS.
template <int V>
struct RoTurns {
  float c[V], s[V];
  __device__ __forceinline__ void load(const float2 *table, int f0) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 x = f0 >= 0 ? table[f0 + i] : float2{1.f, 0.f};
      c[i] = x.x;
      s[i] = x.y;
    }
  }
  __device__ __forceinline__ void apply(float (&x)[2 * V], bool interleaved) const {
    if (interleaved) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float a = x[2 * i], b = x[2 * i + 1];
        x[2 * i] = __builtin_fmaf(a, c[i], -(b * s[i]));
        x[2 * i + 1] = __builtin_fmaf(b, c[i], a * s[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float a = x[i], b = x[V + i];
        x[i] = __builtin_fmaf(a, c[i], -(b * s[i]));
        x[V + i] = __builtin_fmaf(b, c[i], a * s[i]);
      }
    }
    // (held in 32 bits: one instruction that turns and rounds to fp16, which some of the kernels
    // would get, gives other bits)
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) asm("" : "+v"(x[i]));
  }
};

// Values of a chunk: 16 bytes where sizes, strides and addresses allow it, else 8 (four values of
// 2 bytes), else one.  `bits`: all of the call's addresses (bytes) and row strides (values) or-ed.
inline int ro_vector(int esz, int64_t D, int64_t n, uint64_t addresses, uint64_t strides) {
  for (int v = 16 / esz; v > 1; v = v == 8 ? 4 : 1)
    if (n % v == 0 && D % v == 0 && addresses % (v * esz) == 0 && strides % v == 0) return v;
  return 1;
}

}  // namespace la
