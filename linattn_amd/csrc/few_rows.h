// Attention of up to 16 rows over many keys by one wave: what decode steps are made of.
//
// The keys are read once and bound everything, so a wave works on rounds of its own
// (32 keys, 16 in fp32: 8 KiB of K and 8 of V at D = 128), with the next round's K on its
// way into registers and V into the wave's own LDS while one is computed; no barrier.
// S^T = K Q^T by 16x16x32 products straight from the loaded rows (16x16x4 in fp32);
// O^T += V^T P^T with V^T by LDS transpose reads.  P enters that product as the sum of
// two terms of the inputs' type (16 bits of each weight, in fp16 down to 2^-23 of the row's
// largest), which the matrix cores have room for here.
#pragma once

#include "dense_attn.h"

//
// An infinity of V that a row sees meets weights of both signs in that sum (the second
// term's), and what is past the last key is that key again with weight 0: 0 and inf - inf
// where the result is infinite.  The caller looks for sums that are not finite: where its
// rows see every key, which dims of V hold a NaN or an infinity says what they are
// (few_marks, few_mark); else those rows are done again (few_row).

namespace la {

struct DaF32 {
  static constexpr float GAP = 8.f, BIAS = 0.f;
  typedef f32x4 x8;
  typedef float elem;
};

//
// V is read past the caches (nt): 64 caches of 2049 entries 118 -> 110 us, decode over
// 12345 keys 100 -> 93.  K is where NT_K is set, which the decode step gains from (110 ->
// 109, four caches of 16385 entries 62 -> 59) and dense_few_kernel loses (93 -> 99).
template <class T, int D, bool NT_K>
struct FewRows {
  typedef typename T::elem elem;
  typedef typename T::x8 x8;
  static constexpr bool F32 = sizeof(elem) == 4;
  static constexpr int RK = F32 ? 16 : 32;               // keys of a round
  static constexpr int CHE = 16 / (int)sizeof(elem);     // values of a 16-byte chunk
  static constexpr int CH = D / CHE, RP = 64 / CH;       // chunks of a row, rows of an LDS-DMA
  static constexpr int NX = RK / RP;                     // LDS-DMAs of a round's V
  static constexpr int STAGE = RK * D;                   // values of a staged round
  static constexpr int NK = F32 ? D / 16 : D / 32;       // chunks of K a lane holds for 16 keys
  static constexpr int LDS_BYTES = 2 * STAGE * (int)sizeof(elem);  // of one wave

  x8 qf[NK];
  f32x4 acc[D / 16];
  float m, l, thr, nmu;

  // chunk swizzle of a staged row: eight rows' pairs of chunks (fp32: four rows' four
  // chunks, four apart) that are read together lie in different banks
  static __device__ __forceinline__ int swz(int r) {
    return F32 ? 4 * ((r >> 2) & 3) : D == 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3);
  }

  // qrow: row lane % 16 (any valid row where there are fewer)
  __device__ __forceinline__ void begin(const elem *qrow) {
    const int c = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int s = 0; s < NK; ++s) qf[s] = *(const x8 *)(qrow + (F32 ? 16 * s + 4 * c : 32 * s + 8 * c));
    m = thr = __int_as_float(0xff800000);
    l = nmu = 0.f;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // Rounds first, first + step, ... below `rounds`, over keys round * RK ..  krow(key) and
  // vrow(key) point at a key's rows and are asked for keys < end only (keys past it are
  // the last one again, masked).  `lim` is the last key that row lane % 16 sees.  sink(key,
  // s) gets the row's scores (not scaled, -inf where masked) of keys key .. key + 3.  A weight
  // takes its score, the scale and the reference in one fma: what is rounded is their
  // difference, not a score that may be far larger.
  template <class KRow, class VRow, class Sink>
  __device__ __forceinline__ void walk(int first, int step, int rounds, int end, int lim, float qscale,
                                       elem *smem, KRow krow, VRow vrow, Sink sink) {
    const int lane = threadIdx.x & 63, c = lane >> 4, ri = lane & 15;
    const float ninf = __int_as_float(0xff800000);
    const float thr_gap = fminf(T::GAP / qscale, 3e38f);  // (finite: -inf + it stays)
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void_t *)smem);
    x8 kn[RK / 16][NK];
    auto fetch = [&](int r, int slot) {
#pragma unroll
      for (int x = 0; x < NX; ++x) {
        const int rr = RP * x + lane / CH;
        const elem *src = vrow(min(r * RK + rr, end - 1)) + CHE * ((lane % CH) ^ swz(rr));
        const uint32_t m0 = lds0 + (uint32_t)(slot * STAGE * (int)sizeof(elem) + x * 1024);
        asm volatile("global_load_lds_dwordx4 %0, off nt" ::"v"(src), "{m0}"(m0) : "memory");
      }
#pragma unroll
      for (int kt = 0; kt < RK / 16; ++kt) {
        const elem *src = krow(min(r * RK + 16 * kt + ri, end - 1));
#pragma unroll
        for (int s = 0; s < NK; ++s) {
          const x8 *x = (const x8 *)(src + (F32 ? 16 * s + 4 * c : 32 * s + 8 * c));
          if constexpr (NT_K) kn[kt][s] = __builtin_nontemporal_load(x);
          else kn[kt][s] = *x;
        }
      }
    };
    if (first < rounds) fetch(first, 0);
    int slot = 0;
    for (int r = first; r < rounds; r += step) {
      f32x4 st[RK / 16];
      // this round's V is in LDS, and the round before is read out of the other half
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      x8 kc[RK / 16][NK];
#pragma unroll
      for (int kt = 0; kt < RK / 16; ++kt)
#pragma unroll
        for (int s = 0; s < NK; ++s) {
          kc[kt][s] = kn[kt][s];
          settle(kc[kt][s]);
        }
      if (r + step < rounds) fetch(r + step, slot ^ 1);
#pragma unroll
      for (int kt = 0; kt < RK / 16; ++kt) {
        st[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
        // four sums: one chain of all dims would round four times as often (one token over 9000
        // fp32 keys: outputs off by 3.4e-7 of their norm in place of 1.1e-6)
        if constexpr (F32) {
          f32x4 part[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            part[e] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < NK; ++s)
              part[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(kc[kt][s][e], qf[s][e], part[e], 0, 0, 0);
          }
          st[kt] = (part[0] + part[1]) + (part[2] + part[3]);
        } else {
#pragma unroll
          for (int s = 0; s < NK; ++s) st[kt] = T::mfma16(kc[kt][s], qf[s], st[kt]);
        }
      }
      // register e: key 4 c + e
      const int d = lim - r * RK - 4 * c;
      float mx = ninf;
#pragma unroll
      for (int kt = 0; kt < RK / 16; ++kt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          st[kt][e] = 16 * kt + e <= d ? st[kt][e] : ninf;
          mx = fmaxf(mx, st[kt][e]);
        }
        sink(r * RK + 16 * kt + 4 * c, st[kt]);
      }
      if (__ballot(mx > thr) != 0) {
        const float mn = fmaxf(m, pair32_max(pair16_max(mx))), to = da_ref<T>(mn, qscale);
        const float alpha = m == ninf ? 0.f : fast_exp2(to - nmu);  // (both as rounded in the weights)
        m = mn;
        thr = mn + thr_gap;
        nmu = to;
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) acc[dt] *= alpha;
      }
      float part = 0.f;  // (a round's among themselves first: fewer roundings in l)
#pragma unroll
      for (int kt = 0; kt < RK / 16; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          st[kt][e] = fast_exp2(__builtin_fmaf(st[kt][e], qscale, nmu));
          part += st[kt][e];
        }
      l += part;
      const elem *sv = smem + slot * STAGE;
      if constexpr (F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int kr = 4 * c + e;
#pragma unroll
          for (int dt = 0; dt < D / 16; ++dt)
            acc[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(sv[kr * D + 4 * ((4 * dt + (ri >> 2)) ^ swz(kr)) + (ri & 3)],
                                                           st[0][e], acc[dt], 0, 0, 0);
        }
      } else {
        x8 hi, lo;  // k index 8 c + j: key 4 c + j of the first 16, then of the second
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          hi[j] = (elem)st[j >> 2][j & 3];
          lo[j] = (elem)(st[j >> 2][j & 3] - (float)hi[j]);
        }
        const int kr = 4 * c + (ri >> 2);
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
          const int at = kr * D + 8 * ((2 * dt + ((ri & 3) >> 1)) ^ swz(kr)) + 4 * (ri & 1);
          // (row kr + 16 has the same swizzle)
          const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)((const uint16_t *)sv + at));
          const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)((const uint16_t *)sv + at + 16 * D));
          const x8 vt = __builtin_bit_cast(x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
          acc[dt] = T::mfma16(vt, hi, acc[dt]);
          acc[dt] = T::mfma16(vt, lo, acc[dt]);
        }
      }
      slot ^= 1;
    }
    l = pair32_sum(pair16_sum(l));
  }

  // The wave's state into LDS: (reference in log2 units, l) of row i at ml[2 i], its D values at vals[i D ..]
  // (register e of dim tile dt: dim 16 dt + 4 c + e).
  __device__ __forceinline__ void put(float *ml, float *vals) const {
    const int lane = threadIdx.x & 63, c = lane >> 4, ri = lane & 15;
    if (c == 0) {
      ml[2 * ri] = m == __int_as_float(0xff800000) ? m : -nmu;
      ml[2 * ri + 1] = l;
    }
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
      *(f32x4 *)&vals[ri * (D + 4) + 16 * dt + 4 * c] = acc[dt];
  }
  static constexpr int VALS = 16 * (D + 4);  // floats of put's values
};

// Into marks[d] (LDS, D of them, cleared), by all NW waves of a workgroup: whether dim d of V
// holds a NaN (1), an infinity (2) or the negative one (4) for any of the keys a .. e - 1.
template <class E, int D, int NW, class VRow>
__device__ __forceinline__ void few_marks(uint32_t *marks, VRow vrow, int a, int e) {
  constexpr int CHE = 16 / (int)sizeof(E), CH = D / CHE, RP = 64 / CH;
  typedef E x8 __attribute__((ext_vector_type(CHE)));
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const float inf = __int_as_float(0x7f800000);
  uint32_t m = 0;  // three bits of each of the lane's dims
#pragma unroll 4
  for (int key = a + RP * w; key < e; key += RP * NW) {
    const x8 x = *(const x8 *)(vrow(min(key + lane / CH, e - 1)) + CHE * (lane % CH));
#pragma unroll
    for (int i = 0; i < CHE; ++i) {
      const float v = (float)x[i];
      m |= (v != v ? 1u : v == inf ? 2u : v == -inf ? 4u : 0u) << (3 * i);
    }
  }
#pragma unroll
  for (int i = 0; i < CHE; ++i)
    if ((m >> (3 * i)) & 7u) atomicOr(&marks[CHE * (lane % CH) + i], (m >> (3 * i)) & 7u);
}
// The sum of a row that sees all those keys, where the mark is not 0.
__device__ __forceinline__ float few_mark(uint32_t mark) {
  return __int_as_float(mark == 2u ? 0x7f800000 : mark == 4u ? 0xff800000 : 0x7fc00000);
}

// One row over keys a .. e - 1 (krow(key), vrow(key)), by a wave, key by key in fp32 (m in
// log2 units; lane i holds dims i D / 64 ..).  For rows whose matrix products met an
// infinity or a NaN of V in a way that the definition does not: it reads nothing else.
template <class E, int D, class KRow, class VRow>
__device__ __forceinline__ void few_row(const E *q, KRow krow, VRow vrow, int a, int e, float qscale, float *m_out,
                                        float *l_out, float *acc) {
  constexpr int N = D / 64;
  const int lane = threadIdx.x & 63;
  const float ninf = __int_as_float(0xff800000);
  float m = ninf, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  for (int key0 = a; key0 < e; key0 += 64) {
    const E *k = krow(min(key0 + lane, e - 1));
    float s = 0.f;
    for (int d = 0; d < D; ++d) s = __builtin_fmaf((float)q[d], (float)k[d], s);
    s = key0 + lane < e ? s * qscale : ninf;
    float mx = s;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    const float mn = fmaxf(m, mx);
    const float alpha = m == ninf ? 0.f : fast_exp2(m - mn);
    const float pr = fast_exp2(s - (mn == ninf ? 0.f : mn));
    m = mn;
    l = l * alpha + group_sum<64>(pr);
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] *= alpha;
    const int n = min(64, e - key0);
    for (int j = 0; j < n; ++j) {
      const float w = __shfl(pr, j, 64);
      const E *v = vrow(key0 + j) + lane * N;
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = __builtin_fmaf(w, (float)v[i], acc[i]);
    }
  }
  *m_out = m;
  *l_out = l;
}

}  // namespace la
