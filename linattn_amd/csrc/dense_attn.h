// What the kernels of dense attention and of the key weights share: which rows a
// workgroup takes, and how key rows reach LDS.
#pragma once

#include "common.h"

namespace la {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int DA_BS = 64;  // keys of a staged tile

// Element types on the matrix cores: 32 x 32 += (32 x 16) (16 x 32), or 16 x 16 += (16 x
// 32) (32 x 16).
// A row's weights are 2^BIAS exp2(c s - m), where the reference m is raised to a row's
// maximum once that is more than GAP powers of two above it.  fp16 has no room below 2^-14
// (a weight loses bits there, and is 0 from 2^-25 on, while the row's sum, in fp32, has
// it), so weights use the top of its range: they keep their 11 bits down to 2^-29 of the
// row's largest, and what is lost below is at most 2^-40 of it.
// Headroom spares raises of the reference: four caches' chunks of 512 fp16 queries take 229
// us with 2^8 of it, 233 with 2^4, 237 with none; prompts 1 to 4 %
// longer with none; few rows over many keys the same.
struct DaBf16 {
  static constexpr float GAP = 8.f, BIAS = 0.f;
  typedef bf16x8 x8;
  typedef __bf16 elem;
  static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(x8 a, x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
struct DaF16 {
  static constexpr float GAP = 0.f, BIAS = 15.f;
  typedef f16x8 x8;
  typedef _Float16 elem;
  static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(x8 a, x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// 16-byte chunk swizzles of a staged row r.  A K read takes the same chunk of 32 rows in
// passes of two 8-lane groups ({0,3}, {1,2}, ...): rows 8i.. and 8j.. with bit 4
// different.  A transposed V read takes four consecutive chunks of four rows.
template <int D>
__device__ __forceinline__ int da_swz_k(int r) {
  return D == 128 ? (2 * (r & 7)) ^ ((r >> 4) & 1) : ((r >> 1) & 3) | (((r >> 4) & 1) << 2);
}
template <int D>
__device__ __forceinline__ int da_swz_v(int r) {
  return D == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1);
}

// Sequences of a call, as the kernels read them.
struct DaSeqs {
  const int32_t *cu_q, *cu_k, *q_len, *k_len;
  int64_t Tq, Tk;
  int32_t B, G;
};

// The rows of a tile: rows r0 .. r0 + R - 1 of the lq * G (query, head of the group) pairs
// of sequence b and one KV head, row r being query r / G of head r % G.
struct DaTile {
  int32_t b;       // -1: none, and r0 is the number of tiles there are
  int32_t r0, lq, lk;
  int64_t q0, k0;  // packed: first row of the sequence in q and in k
};

__device__ __forceinline__ int32_t da_cu(const int32_t *cu, int i, int64_t rows) {
  return (int32_t)min(max((int64_t)cu[i], (int64_t)0), rows);
}

// Sum and maximum over the wave, on the vector unit (as group_sum does it: a shuffle goes
// through LDS, and the search below makes many).
template <int CTRL>
__device__ __forceinline__ int32_t da_dpp(int32_t x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, false);
}
template <class F>
__device__ __forceinline__ int32_t da_wave_fold(int32_t x, F f) {
  x = f(x, da_dpp<0xB1>(x));
  x = f(x, da_dpp<0x4E>(x));
  x = f(x, da_dpp<0x141>(x));
  x = f(x, da_dpp<0x140>(x));
  const auto a = __builtin_amdgcn_permlane16_swap((uint32_t)x, (uint32_t)x, false, false);
  x = f((int32_t)a[0], (int32_t)a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap((uint32_t)x, (uint32_t)x, false, false);
  return __builtin_amdgcn_readfirstlane(f((int32_t)b[0], (int32_t)b[1]));
}
__device__ __forceinline__ int32_t da_wave_sum(int32_t x) {
  return da_wave_fold(x, [](int32_t a, int32_t b) { return a + b; });
}
__device__ __forceinline__ int32_t da_wave_max(int32_t x) {
  return da_wave_fold(x, [](int32_t a, int32_t b) { return max(a, b); });
}

__device__ __forceinline__ void da_seq(const DaSeqs &s, DaTile &t) {
  if (s.cu_q) {
    const int32_t a = da_cu(s.cu_q, t.b, s.Tq), e = da_cu(s.cu_q, t.b + 1, s.Tq);
    t.q0 = a;
    t.lq = max(e - a, 0);
    const int32_t *ck = s.cu_k ? s.cu_k : s.cu_q;
    const int32_t c = da_cu(ck, t.b, s.Tk), d = da_cu(ck, t.b + 1, s.Tk);
    t.k0 = c;
    t.lk = max(d - c, 0);
  } else {
    t.q0 = t.k0 = 0;
    t.lq = (int32_t)(s.q_len ? min(max((int64_t)s.q_len[t.b], (int64_t)0), s.Tq) : s.Tq);
    t.lk = (int32_t)(s.k_len ? min(max((int64_t)s.k_len[t.b], (int64_t)0), s.Tk) : s.Tk);
  }
}

// What is added to a row's scores (log2 units) for its weights, given the reference m in
// the scores' units.  Rounded such that where GAP is 0 no weight passes 2^BIAS, however
// large the scores.
template <class T>
__device__ __forceinline__ float da_ref(float m, float qscale) {
  if (m == __int_as_float(0xff800000)) return 0.f;
  if (T::BIAS == 0.f) return -m * qscale;
  return __builtin_fmaf(-m, qscale, T::BIAS - fabsf(m * qscale) * 0x1p-23f);
}

// A pointer, and a tile, that every lane has the same of, in scalar registers.
template <class P>
__device__ __forceinline__ P *da_scalar(P *x) {
  const uint64_t u = (uint64_t)(uintptr_t)x;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u), hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
  return (P *)(uintptr_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ DaTile da_uniform(DaTile t) {
  t.b = __builtin_amdgcn_readfirstlane(t.b);
  t.r0 = __builtin_amdgcn_readfirstlane(t.r0);
  t.lq = __builtin_amdgcn_readfirstlane(t.lq);
  t.lk = __builtin_amdgcn_readfirstlane(t.lk);
  t.q0 = __builtin_amdgcn_readfirstlane((int32_t)t.q0);
  t.k0 = __builtin_amdgcn_readfirstlane((int32_t)t.k0);
  return t;
}

// Tile number i of R rows, of queries (times the group's heads) or, by_k, of keys: the
// sequences' last tiles (the longest causal rows) first, so that a launch does not end
// with its longest workgroups.  Packed sequences: of the tiles ordered by their number
// within the sequence, descending, the i-th; every wave finds it by counting, the first 64
// sequences from registers.  Batched: every sequence has a tile of each number (one past
// its length has no live rows).
__device__ __forceinline__ DaTile da_tile(const DaSeqs &s, int32_t i, int32_t ntile, int R, bool by_k) {
  DaTile t;
  t.b = -1;
  t.r0 = t.lq = t.lk = 0;
  t.q0 = t.k0 = 0;
  if (!s.cu_q) {
    const int32_t per = ntile / s.B;
    t.b = i % s.B;
    t.r0 = (per - 1 - i / s.B) * R;
    da_seq(s, t);
    return t;
  }
  const int lane = threadIdx.x & 63;
  const int32_t *cu_k = s.cu_k ? s.cu_k : s.cu_q, *cu = by_k ? cu_k : s.cu_q;
  const int64_t rows = by_k ? s.Tk : s.Tq;
  const int32_t mul = by_k ? 1 : s.G;
  auto tiles = [&](int32_t n) -> int32_t { return (int32_t)(((int64_t)max(n, 0) * mul + R - 1) / R); };
  auto tiles_of = [&](int b) -> int32_t { return tiles(da_cu(cu, b + 1, rows) - da_cu(cu, b, rows)); };  // (b < B)
  // this lane's sequence, of the first 64: where its queries and keys begin and end
  const int bl = min(lane, s.B - 1);
  const int32_t qa = da_cu(s.cu_q, bl, s.Tq), qe = da_cu(s.cu_q, bl + 1, s.Tq);
  const int32_t ka = da_cu(cu_k, bl, s.Tk), ke = da_cu(cu_k, bl + 1, s.Tk);
  const int32_t mine = lane < s.B ? tiles(by_k ? ke - ka : qe - qa) : 0;
  auto above = [&](int32_t level) -> int32_t {  // tiles numbered `level` or more
    int32_t c = max(mine - level, 0);
    for (int b = 64 + lane; b < s.B; b += 64) c += max(tiles_of(b) - level, 0);
    return da_wave_sum(c);
  };
  const int32_t all = above(0);
  if (i >= all) {
    t.r0 = all;
    return t;
  }
  int32_t lo;
  if (s.B == 1) {
    t.b = 0;
    lo = all - 1 - i;
  } else {
    int32_t most = mine;
    for (int b = 64 + lane; b < s.B; b += 64) most = max(most, tiles_of(b));
    lo = 0;
    int32_t hi = da_wave_max(most);  // above(lo) > i >= above(hi)
    while (hi - lo > 1) {
      const int32_t mid = (lo + hi) >> 1;
      if (above(mid) > i) lo = mid;
      else hi = mid;
    }
    int32_t rank = i - above(hi);
    for (int b0 = 0; b0 < s.B; b0 += 64) {
      const int b = b0 + lane;
      const uint64_t has = __ballot((b0 == 0 ? mine : b < s.B ? tiles_of(b) : 0) > lo);
      const int32_t c = __popcll(has);
      if (rank < c) {
        const int before = __popcll(has & ((1ull << lane) - 1ull));
        const uint64_t at = __ballot(((has >> lane) & 1) && before == rank);
        t.b = b0 + __ffsll((unsigned long long)at) - 1;
        break;
      }
      rank -= c;
    }
    t.b = __builtin_amdgcn_readfirstlane(t.b);
  }
  t.r0 = lo * R;
  if (t.b >= 64) {
    da_seq(s, t);
    return t;
  }
  t.q0 = __builtin_amdgcn_readlane(qa, t.b);
  t.lq = max(__builtin_amdgcn_readlane(qe, t.b) - (int32_t)t.q0, 0);
  t.k0 = __builtin_amdgcn_readlane(ka, t.b);
  t.lk = max(__builtin_amdgcn_readlane(ke, t.b) - (int32_t)t.k0, 0);
  return t;
}

// Tiles of R rows that a call needs at most, for one KV head.
inline int64_t da_tiles(bool packed, int64_t B, int64_t Tq, int64_t G, int64_t R) {
  return packed ? Tq * G / R + B + 1 : B * ceil_div(Tq * G, R);
}

// Workgroup -> (stream of tiles that share keys, tile): all streams' first tiles first, so
// that the longest start first.  Consecutive workgroups go to the 8 XCDs in turn: with a
// multiple of 8 streams each XCD has streams of its own, whose keys its L2 holds.
__device__ __forceinline__ void da_stream(uint32_t wg, uint32_t ns, uint32_t &stream, uint32_t &tix) {
  stream = wg % ns;
  tix = wg / ns;
}

}  // namespace la
