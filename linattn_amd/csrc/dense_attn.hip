// Dense attention of prompts, chunks and single tokens with grouped heads, batched or
// packed (la_dense_attention; dense_attention, core.py:148-181).
//
// A workgroup takes R rows of one KV head of one sequence: row r is query r / G of head
// r % G of its group, so the heads of a group share every staged key, and a tile's rows
// end at nearly the same key.  It walks the keys in tiles of 64 with the running
// maximum and sum of a softmax: S^T = K Q^T, P = exp2(c S - m), O^T += V^T P^T.
#include <algorithm>

#include "few_rows.h"

namespace la {

struct DaKP {
  DaSeqs s;
  const void *q, *k, *v;
  void *out;
  float *lse;
  float *ws_ml, *ws_acc;  // parts: [row of q][head][split] (max, sum) and D values
  int64_t q_sb, q_sh, q_st, k_sb, k_sh, k_st, v_sb, v_sh, v_st, o_sb, o_sh, o_st, l_sb, l_sh;
  int32_t Hq, Hkv, ntile, splits, causal, out_dt, zero_rest;
  float qscale, thr_gap;  // log2(e) scale; the type's GAP / qscale
};

constexpr float DA_LN2 = 0.69314718055994530942f;

__device__ __forceinline__ float da_ninf() { return __int_as_float(0xff800000); }

// Four outputs of a row, 8- or 16-byte aligned.
__device__ __forceinline__ void da_store4(void *out, int64_t at, int dt, float x0, float x1, float x2, float x3) {
  if (dt == LA_F32) {
    *(float4 *)((float *)out + at) = float4{x0, x1, x2, x3};
  } else if (dt == LA_BF16) {
    *(uint2 *)((uint16_t *)out + at) =
        uint2{(uint32_t)f32_to_bf16_bits(x0) | ((uint32_t)f32_to_bf16_bits(x1) << 16),
              (uint32_t)f32_to_bf16_bits(x2) | ((uint32_t)f32_to_bf16_bits(x3) << 16)};
  } else {
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    *(f16x4 *)((_Float16 *)out + at) = f16x4{(_Float16)x0, (_Float16)x1, (_Float16)x2, (_Float16)x3};
  }
}
__device__ __forceinline__ void da_store1(void *out, int64_t at, int dt, float x) { store_from_f32(out, at, dt, x); }

// Where row (query t, head h) of a tile's sequence lies.
__device__ __forceinline__ int64_t da_out_at(const DaKP &p, const DaTile &tl, int64_t t, int h) {
  return (p.s.cu_q ? (tl.q0 + t) * p.o_st : tl.b * p.o_sb + t * p.o_st) + h * p.o_sh;
}
__device__ __forceinline__ int64_t da_lse_at(const DaKP &p, const DaTile &tl, int64_t t, int h) {
  return (p.s.cu_q ? tl.q0 + t : tl.b * p.l_sb + t) + h * p.l_sh;
}
__device__ __forceinline__ int64_t da_part_at(const DaKP &p, const DaTile &tl, int64_t t, int h, int split) {
  return (((p.s.cu_q ? tl.q0 + t : tl.b * p.s.Tq + t) * p.Hq + h) * p.splits) + split;
}

// Rows that no sequence holds: a batched tile's rows past the sequence's last query
// (first split), or, by the workgroups that got no tile, the packed rows outside of
// cu_q[0] .. cu_q[B].
template <int D>
__device__ __forceinline__ void da_zero_row(const DaKP &p, int64_t o, int64_t l, int lane) {
  for (int d = lane; d < D; d += 64) da_store1(p.out, o + d, p.out_dt, 0.f);
  if (p.lse && lane == 0) p.lse[l] = da_ninf();
}
template <int D>
__device__ void da_rest(const DaKP &p, const DaTile &tl, int R, int kvh, int split, int tix, int w, int nw) {
  if (split != 0) return;
  const int lane = threadIdx.x & 63, G = p.s.G;
  if (!p.s.cu_q) {
    const int64_t end = min((int64_t)tl.r0 + R, p.s.Tq * G);
    for (int64_t r = max((int64_t)tl.r0, (int64_t)tl.lq * G) + w; r < end; r += nw)
      da_zero_row<D>(p, da_out_at(p, tl, r / G, kvh * G + (int)(r % G)),
                     da_lse_at(p, tl, r / G, kvh * G + (int)(r % G)), lane);
    return;
  }
  if (!p.zero_rest || tl.b >= 0) return;
  const int64_t first = da_cu(p.s.cu_q, 0, p.s.Tq);
  const int64_t last = max(first, (int64_t)da_cu(p.s.cu_q, p.s.B, p.s.Tq));
  const int64_t n = (first + p.s.Tq - last) * G;
  for (int64_t r = (int64_t)(tix - tl.r0) * nw + w; r < n; r += (int64_t)(p.ntile - tl.r0) * nw) {
    int64_t t = r / G;
    if (t >= first) t += last - first;
    const int h = kvh * G + (int)(r % G);
    da_zero_row<D>(p, t * p.o_st + h * p.o_sh, t + h * p.l_sh, lane);
  }
}

// Rows r_first + i, i = i0, i0 + step, .. below NR, whose results are not finite, of which
// bit i of `bad` says so: those with an infinity or NaN of V among what their tiles (keys
// a .. end - 1) held and they do not see are done again; the others stand, but for ALL
// (few_row), and in fp16, where a weight below 2^-40 of the row's largest is 0 and its
// product with an infinity NaN: a dim's first keys with NaN and either infinity say what it
// is for each row.  (What a tile holds past the last key is that key again.)  Called last,
// when the rows are stored and the registers free.
template <class T, int D, int NR, bool ALL>
__device__ __forceinline__ void da_again(const DaKP &p, const DaTile &tl, int kvh, int split, int r_first,
                                          uint32_t bad, int a, int end, int i0, int step) {
  typedef typename T::elem E;
  const int lane = threadIdx.x & 63, G = p.s.G;
  const E *kb = (const E *)p.k + (p.s.cu_q ? tl.k0 * p.k_st : tl.b * p.k_sb) + kvh * p.k_sh;
  const E *vb = (const E *)p.v + (p.s.cu_q ? tl.k0 * p.v_st : tl.b * p.v_sb) + kvh * p.v_sh;
  constexpr bool LOST = !ALL && T::BIAS > 0.f;
  constexpr int N = D / 64;
  const float inf = __int_as_float(0x7f800000);
  int32_t at[3][N];  // of dim lane + 64 x
#pragma unroll
  for (int x = 0; x < N; ++x) at[0][x] = at[1][x] = at[2][x] = INT32_MAX;
  if constexpr (LOST) {
    const int32_t e = min(end, tl.lk);
#pragma unroll 8
    for (int32_t key = a; key < e; ++key)
#pragma unroll
      for (int x = 0; x < N; ++x) {
        const float v = (float)vb[key * p.v_st + lane + 64 * x];
        at[0][x] = min(at[0][x], v != v ? key : INT32_MAX);
        at[1][x] = min(at[1][x], v == inf ? key : INT32_MAX);
        at[2][x] = min(at[2][x], v == -inf ? key : INT32_MAX);
      }
  }
  wait_vmcnt<0>();  // (stores over those)
#pragma unroll 1
  for (int i = i0; i < NR; i += step) {
    if (!((bad >> i) & 1u)) continue;
    const int r = r_first + i, t = r / G, h = kvh * G + r % G;
    const int lim = p.causal ? min(tl.lk - 1, tl.lk - tl.lq + t) : tl.lk - 1;
    bool met = ALL;
    for (int key = max(max(lim + 1, a), 0); key < end && !ALL; ++key)
      for (int d = lane; d < D; d += 64)
        met = met || !(fabsf((float)vb[(int64_t)min(key, tl.lk - 1) * p.v_st + d]) < inf);
    if (__ballot(met) == 0) {
#pragma unroll
      for (int x = 0; x < N; ++x) {
        const bool up = at[1][x] <= lim, down = at[2][x] <= lim, nan = at[0][x] <= lim || (up && down);
        if (!nan && !up && !down) continue;
        const float y = nan ? __int_as_float(0x7fc00000) : up ? inf : -inf;
        if (p.splits > 1) p.ws_acc[da_part_at(p, tl, t, h, split) * D + lane + 64 * x] = y;
        else da_store1(p.out, da_out_at(p, tl, t, h) + lane + 64 * x, p.out_dt, y);
      }
      continue;
    }
    const E *q = (const E *)p.q + (p.s.cu_q ? (tl.q0 + t) * p.q_st : tl.b * p.q_sb + t * p.q_st) + h * p.q_sh;
    float m, l, acc[N];
    few_row<E, D>(q, [&](int key) { return kb + key * p.k_st; }, [&](int key) { return vb + key * p.v_st; }, a,
                  min(end, lim + 1), p.qscale, &m, &l, acc);
    if (p.splits > 1) {
      const int64_t pi = da_part_at(p, tl, t, h, split);
      if (lane == 0) {
        p.ws_ml[2 * pi] = m;
        p.ws_ml[2 * pi + 1] = l;
      }
      for (int x = 0; x < N; ++x) p.ws_acc[pi * D + lane * N + x] = acc[x];
      continue;
    }
    const int64_t o = da_out_at(p, tl, t, h);
    for (int x = 0; x < N; ++x)
      da_store1(p.out, o + lane * N + x, p.out_dt, l == 0.f ? 0.f : acc[x] / l);
    if (p.lse && lane == 0) p.lse[da_lse_at(p, tl, t, h)] = l == 0.f ? da_ninf() : (m + __log2f(l)) * DA_LN2;
  }
}

// bf16 / fp16 rows: NW waves of 32 rows.  K and V tiles go global -> LDS by LDS-DMA, K a
// tile ahead into the other of two slots, V while its tile is scored: 48 KiB a workgroup
// and at most 168 registers make three workgroups a CU, and with three waves a SIMD one
// wave's softmax runs beside another's products (two waves and two slots each: 7.8 ms for
// 32768 tokens of 32 heads on 8; three, on the same machine: 7.4, on others to 7.95, 1.11
// to 1.20 PFLOP/s; tile j + 1 scored beside the softmax of tile j in one wave's
// instructions: 10.5).  S^T by 32x32x16 products (A = K rows, B = q held
// in registers) leaves a lane 16 scores of one row, so masks, maxima and sums are per
// lane; O^T takes P from the same registers (the contraction index is mapped to the keys
// a lane holds) and V^T by LDS transpose reads.  P is rounded to the inputs' type for
// that product (to half a step, 2^-8 or 2^-11 of each weight, independently: as much as
// the output's own rounding; for fp16 of weights down to 2^-29 of the largest, DaF16); its
// sum l, and with it lse, is of the fp32 values.
// Bound by matrix and vector work together: over 32768 tokens the matrix unit is busy for
// 67 % of the cycles and the vector unit for 54 (the clock, 1.6 GHz then, gives way to
// both; a large bf16 product reaches 1.4 PFLOP/s).  Short sequences are bound by a
// workgroup's beginning and end: both units are busy for 49 % over twelve sequences of
// 14567 tokens; 14567 tokens of 32 heads on 8 run at 1.12 PFLOP/s as one sequence, 1.05 as four, 0.84 as
// twelve and 0.61 as twenty-four.
template <class T, int D, int NW>
__global__ __launch_bounds__(64 * NW, 3) void dense_attn_kernel(DaKP p) {
  constexpr int R = 32 * NW, BLK = DA_BS * D, CH = D / 8, RP = 64 / CH, NX = DA_BS / RP / NW;
  constexpr int NS = D / 16, ND = D / 32;
  typedef typename T::x8 x8;
  typedef typename T::elem elem;
  __shared__ __align__(16) uint16_t smem[3 * BLK];  // K slots 0, 1, then V
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hf = lane >> 5, r32 = lane & 31;
  uint32_t stream, tix;
  da_stream(blockIdx.x, (uint32_t)p.Hkv * p.splits, stream, tix);
  const int kvh = (int)(stream / (uint32_t)p.splits), split = (int)(stream % (uint32_t)p.splits);
  const DaTile tl = da_uniform(da_tile(p.s, (int)tix, p.ntile, R, false));
  const int G = p.s.G;
  if (tl.b < 0 || tl.r0 + R > tl.lq * G) da_rest<D>(p, tl, R, kvh, split, (int)tix, w, NW);
  if (tl.b < 0 || tl.r0 >= tl.lq * G) return;

  const int nrow = tl.lq * G, diag = tl.lk - tl.lq;
  auto limit = [&](int t) { return p.causal ? diag + t : tl.lk - 1; };  // last key seen
  const int r_first = tl.r0 + 32 * w;
  const int r_mine = min(r_first + r32, nrow - 1);
  const bool live = r_first + r32 < nrow, wave_live = r_first < nrow;
  const int t = r_mine / G, h = kvh * G + r_mine % G;
  const int lim = limit(t);
  const int lim_lo = __builtin_amdgcn_readfirstlane(limit(min(r_first, nrow - 1) / G));
  const int lim_hi = __builtin_amdgcn_readfirstlane(limit(min(r_first + 31, nrow - 1) / G));
  const int lim_tile = __builtin_amdgcn_readfirstlane(limit((min(tl.r0 + R, nrow) - 1) / G));
  const int n_all = lim_tile < 0 ? 0 : lim_tile / DA_BS + 1;
  int j0 = 0, j1 = n_all;
  if (p.splits > 1) {
    j0 = (int)((int64_t)n_all * split / p.splits);
    j1 = (int)((int64_t)n_all * (split + 1) / p.splits);
  }
  j0 = __builtin_amdgcn_readfirstlane(j0);
  j1 = __builtin_amdgcn_readfirstlane(j1);

  const uint16_t *kbh = (const uint16_t *)p.k + (p.s.cu_q ? tl.k0 * p.k_st : tl.b * p.k_sb) + kvh * p.k_sh;
  const uint16_t *vbh = (const uint16_t *)p.v + (p.s.cu_q ? tl.k0 * p.v_st : tl.b * p.v_sb) + kvh * p.v_sh;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void_t *)smem);
  // LDS-DMA: instruction x of wave w fills rows RP (NW x + w) + lane / CH, from a scalar base
  // and 32-bit offsets.  Rows past the last key are that key again (masked).
  uint32_t ko[NX], vo[NX];
#pragma unroll
  for (int x = 0; x < NX; ++x) {
    const int rr = RP * (NW * x + w) + lane / CH;
    ko[x] = (uint32_t)((rr * (uint32_t)p.k_st + 8 * ((lane % CH) ^ da_swz_k<D>(rr))) * 2);
    vo[x] = (uint32_t)((rr * (uint32_t)p.v_st + 8 * ((lane % CH) ^ da_swz_v<D>(rr))) * 2);
  }
  auto dma = [&](const uint16_t *bh, int64_t st, const uint32_t (&off)[NX], int kb, int slot) __attribute__((always_inline)) {
    const uint16_t *base = da_scalar(bh + (int64_t)kb * DA_BS * st);
    const int last = tl.lk - 1 - kb * DA_BS;
    if (last >= DA_BS - 1) {
#pragma unroll
      for (int x = 0; x < NX; ++x)
        asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(off[x]), "s"(base),
                     "{m0}"(lds0 + 2 * (slot * BLK + (NW * x + w) * 512)) : "memory");
    } else {
#pragma unroll
      for (int x = 0; x < NX; ++x) {
        const int past = max(RP * (NW * x + w) + lane / CH - last, 0);  // rows back to the last key
        asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(off[x] - past * (uint32_t)st * 2u), "s"(base),
                     "{m0}"(lds0 + 2 * (slot * BLK + (NW * x + w) * 512)) : "memory");
      }
    }
  };
  auto dma_k = [&](int kb) __attribute__((always_inline)) { dma(kbh, p.k_st, ko, kb, (kb - j0) & 1); };
  auto dma_v = [&](int kb) __attribute__((always_inline)) { dma(vbh, p.v_st, vo, kb, 2); };
  if (j0 < j1) {  // (the first tile is on its way while q is loaded)
    dma_k(j0);
    dma_v(j0);
  }

  x8 qf[NS];  // B operand: dims 16 s + 8 hf ..
  {
    const elem *qp = (const elem *)p.q + (p.s.cu_q ? (tl.q0 + t) * p.q_st : tl.b * p.q_sb + t * p.q_st) +
                     h * p.q_sh + 8 * hf;
#pragma unroll
    for (int s = 0; s < NS; ++s) qf[s] = *(const x8 *)(qp + 16 * s);
  }
#pragma unroll
  for (int s = 0; s < NS; ++s) settle(qf[s]);

  float m = da_ninf(), thr = da_ninf(), l = 0.f, nmu = 0.f;
  f32x16 acc[ND];
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[dt][i] = 0.f;

  // Byte offsets of this lane's first reads of a slot.  Swizzles only flip the chunk bits,
  // so the other reads are these with bits flipped (done anew for every tile: the
  // registers are worth more).
  //   K: row r32, chunk hf of each pair s
  //   V^T: 16-lane group c of the wave points at rows k0 + i / 4 and reads columns 32 dt +
  //   16 (c % 2) + (its lane) of four keys
  const uint32_t k_at = 2 * (r32 * D + 8 * (hf ^ da_swz_k<D>(r32)));
  const int v_row = 4 * hf + ((lane & 15) >> 2);
  const uint32_t v_at = 2 * (2 * BLK + v_row * D + 8 * ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ da_swz_v<D>(v_row)) +
                             4 * (lane & 1));
  const char *lds = (const char *)smem;
  // scores of tile j; register i of a half holds key 8 (i / 4) + 4 hf + i % 4
  auto scores = [&](int j, f32x16 (&st)[2]) __attribute__((always_inline)) {
    const uint32_t at = k_at + 2 * ((j - j0) & 1) * BLK;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
      for (int i = 0; i < 16; ++i) st[kt][i] = 0.f;
    }
#pragma unroll
    for (int s = 0; s < NS; ++s) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)  // (row r32 + 32 has the same swizzle)
        st[kt] = T::mfma(*(const x8 *)(lds + (at ^ (32 * s)) + 64 * kt * D), qf[s], st[kt]);
    }
  };
  auto largest = [&](const f32x16 (&st)[2]) __attribute__((always_inline)) -> float {
    float mx = fmaxf(st[0][0], st[0][1]);
#pragma unroll
    for (int i = 2; i < 16; i += 2) mx = fmaxf(fmaxf(mx, st[0][i]), st[0][i + 1]);
#pragma unroll
    for (int i = 0; i < 16; i += 2) mx = fmaxf(fmaxf(mx, st[1][i]), st[1][i + 1]);
    return mx;
  };
  // masks tile j where it has to be, and raises the reference maximum only past its
  // headroom (T::GAP); both halves of a row keep the same one
  auto settle_max = [&](int j, f32x16 (&st)[2], float mx) __attribute__((always_inline)) {
    if (j * DA_BS + DA_BS - 1 > lim_lo) {
      const int d = lim - j * DA_BS - 4 * hf;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          st[kt][i] = 32 * kt + 8 * (i >> 2) + (i & 3) <= d ? st[kt][i] : da_ninf();
      mx = largest(st);
    }
    if (__ballot(mx > thr) != 0) {
      const float mn = fmaxf(m, pair32_max(mx)), to = da_ref<T>(mn, p.qscale);
      const float alpha = m == da_ninf() ? 0.f : fast_exp2(to - nmu);  // (both as rounded in the weights)
      m = mn;
      thr = mn + p.thr_gap;
      nmu = to;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[dt][i] *= alpha;
    }
  };
  // weights of half kt of a tile, and their product with V.  The half's weights are added
  // among themselves first: over 32768 keys one long chain of additions loses more than
  // all other roundings of the log-sum.
  auto weigh = [&](f32x16 &st, x8 (&pw)[2]) __attribute__((always_inline)) {
    float part[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      st[i] = fast_exp2(__builtin_fmaf(st[i], p.qscale, nmu));
      part[i & 1] = i < 2 ? st[i] : part[i & 1] + st[i];
      pw[i >> 3][i & 7] = (elem)st[i];
    }
    l += part[0] + part[1];
  };
  auto values = [&](int j, int kt, const x8 (&pw)[2]) __attribute__((always_inline)) {
    const uint32_t at = v_at;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) {
        const char *v = lds + (at ^ (64 * dt)) + 2 * (32 * kt + 16 * ks) * D;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)v);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(v + 16 * D));
        acc[dt] = T::mfma(__builtin_bit_cast(x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)), pw[ks], acc[dt]);
      }
    }
  };

  const int jw = wave_live && lim_hi >= 0 ? min(lim_hi / DA_BS, j1 - 1) : -1;  // this wave's last tile
  for (int j = j0; j < j1; ++j) {
    wait_vmcnt<0>();
    lds_barrier();  // K of tile j has landed for every wave, tile j - 1 is read
    if (j > j0) dma_v(j);
    if (j + 1 < j1) dma_k(j + 1);
    f32x16 st[2];
    x8 pw[2];
    if (j <= jw) {
      scores(j, st);
      settle_max(j, st, largest(st));
      weigh(st[0], pw);
    }
    if (j + 1 < j1) wait_vmcnt<NX>();
    else wait_vmcnt<0>();
    lds_barrier();  // V of tile j has landed
    if (j <= jw) {
      values(j, 0, pw);
      weigh(st[1], pw);
      values(j, 1, pw);
    }
  }
  if (!wave_live) return;
  l = pair32_sum(l);
  // results that are not finite (with scores that are not numbers, l is not, and the row stands)
  float sum = 0.f;
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) sum = __builtin_fmaf(acc[dt][i], 0.f, sum);
  const uint64_t bad = __ballot(sum != 0.f && l < __int_as_float(0x7f800000));  // (sum: NaN)
  // register i of dim tile dt holds dim 32 dt + 8 (i / 4) + 4 hf + i % 4
  if (live && p.splits > 1) {
    const int64_t pi = da_part_at(p, tl, t, h, split);
    if (hf == 0) {
      p.ws_ml[2 * pi] = m == da_ninf() ? m : -nmu;
      p.ws_ml[2 * pi + 1] = l;
    }
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(float4 *)(p.ws_acc + pi * D + 32 * dt + 8 * i + 4 * hf) =
            float4{acc[dt][4 * i], acc[dt][4 * i + 1], acc[dt][4 * i + 2], acc[dt][4 * i + 3]};
  } else if (live) {
    const bool none = l == 0.f;  // no key seen
    const float inv = none ? 0.f : 1.f / l;
    const int64_t o = da_out_at(p, tl, t, h);
    if (p.out_dt == LA_F32) {
#pragma unroll
      for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *(float4 *)((float *)p.out + o + 32 * dt + 8 * i + 4 * hf) =
              float4{acc[dt][4 * i] * inv, acc[dt][4 * i + 1] * inv, acc[dt][4 * i + 2] * inv, acc[dt][4 * i + 3] * inv};
    } else {  // the halves of a row trade fours, so that a lane stores eight values
      typedef elem x4 __attribute__((ext_vector_type(4)));
#pragma unroll
      for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          uint2 y[2];
#pragma unroll
          for (int x = 0; x < 2; ++x)
            y[x] = __builtin_bit_cast(uint2, x4{(elem)(acc[dt][4 * (i + x)] * inv), (elem)(acc[dt][4 * (i + x) + 1] * inv),
                                                (elem)(acc[dt][4 * (i + x) + 2] * inv), (elem)(acc[dt][4 * (i + x) + 3] * inv)});
          const auto a = __builtin_amdgcn_permlane32_swap(y[0].x, y[1].x, false, false);
          const auto c = __builtin_amdgcn_permlane32_swap(y[0].y, y[1].y, false, false);
          *(uint4 *)((elem *)p.out + o + 32 * dt + 8 * (i + hf)) = uint4{a[0], c[0], a[1], c[1]};
        }
    }
    if (p.lse && hf == 0) p.lse[da_lse_at(p, tl, t, h)] = none ? da_ninf() : (__log2f(l) - nmu) * DA_LN2;  // (as rounded in the weights)
  }
  if (bad != 0)
    da_again<T, D, 32, false>(p, tl, kvh, split, r_first, (uint32_t)(bad | (bad >> 32)) & (uint32_t)__ballot(live),
                                 j0 * DA_BS, min(j1, lim_hi / DA_BS + 1) * DA_BS, 0, 1);
}

// fp32 rows: four waves of 16 rows on 16x16x4 products, all of it fp32.  A staged tile is
// 32 keys; lane (c, i) = (lane / 16, lane % 16) reads 16-byte chunk 4 s + c of K row i,
// whose four values feed four products (dims 16 s + 4 c + e), and holds P of row i for
// keys 4 c + e, which the product over V takes in that order.  Bound by the fp32 matrix
// rate: 8192 tokens of 32 heads on 8 take 4.33 ms at D = 128, 127 TFLOP/s (a large fp32
// product 154); four prompts of 202 tokens together 8.5 us, dependent loads.
template <int D>
__global__ __launch_bounds__(256, 2) void dense_attn_f32_kernel(DaKP p) {
  constexpr int NW = 4, R = 16 * NW, BS = 32, BLK = BS * D, CH = D / 4, RP = 64 / CH, NX = BS / RP / NW;
  constexpr int NS = D / 16;
  __shared__ __align__(16) float smem[4 * BLK];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane >> 4, ri = lane & 15;
  uint32_t stream, tix;
  da_stream(blockIdx.x, (uint32_t)p.Hkv * p.splits, stream, tix);
  const int kvh = (int)(stream / (uint32_t)p.splits), split = (int)(stream % (uint32_t)p.splits);
  const DaTile tl = da_uniform(da_tile(p.s, (int)tix, p.ntile, R, false));
  const int G = p.s.G;
  if (tl.b < 0 || tl.r0 + R > tl.lq * G) da_rest<D>(p, tl, R, kvh, split, (int)tix, w, NW);
  if (tl.b < 0 || tl.r0 >= tl.lq * G) return;

  const int nrow = tl.lq * G, diag = tl.lk - tl.lq;
  auto limit = [&](int t) { return p.causal ? diag + t : tl.lk - 1; };
  const int r_first = tl.r0 + 16 * w;
  const int r_mine = min(r_first + ri, nrow - 1);
  const bool live = r_first + ri < nrow, wave_live = r_first < nrow;
  const int t = r_mine / G, h = kvh * G + r_mine % G;
  const int lim = limit(t);
  const int lim_lo = __builtin_amdgcn_readfirstlane(limit(min(r_first, nrow - 1) / G));
  const int lim_hi = __builtin_amdgcn_readfirstlane(limit(min(r_first + 15, nrow - 1) / G));
  const int lim_tile = __builtin_amdgcn_readfirstlane(limit((min(tl.r0 + R, nrow) - 1) / G));
  const int n_all = lim_tile < 0 ? 0 : lim_tile / BS + 1;
  int j0 = 0, j1 = n_all;
  if (p.splits > 1) {
    j0 = (int)((int64_t)n_all * split / p.splits);
    j1 = (int)((int64_t)n_all * (split + 1) / p.splits);
  }
  j0 = __builtin_amdgcn_readfirstlane(j0);
  j1 = __builtin_amdgcn_readfirstlane(j1);

  f32x4 qf[NS];
  {
    const float *qp = (const float *)p.q + (p.s.cu_q ? (tl.q0 + t) * p.q_st : tl.b * p.q_sb + t * p.q_st) +
                      h * p.q_sh + 4 * c;
#pragma unroll
    for (int s = 0; s < NS; ++s) qf[s] = *(const f32x4 *)(qp + 16 * s);
  }
  const float *kbh = (const float *)p.k + (p.s.cu_q ? tl.k0 * p.k_st : tl.b * p.k_sb) + kvh * p.k_sh;
  const float *vbh = (const float *)p.v + (p.s.cu_q ? tl.k0 * p.v_st : tl.b * p.v_sb) + kvh * p.v_sh;
  auto swz_k = [](int r) { return 2 * (r & 7); };
  auto swz_v = [](int r) { return 4 * ((r >> 2) & 3); };
  auto dma = [&](int kb, int slot) {
#pragma unroll
    for (int x = 0; x < NX; ++x) {
      const int u = NW * x + w, rr = RP * u + lane / CH;
      const int64_t key = min(kb * BS + rr, tl.lk - 1);
      dma16(kbh + key * p.k_st + 4 * ((lane % CH) ^ swz_k(rr)), smem + slot * BLK + u * 256);
      dma16(vbh + key * p.v_st + 4 * ((lane % CH) ^ swz_v(rr)), smem + (2 + slot) * BLK + u * 256);
    }
  };

  float m = da_ninf(), thr = da_ninf(), l = 0.f, nmu = 0.f;
  // acc of 16 tiles at a time is added to total: one long chain of products' sums, four
  // keys a step, would round as often as there are steps
  f32x4 acc[NS], total[NS];
#pragma unroll
  for (int dt = 0; dt < NS; ++dt) acc[dt] = total[dt] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (j0 < j1) dma(j0, 0);
  for (int j = j0; j < j1; ++j) {
    const int par = (j - j0) & 1;
    wait_vmcnt<0>();
    lds_barrier();
    if (j + 1 < j1) dma(j + 1, par ^ 1);
    if (!wave_live || j * BS > lim_hi) continue;
    const float *sk = smem + par * BLK, *sv = smem + (2 + par) * BLK;
    f32x4 st[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      st[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
      const int kr = 16 * kt + ri;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const f32x4 a = *(const f32x4 *)&sk[kr * D + 4 * ((4 * s + c) ^ swz_k(kr))];
#pragma unroll
        for (int e = 0; e < 4; ++e) st[kt] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], qf[s][e], st[kt], 0, 0, 0);
      }
    }
    // register e of a tile holds key 4 c + e
    if (j * BS + BS - 1 > lim_lo) {
      const int d = lim - j * BS - 4 * c;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) st[kt][e] = 16 * kt + e <= d ? st[kt][e] : da_ninf();
    }
    float mx = da_ninf();
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = fmaxf(mx, st[kt][e]);
    if (__ballot(mx > thr) != 0) {
      const float mn = fmaxf(m, pair32_max(pair16_max(mx))), to = da_ref<DaF32>(mn, p.qscale);
      const float alpha = m == da_ninf() ? 0.f : fast_exp2(to - nmu);
      m = mn;
      thr = mn + p.thr_gap;
      nmu = to;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < NS; ++dt) {
        acc[dt] *= alpha;
        total[dt] *= alpha;
      }
    }
    float part = 0.f;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float pr = fast_exp2(__builtin_fmaf(st[kt][e], p.qscale, nmu));
        part += pr;
        const int kr = 16 * kt + 4 * c + e;
#pragma unroll
        for (int dt = 0; dt < NS; ++dt)
          acc[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(
              sv[kr * D + 4 * ((4 * dt + (ri >> 2)) ^ swz_v(kr)) + (ri & 3)], pr, acc[dt], 0, 0, 0);
      }
    l += part;
    if ((j - j0) % 16 == 15) {
#pragma unroll
      for (int dt = 0; dt < NS; ++dt) {
        total[dt] += acc[dt];
        acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
  }
  if (!wave_live) return;
#pragma unroll
  for (int dt = 0; dt < NS; ++dt) acc[dt] += total[dt];
  l = pair32_sum(pair16_sum(l));
  float sum = 0.f;
#pragma unroll
  for (int dt = 0; dt < NS; ++dt)
#pragma unroll
    for (int e = 0; e < 4; ++e) sum = __builtin_fmaf(acc[dt][e], 0.f, sum);
  uint64_t bad = __ballot(sum != 0.f && l < __int_as_float(0x7f800000));
  // register e of dim tile dt holds dim 16 dt + 4 c + e
  if (live && p.splits > 1) {
    const int64_t pi = da_part_at(p, tl, t, h, split);
    if (c == 0) {
      p.ws_ml[2 * pi] = m == da_ninf() ? m : -nmu;
      p.ws_ml[2 * pi + 1] = l;
    }
#pragma unroll
    for (int dt = 0; dt < NS; ++dt)
      *(float4 *)(p.ws_acc + pi * D + 16 * dt + 4 * c) = float4{acc[dt][0], acc[dt][1], acc[dt][2], acc[dt][3]};
  } else if (live) {
    const bool none = l == 0.f;
    const float inv = none ? 0.f : 1.f / l;
    const int64_t o = da_out_at(p, tl, t, h) + 4 * c;
#pragma unroll
    for (int dt = 0; dt < NS; ++dt)
      da_store4(p.out, o + 16 * dt, p.out_dt, acc[dt][0] * inv, acc[dt][1] * inv, acc[dt][2] * inv, acc[dt][3] * inv);
    if (p.lse && c == 0) p.lse[da_lse_at(p, tl, t, h)] = none ? da_ninf() : (__log2f(l) - nmu) * DA_LN2;
  }
  if (bad != 0) {
    bad |= bad >> 32;
    da_again<DaF32, D, 16, false>(p, tl, kvh, split, r_first, (uint32_t)((bad | (bad >> 16)) & __ballot(live) & 0xffffu),
                                  j0 * BS, min(j1, lim_hi / BS + 1) * BS, 0, 1);
  }
}

// At most 16 rows a sequence and KV head (decode steps): the four waves of a workgroup
// take rounds of keys in turn (few_rows.h) and join in LDS.  Bound by the reads: one token
// over sixteen caches of 4278 to 12345 keys (469 MB), 93 us with the join, 5.0 TB/s; over
// one cache of 16384 keys 20 us, half of it launches and dependent loads.
template <class T, int D>
__global__ __launch_bounds__(256, 2) void dense_few_kernel(DaKP p) {
  typedef FewRows<T, D, false> FR;
  typedef typename FR::elem elem;
  constexpr int NW = 4;
  constexpr int LDS_MERGE = NW * (FR::VALS + 32) * 4;
  constexpr int LDS = NW * FR::LDS_BYTES > LDS_MERGE ? NW * FR::LDS_BYTES : LDS_MERGE;
  __shared__ __align__(16) char smem[LDS];
  __shared__ uint32_t s_bad;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t stream, split_u;
  da_stream(blockIdx.x, (uint32_t)(p.Hkv * p.s.B), stream, split_u);
  const int kvh = (int)(stream % (uint32_t)p.Hkv), split = (int)split_u, G = p.s.G;
  DaTile tl{};
  tl.b = (int32_t)(stream / (uint32_t)p.Hkv);
  da_seq(p.s, tl);
  tl = da_uniform(tl);
  const int R = (int)p.s.Tq * G, nrow = tl.lq * G;
  if (nrow < R) da_rest<D>(p, tl, R, kvh, split, 0, w, NW);
  if (nrow == 0) return;
  const int diag = tl.lk - tl.lq;
  auto limit = [&](int t) { return p.causal ? diag + t : tl.lk - 1; };
  const int row = min(lane & 15, nrow - 1), t = row / G;
  const int last = __builtin_amdgcn_readfirstlane(limit(tl.lq - 1));  // the last key any row sees
  const int rounds = last < 0 ? 0 : last / FR::RK + 1;
  const int r0 = (int)((int64_t)rounds * split / p.splits), r1 = (int)((int64_t)rounds * (split + 1) / p.splits);
  const elem *kb = (const elem *)p.k + tl.b * p.k_sb + kvh * p.k_sh, *vb = (const elem *)p.v + tl.b * p.v_sb + kvh * p.v_sh;
  if (threadIdx.x == 0) s_bad = 0u;
  FR fr;
  fr.begin((const elem *)p.q + tl.b * p.q_sb + t * p.q_st + (kvh * G + row % G) * p.q_sh);
  fr.walk(r0 + w, NW, r1, tl.lk, limit(t), p.qscale, (elem *)(smem + w * FR::LDS_BYTES),
          [&](int key) { return kb + key * p.k_st; }, [&](int key) { return vb + key * p.v_st; }, [](int, f32x4) {});
  __syncthreads();
  float *ml = (float *)smem, *vals = ml + NW * 32;
  fr.put(ml + w * 32, vals + w * FR::VALS);
  __syncthreads();
  for (int e = threadIdx.x; e < nrow * D; e += 256) {
    const int g = e / D, d = e % D, te = g / G, h = kvh * G + g % G;
    float m = da_ninf();
#pragma unroll
    for (int x = 0; x < NW; ++x) m = fmaxf(m, ml[x * 32 + 2 * g]);
    float l = 0.f, a = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const float f = fast_exp2(ml[x * 32 + 2 * g] - (m == da_ninf() ? 0.f : m));
      l = __builtin_fmaf(ml[x * 32 + 2 * g + 1], f, l);
      a = __builtin_fmaf(vals[x * FR::VALS + g * (D + 4) + d], f, a);
    }
    // (with scores that are not numbers, l is not, and the row stands)
    if (!(fabsf(a) < __int_as_float(0x7f800000)) && l > 0.f && l < __int_as_float(0x7f800000)) atomicOr(&s_bad, 1u << g);
    if (l == 0.f) a = 0.f;  // (no key seen)
    if (p.splits > 1) {
      const int64_t pi = da_part_at(p, tl, te, h, split);
      p.ws_acc[pi * D + d] = a;
      if (d == 0) {
        p.ws_ml[2 * pi] = m;
        p.ws_ml[2 * pi + 1] = l;
      }
    } else {
      da_store1(p.out, da_out_at(p, tl, te, h) + d, p.out_dt, l == 0.f ? 0.f : a / l);
      if (p.lse && d == 0) p.lse[da_lse_at(p, tl, te, h)] = l == 0.f ? da_ninf() : (m + __log2f(l)) * DA_LN2;
    }
  }
  __syncthreads();
  if (s_bad == 0u) return;
  uint32_t *marks = (uint32_t *)smem;  // (of which all is read)
  if (threadIdx.x < D) marks[threadIdx.x] = 0u;
  wait_vmcnt<0>();
  __syncthreads();  // (every wave's stores are done, which those below replace)
  if (!p.causal || tl.lq == 1) {  // (every row sees every key)
    few_marks<elem, D, NW>(marks, [&](int key) { return vb + key * p.v_st; }, r0 * FR::RK, min(tl.lk, r1 * FR::RK));
    __syncthreads();
    for (int e = threadIdx.x; e < nrow * D; e += 256) {
      const int g = e / D, d = e % D, te = g / G, h = kvh * G + g % G;
      if (!((s_bad >> g) & 1u) || marks[d] == 0u) continue;
      if (p.splits > 1) p.ws_acc[da_part_at(p, tl, te, h, split) * D + d] = few_mark(marks[d]);
      else da_store1(p.out, da_out_at(p, tl, te, h) + d, p.out_dt, few_mark(marks[d]));
    }
    return;
  }
  da_again<T, D, 16, true>(p, tl, kvh, split, 0, s_bad, r0 * FR::RK, r1 * FR::RK, w, NW);
}

// Joins the parts of a row: a wave a row (4-6 us, its launch).
template <int D>
__global__ __launch_bounds__(256) void dense_combine_kernel(DaKP p, int64_t rows) {
  constexpr int N = D / 64;
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int h = (int)(row % p.Hq);
  const int64_t qr = row / p.Hq;
  int64_t o, lo;
  if (p.s.cu_q) {
    if (qr < da_cu(p.s.cu_q, 0, p.s.Tq) || qr >= da_cu(p.s.cu_q, p.s.B, p.s.Tq)) return;
    o = qr * p.o_st + h * p.o_sh;
    lo = qr + h * p.l_sh;
  } else {
    const int64_t b = qr / p.s.Tq, t = qr % p.s.Tq;
    if (p.s.q_len && t >= p.s.q_len[b]) return;  // (zeros, by the tiles)
    o = b * p.o_sb + t * p.o_st + h * p.o_sh;
    lo = b * p.l_sb + t + h * p.l_sh;
  }
  // a lane a part (at most 64)
  const float2 ml = lane < p.splits ? ((const float2 *)p.ws_ml)[row * p.splits + lane] : float2{da_ninf(), 0.f};
  float m = ml.x;
#pragma unroll
  for (int o2 = 32; o2 >= 1; o2 >>= 1) m = fmaxf(m, __shfl_xor(m, o2, 64));
  const bool empty = ml.x == da_ninf() && ml.y == 0.f;
  const float f = empty ? 0.f : fast_exp2(ml.x - (m == da_ninf() ? 0.f : m));
  const float l = group_sum<64>(empty ? 0.f : ml.y * f);
  float acc[N];
#pragma unroll
  for (int x = 0; x < N; ++x) acc[x] = 0.f;
  const float *a = p.ws_acc + row * p.splits * D + lane * N;
  for (int i0 = 0; i0 < p.splits; i0 += 8) {
    float v[8][N];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int x = 0; x < N; ++x) v[i][x] = a[(int64_t)min(i0 + i, p.splits - 1) * D + x];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float fi = __shfl(i0 + i < p.splits ? f : 0.f, (i0 + i) & 63, 64);
#pragma unroll
      for (int x = 0; x < N; ++x) acc[x] = __builtin_fmaf(i0 + i < p.splits ? v[i][x] : 0.f, fi, acc[x]);
    }
  }
  const bool none = l == 0.f;
  const float inv = none ? 0.f : 1.f / l;
#pragma unroll
  for (int x = 0; x < N; ++x) da_store1(p.out, o + lane * N + x, p.out_dt, acc[x] * inv);
  if (p.lse && lane == 0) p.lse[lo] = none ? da_ninf() : (m + __log2f(l)) * DA_LN2;
}

// ------------------------------------------------------------------ host ----
struct DaPlan {
  bool few = false;     // dense_few_kernel
  int rows = 128;       // of a workgroup
  int64_t ntile = 0, splits = 1;
  size_t ml = 0, bytes = 0;
};

static DaPlan da_plan(const la_dense_attn_args *a) {
  DaPlan pl;
  const bool packed = a->cu_q != nullptr, f32 = a->dtype == LA_F32;
  const int64_t G = a->Hq / a->Hkv;
  pl.few = !packed && a->Tq * G <= 16;
  pl.rows = pl.few ? 16 : f32 ? 64 : 128;
  pl.ntile = pl.few ? a->B : da_tiles(packed, a->B, a->Tq, G, pl.rows);
  // parts of at least four staged tiles, two workgroups a CU (few rows: four, since the
  // sequences' lengths differ; more rows: chunks of 512 queries over caches of 2781 to 8192
  // keys take 233 us whole and 282 in two parts each)
  const int64_t wgs = pl.ntile * a->Hkv, keys = packed ? ceil_div(a->Tk, a->B) : a->Tk;
  const int64_t want = (int64_t)(pl.few ? 4 : 2) * num_cus() / std::max<int64_t>(1, wgs);
  pl.splits = std::max<int64_t>(1, std::min<int64_t>({want, keys / (4 * DA_BS), 64}));
  if (pl.splits > 1) {
    const int64_t parts = (packed ? 1 : a->B) * a->Tq * a->Hq * pl.splits;
    pl.ml = ((size_t)parts * 2 * sizeof(float) + 255) / 256 * 256;
    pl.bytes = pl.ml + (size_t)parts * a->D * sizeof(float);
  }
  return pl;
}

static int da_check(const la_dense_attn_args *a) {
  LA_REQUIRE(a != nullptr, "la_dense_attention: null args");
  LA_REQUIRE(a->B > 0 && a->Hq > 0 && a->Hkv > 0 && a->Tq >= 0 && a->Tk >= 0, "la_dense_attention: sizes must be positive");
  LA_REQUIRE(a->Hq % a->Hkv == 0, "la_dense_attention: Hq must be a multiple of Hkv");
  LA_REQUIRE(a->D == 64 || a->D == 128, "la_dense_attention: head_dim %lld (64 or 128)", (long long)a->D);
  LA_REQUIRE(a->dtype == LA_F32 || a->dtype == LA_BF16 || a->dtype == LA_F16, "la_dense_attention: dtype");
  LA_REQUIRE(a->out_dtype == a->dtype || a->out_dtype == LA_F32, "la_dense_attention: out_dtype is dtype or fp32");
  LA_REQUIRE(a->scale > 0.f && a->scale < 1e30f, "la_dense_attention: scale must be positive");
  LA_REQUIRE(a->B < ((int64_t)1 << 24) && a->Tk < ((int64_t)1 << 30) && a->Tq * (a->Hq / a->Hkv) < ((int64_t)1 << 30),
             "la_dense_attention: sizes past 2^30 rows");
  LA_REQUIRE(a->cu_q || !a->cu_k, "la_dense_attention: cu_k without cu_q");
  LA_REQUIRE(!(a->cu_q && (a->q_len || a->k_len)), "la_dense_attention: lengths are for batched calls");
  return LA_OK;
}

static int da_rows_ok(const char *what, const void *p, int64_t esz, int64_t sb, int64_t sh, int64_t st, int64_t heads,
                      int64_t rows) {
  const int64_t n = 16 / esz;
  if (heads == 1) sh = 0;
  if (rows == 1) st = 0;
  LA_REQUIRE(p != nullptr, "la_dense_attention: null %s", what);
  LA_REQUIRE((uintptr_t)p % 16 == 0 && sb % n == 0 && sh % n == 0 && st % n == 0,
             "la_dense_attention: rows of %s must be 16-byte aligned", what);
  return LA_OK;
}

template <class K>
static int da_launch(K kernel, int64_t wgs, int threads, const DaKP &p, hipStream_t st) {
  kernel<<<dim3((uint32_t)wgs), dim3(threads), 0, st>>>(p);
  LA_LAUNCHED();
  return LA_OK;
}

}  // namespace la

extern "C" size_t la_dense_attention_workspace(const la_dense_attn_args *a) {
  if (la::da_check(a) != LA_OK || a->Tq == 0) return 0;
  return la::da_plan(a).bytes;
}

extern "C" int la_dense_attention(const la_dense_attn_args *a, void *stream) {
  using namespace la;
  if (int rc = da_check(a)) return rc;
  if (a->Tq == 0) return LA_OK;
  const int64_t esz = a->dtype == LA_F32 ? 4 : 2;
  const int64_t osz = a->out_dtype == LA_F32 ? 4 : 2;
  const bool packed = a->cu_q != nullptr;
  auto sb = [&](int64_t s) { return packed || a->B == 1 ? 0 : s; };
  if (int rc = da_rows_ok("q", a->q, esz, sb(a->q_sb), a->q_sh, a->q_st, a->Hq, a->Tq)) return rc;
  if (a->Tk > 0) {
    if (int rc = da_rows_ok("k", a->k, esz, sb(a->k_sb), a->k_sh, a->k_st, a->Hkv, a->Tk)) return rc;
    LA_REQUIRE(a->Tk == 1 || (a->k_st >= 0 && a->v_st >= 0 && a->k_st < (1 << 24) && a->v_st < (1 << 24)),
               "la_dense_attention: key rows 2^24 values apart or more");
    if (int rc = da_rows_ok("v", a->v, esz, sb(a->v_sb), a->v_sh, a->v_st, a->Hkv, a->Tk)) return rc;
  }
  if (int rc = da_rows_ok("out", a->out, osz, sb(a->o_sb), a->o_sh, a->o_st, a->Hq, a->Tq)) return rc;
  const int64_t nb = packed ? 1 : a->B;
  auto cover = [&](const void *x, int64_t es, int64_t b, int64_t h, int64_t t, int64_t heads, int64_t rows) {
    return Cover(x, a->D * es, {b * es, nb}, {h * es, heads}, {t * es, rows});
  };
  const Cover out = cover(a->out, osz, a->o_sb, a->o_sh, a->o_st, a->Hq, a->Tq);
  LA_REQUIRE(!overlap(out, cover(a->q, esz, a->q_sb, a->q_sh, a->q_st, a->Hq, a->Tq)) &&
                 !overlap(out, cover(a->k, esz, a->k_sb, a->k_sh, a->k_st, a->Hkv, a->Tk)) &&
                 !overlap(out, cover(a->v, esz, a->v_sb, a->v_sh, a->v_st, a->Hkv, a->Tk)),
             "la_dense_attention: out shares memory with an input");
  const DaPlan pl = da_plan(a);
  if (pl.bytes > 0 && (!a->workspace || a->ws_bytes < (int64_t)pl.bytes))
    return fail(LA_ERR_WORKSPACE, "la_dense_attention: workspace %lld < %lld bytes", (long long)a->ws_bytes,
                (long long)pl.bytes);
  LA_REQUIRE((uintptr_t)a->workspace % 256 == 0 || pl.bytes == 0, "la_dense_attention: workspace alignment");
  const int64_t wgs = pl.ntile * a->Hkv * pl.splits;
  LA_REQUIRE(grid_fits(wgs, 256), "la_dense_attention: too many rows");
  DaKP p{};
  p.s = DaSeqs{a->cu_q, a->cu_k, a->q_len, a->k_len, a->Tq, a->Tk, (int32_t)a->B, (int32_t)(a->Hq / a->Hkv)};
  p.q = a->q; p.k = a->k; p.v = a->v; p.out = a->out; p.lse = a->lse;
  p.ws_ml = (float *)a->workspace;
  p.ws_acc = (float *)((char *)a->workspace + pl.ml);
  p.q_sb = a->q_sb; p.q_sh = a->q_sh; p.q_st = a->q_st;
  p.k_sb = a->k_sb; p.k_sh = a->k_sh; p.k_st = a->k_st;
  p.v_sb = a->v_sb; p.v_sh = a->v_sh; p.v_st = a->v_st;
  p.o_sb = a->o_sb; p.o_sh = a->o_sh; p.o_st = a->o_st;
  p.l_sb = a->l_sb; p.l_sh = a->l_sh;
  p.Hq = (int32_t)a->Hq; p.Hkv = (int32_t)a->Hkv;
  p.ntile = (int32_t)pl.ntile; p.splits = (int32_t)pl.splits;
  p.causal = a->causal != 0; p.out_dt = a->out_dtype; p.zero_rest = a->zero_rest != 0;
  p.qscale = a->scale * 1.44269504088896340736f;
  p.thr_gap = std::min((a->dtype == LA_F16 ? DaF16::GAP : DaBf16::GAP) / p.qscale, 3e38f);  // (finite: -inf + it stays)
  hipStream_t st = (hipStream_t)stream;
  int rc;
  const bool d128 = a->D == 128;
  if (pl.few) {
    if (a->dtype == LA_F32)
      rc = d128 ? da_launch(dense_few_kernel<DaF32, 128>, wgs, 256, p, st) : da_launch(dense_few_kernel<DaF32, 64>, wgs, 256, p, st);
    else if (a->dtype == LA_BF16)
      rc = d128 ? da_launch(dense_few_kernel<DaBf16, 128>, wgs, 256, p, st) : da_launch(dense_few_kernel<DaBf16, 64>, wgs, 256, p, st);
    else
      rc = d128 ? da_launch(dense_few_kernel<DaF16, 128>, wgs, 256, p, st) : da_launch(dense_few_kernel<DaF16, 64>, wgs, 256, p, st);
  } else if (a->dtype == LA_F32) {
    rc = d128 ? da_launch(dense_attn_f32_kernel<128>, wgs, 256, p, st) : da_launch(dense_attn_f32_kernel<64>, wgs, 256, p, st);
  } else if (a->dtype == LA_BF16) {
    rc = d128 ? da_launch(dense_attn_kernel<DaBf16, 128, 4>, wgs, 256, p, st) : da_launch(dense_attn_kernel<DaBf16, 64, 4>, wgs, 256, p, st);
  } else {
    rc = d128 ? da_launch(dense_attn_kernel<DaF16, 128, 4>, wgs, 256, p, st) : da_launch(dense_attn_kernel<DaF16, 64, 4>, wgs, 256, p, st);
  }
  if (rc != LA_OK || pl.splits == 1) return rc;
  const int64_t rows = (packed ? 1 : a->B) * a->Tq * a->Hq;
  const dim3 grid((uint32_t)ceil_div(rows, 4));
  if (a->D == 128) dense_combine_kernel<128><<<grid, 256, 0, st>>>(p, rows);
  else dense_combine_kernel<64><<<grid, 256, 0, st>>>(p, rows);
  LA_LAUNCHED();
  return LA_OK;
}
