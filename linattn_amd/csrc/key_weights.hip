// The attention weight each key gathers (la_key_weights): column sums of the softmax
// whose rows' log sums la_dense_attention returned.
//
// A workgroup takes a tile of keys of one KV head and keeps them in registers; it walks
// the rows (query, head of the group) that see them, staged in LDS: S^T = K Q^T on the
// matrix cores, P = exp2(c S - lse) in place, added lane by lane (a lane holds one row
// and 16 keys of a product), and summed over the lanes every 32 staged tiles.  Nothing is
// normalised or joined on the way, so the rows of a tile can be split over workgroups;
// their sums are added in order by a second kernel: no atomics.
#include <algorithm>

#include "dense_attn.h"

namespace la {

struct KwKP {
  DaSeqs s;
  const void *q, *k;
  const float *lse;
  float *out, *ws;  // ws: [split][what out has, densely]
  int64_t q_sb, q_sh, q_st, k_sb, k_sh, k_st, l_sb, l_sh, w_sb, w_sh, last, ws_split;
  int32_t Hq, Hkv, ntile, splits, causal, accumulate, zero_rest;
  int32_t ms;  // log2 of the heads in a staged tile of rows
  float qscale;
};

// A tile's keys, and the staged tiles of rows it walks: 2^ms heads by RT / 2^ms queries
// each, from query t0 on, a group of heads after the other.
struct KwTile {
  DaTile t;       // sequence (q0, k0, lq, lk as given), b < 0: none
  int32_t s0;     // first key
  int32_t t0, n;  // first query; this split's staged tiles
  int32_t tb, g;  // query and head of the group that the first of them begins with
};

template <int KT, int RT>
__device__ __forceinline__ KwTile kw_tile(const KwKP &p, int tix, int split) {
  KwTile x;
  x.t = da_uniform(da_tile(p.s, tix, p.ntile, KT, true));
  x.s0 = x.t0 = x.n = x.tb = x.g = 0;
  if (x.t.b < 0) return x;
  // da_tile's first tiles are the sequences' last; the first keys are seen by most rows
  const int32_t n = p.s.cu_q ? x.t.lk : (int32_t)p.s.Tk;
  x.s0 = ((n + KT - 1) / KT) * KT - KT - x.t.r0;
  if (x.s0 >= x.t.lk) return x;
  x.t0 = p.last > 0 ? (int32_t)max((int64_t)x.t.lq - p.last, (int64_t)0) : 0;
  if (p.causal) x.t0 = max(x.t0, x.s0 - (x.t.lk - x.t.lq));
  const int qpt = RT >> p.ms;
  const uint32_t ntq = (uint32_t)(max(x.t.lq - x.t0, 0) + qpt - 1) / (uint32_t)qpt;
  const uint32_t all = ntq * (uint32_t)(p.s.G >> p.ms), per = (all + p.splits - 1) / p.splits;
  const uint32_t i0 = min(per * split, all), i1 = min(i0 + per, all);
  x.n = __builtin_amdgcn_readfirstlane(i1 - i0);
  x.t0 = __builtin_amdgcn_readfirstlane(x.t0);
  if (x.n == 0) return x;
  x.g = __builtin_amdgcn_readfirstlane((i0 / ntq) << p.ms);
  x.tb = __builtin_amdgcn_readfirstlane(x.t0 + (int)(i0 % ntq) * qpt);
  return x;
}

// Where key s of the tile goes, and whether it is written here.
template <class F>
__device__ __forceinline__ void kw_put(const KwKP &p, const KwTile &x, int kvh, int split, int s, F value) {
  const int64_t n = p.s.cu_q ? x.t.lk : p.s.Tk;
  if (s >= n) return;
  const float v = s < x.t.lk ? value() : 0.f;
  const int64_t row = (p.s.cu_q ? x.t.k0 : 0) + s;
  if (p.splits > 1) {
    p.ws[split * p.ws_split + ((int64_t)(p.s.cu_q ? 0 : x.t.b) * p.Hkv + kvh) * p.s.Tk + row] = v;
    return;
  }
  float *o = p.out + (p.s.cu_q ? 0 : x.t.b * p.w_sb) + kvh * p.w_sh + row;
  *o = p.accumulate ? *o + v : v;
}

// Packed keys of no sequence, by the workgroups that got no tile.
__device__ __forceinline__ void kw_rest(const KwKP &p, const KwTile &x, int kvh, int split, int tix) {
  if (!p.zero_rest || split != 0 || x.t.b >= 0 || !p.s.cu_q) return;
  const int32_t *ck = p.s.cu_k ? p.s.cu_k : p.s.cu_q;
  const int64_t first = da_cu(ck, 0, p.s.Tk), last = max(first, (int64_t)da_cu(ck, p.s.B, p.s.Tk));
  const int64_t n = first + p.s.Tk - last;
  for (int64_t i = (int64_t)(tix - x.t.r0) * blockDim.x + threadIdx.x; i < n;
       i += (int64_t)(p.ntile - x.t.r0) * blockDim.x)
    p.out[kvh * p.w_sh + (i < first ? i : i + last - first)] = 0.f;
}

// The next staged tile of queries tb .. and heads g ..
__device__ __forceinline__ void kw_next(const KwKP &p, const KwTile &x, int qpt, int &tb, int &g) {
  tb += qpt;
  if (tb >= x.t.lq) {
    tb = x.t0;
    g += 1 << p.ms;
  }
}

// Staged tiles after which a tile's running sums are added to its totals: over 128 000 rows
// a chain of additions a lane loses five times what the weights' own roundings do.
constexpr int KW_RUN = 32;

// bf16 / fp16: four waves of 64 keys.  Rows are staged 64 at a time by LDS-DMA, with their
// lse (each wave its own copy, so that every wave counts the same loads), NSLOT - 1 tiles
// ahead.  14567 tokens of 32 heads on 8 run at 0.95 PFLOP/s as one sequence, and as twelve
// of 115 to 3039 at 0.8 (162 to 166 us): there the vector unit (fma, exp and add of each
// weight) is busy for 52 % of the cycles, the matrix unit for 35, and waves wait for the
// staged tiles that their own keys skip (the diagonal) and for one another.  For few
// queries it is latency, the keys having to arrive before a workgroup's first product: the
// last 64 queries of 50001 tokens, 105 MB, take 51 to 54 us, vector unit 35 %, matrix 18.  (Two waves of 64 keys a
// workgroup: 254 and 86 us, the copies' instructions double; eight: 191 and 68, nothing runs
// beside a workgroup's loads; three workgroups a CU without the interleaving: 249 and 60.)
template <class T, int D>
__global__ __launch_bounds__(256, 2) void key_weights_kernel(KwKP p) {
  constexpr int NW = 4, KT = 64 * NW, BLK = DA_BS * D, CH = D / 8, RP = 64 / CH, NX = DA_BS / RP / NW;
  constexpr int NS = D / 16, NSLOT = 4;
  typedef typename T::x8 x8;
  typedef typename T::elem elem;
  __shared__ __align__(16) uint16_t smem[NSLOT * BLK];
  __shared__ float s_lse[NSLOT][NW][DA_BS];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hf = lane >> 5, r32 = lane & 31, G = p.s.G;
  uint32_t stream, tix;
  da_stream(blockIdx.x, (uint32_t)p.Hkv * p.splits, stream, tix);
  const int kvh = (int)(stream / (uint32_t)p.splits), split = (int)(stream % (uint32_t)p.splits);
  const KwTile x = kw_tile<KT, DA_BS>(p, (int)tix, split);
  kw_rest(p, x, kvh, split, (int)tix);
  if (x.t.b < 0) return;

  const int s_w = x.s0 + 64 * w;  // this wave's keys
  const int diag = x.t.lk - x.t.lq;
  f32x16 acc[2];
#pragma unroll
  for (int kt = 0; kt < 2; ++kt)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[kt][i] = 0.f;

  // What acc gathered added to total, and acc begun again: sums over the 32 lanes of a
  // half, each step adding two registers' halves of the lanes into one register, until
  // lane l has register l / 2.
  float total[2] = {0.f, 0.f};
  auto fold_in = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const auto y = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[kt][i]), __float_as_uint(acc[kt][i + 8]), false, false);
        v[i] = __uint_as_float(y[0]) + __uint_as_float(y[1]);
      }
      auto fold = [&](float lo, float hi, bool up, auto other) { return (up ? hi : lo) + other(up ? lo : hi); };
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = fold(v[i], v[i + 4], lane & 8, [](float y) { return dpp_f32<0x128>(y); });
#pragma unroll
      for (int i = 0; i < 2; ++i) v[i] = fold(v[i], v[i + 2], lane & 4, [](float y) { return dpp_f32<0x141>(y); });
      v[0] = fold(v[0], v[1], lane & 2, [](float y) { return dpp_f32<0x1B>(y); });
      total[kt] += v[0] + dpp_f32<0xB1>(v[0]);
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[kt][i] = 0.f;
    }
  };

  const int n = x.n, qs = 6 - p.ms, qpt = 1 << qs;
  if (n > 0) {
    const elem *qbh = (const elem *)p.q + (p.s.cu_q ? x.t.q0 * p.q_st : x.t.b * p.q_sb) + kvh * G * p.q_sh;
    const float *lbh = p.lse + (p.s.cu_q ? x.t.q0 : x.t.b * p.l_sb) + kvh * G * p.l_sh;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void_t *)smem);
    const uint32_t ldl0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void_t *)s_lse);
    // what this lane copies of a staged tile, from a scalar base: of q, rows RP (NW i + w) +
    // lane / CH, and one row's lse; queries past the last are copies of it
    uint32_t qo[NX];
#pragma unroll
    for (int i = 0; i < NX; ++i) {
      const int rr = RP * (NW * i + w) + lane / CH;
      qo[i] = 2u * (uint32_t)((rr & (qpt - 1)) * p.q_st + (rr >> qs) * p.q_sh + 8 * ((lane % CH) ^ da_swz_k<D>(rr)));
    }
    const uint32_t lo = 4u * (uint32_t)((lane & (qpt - 1)) + (lane >> qs) * p.l_sh);
    int d_tb = x.tb, d_g = x.g;
    auto dma = [&](int slot) __attribute__((always_inline)) {  // the next tile
      const elem *qb = da_scalar(qbh + d_tb * p.q_st + d_g * p.q_sh);
      const float *lb = da_scalar(lbh + d_tb + d_g * p.l_sh);
      const int last = x.t.lq - 1 - d_tb;
      if (last >= qpt - 1) {
#pragma unroll
        for (int i = 0; i < NX; ++i)
          asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(qo[i]), "s"(qb),
                       "{m0}"(lds0 + 2 * (slot * BLK + (NW * i + w) * 512)) : "memory");
        asm volatile("global_load_lds_dword %0, %1" ::"v"(lo), "s"(lb),
                     "{m0}"(ldl0 + 4 * ((slot * NW + w) * DA_BS)) : "memory");
      } else {
#pragma unroll
        for (int i = 0; i < NX; ++i) {
          const int past = max(((RP * (NW * i + w) + lane / CH) & (qpt - 1)) - last, 0);
          asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(qo[i] - past * (uint32_t)p.q_st * 2u), "s"(qb),
                       "{m0}"(lds0 + 2 * (slot * BLK + (NW * i + w) * 512)) : "memory");
        }
        asm volatile("global_load_lds_dword %0, %1" ::"v"(lo - 4u * (uint32_t)max((lane & (qpt - 1)) - last, 0)), "s"(lb),
                     "{m0}"(ldl0 + 4 * ((slot * NW + w) * DA_BS)) : "memory");
      }
      kw_next(p, x, qpt, d_tb, d_g);
    };
    x8 kf[2][NS];  // A operand: key 32 kt + r32, dims 16 s + 8 hf ..
    const elem *kbh = (const elem *)p.k + (p.s.cu_q ? x.t.k0 * p.k_st : x.t.b * p.k_sb) + kvh * p.k_sh;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const int64_t key = min(s_w + 32 * kt + r32, x.t.lk - 1);
#pragma unroll
      for (int s = 0; s < NS; ++s) kf[kt][s] = *(const x8 *)(kbh + key * p.k_st + 16 * s + 8 * hf);
    }
    for (int j = 0; j < NSLOT - 1; ++j) {
      if (j < n) dma(j);
    }
    // queries from these on see any, and all, of the wave's keys
    const int t_any = p.causal ? s_w - diag : 0;
    const int t_all = p.causal ? s_w + 63 - diag : s_w + 63 < x.t.lk ? 0 : INT32_MAX;
    int tb = x.tb, g = x.g;
    // products of a half of the staged rows; -lse of its rows in log2 units (-inf: adds nothing)
    auto products = [&](int j, int h, f32x16 (&st)[2]) __attribute__((always_inline)) -> float {
      const uint16_t *sq = smem + (j % NSLOT) * BLK;
      const int rl = 32 * h + r32, sw = da_swz_k<D>(rl);
      const float ls = s_lse[j % NSLOT][w][rl];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) st[kt][i] = 0.f;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const x8 qf = *(const x8 *)&sq[rl * D + 8 * ((2 * s + hf) ^ sw)];
        st[0] = T::mfma(kf[0][s], qf, st[0]);
        st[1] = T::mfma(kf[1][s], qf, st[1]);
      }
      return ls == __int_as_float(0xff800000) ? ls : -ls * 1.44269504088896340736f;
    };
    auto weigh = [&](const f32x16 (&st)[2], float nl) __attribute__((always_inline)) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[kt][i] += fast_exp2(__builtin_fmaf(st[kt][i], p.qscale, nl));
    };
    // a half's products while the half before is weighed: the matrix and the vector unit
    // take about as long, and a wave's own instructions must fill both
    auto interleave = [&]() __attribute__((always_inline)) {
      __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
      for (int i = 0; i < 2 * NS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 64 / (2 * NS), 0);
        __builtin_amdgcn_sched_group_barrier(0x400, 32 / (2 * NS), 0);
        if (i % 2) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
    };
    const float none = __int_as_float(0xff800000);
    f32x16 sa[2], sb[2];
    float nb = none;  // sb holds nothing yet
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) sb[kt][i] = 0.f;
    auto masked = [&](int j) __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float nl = products(j, h, sa);
        const int t = tb + ((32 * h + r32) & (qpt - 1));
        const bool out = t >= x.t.lq || s_lse[j % NSLOT][w][32 * h + r32] == none;
        const int seen = out ? -1 : p.causal ? diag + t : x.t.lk - 1;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          // register i: key 8 (i / 4) + 4 hf + i % 4
          const int d = seen - (s_w + 32 * kt + 4 * hf);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float e = fast_exp2(__builtin_fmaf(sa[kt][i], p.qscale, nl));
            acc[kt][i] += 8 * (i >> 2) + (i & 3) <= d ? e : 0.f;
          }
        }
      }
    };
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int s = 0; s < NS; ++s) settle(kf[kt][s]);  // (here, not in the loop, where it would wait for all tiles)
    constexpr int PER = NX + 1;  // loads of a tile
    for (int j = 0; j < n; ++j, kw_next(p, x, qpt, tb, g)) {
      // tile j has landed: the loads after it are those of the tiles ahead
      if (j + 2 < n) wait_vmcnt<2 * PER>();
      else if (j + 1 < n) wait_vmcnt<PER>();
      else wait_vmcnt<0>();
      // (a row with lse -inf adds nothing even where its scores are not numbers; the wave's own copy)
      const uint64_t absent = __ballot(s_lse[j % NSLOT][w][lane] == none);
      lds_barrier();  // for every wave, and tile j - 1 is read
      if (j + NSLOT - 1 < n) dma((j + NSLOT - 1) % NSLOT);
      if (j % KW_RUN == KW_RUN - 1) fold_in();
      if (tb + qpt <= t_any) continue;
      const bool whole = t_all <= tb && tb + qpt <= x.t.lq && absent == 0;
      if (whole) {
        const float na = products(j, 0, sa);
        weigh(sb, nb);
        interleave();
        nb = products(j, 1, sb);
        weigh(sa, na);
        interleave();
      } else {
        masked(j);
      }
    }
    weigh(sb, nb);
    fold_in();
  }
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
    const int i = r32 >> 1;
    if ((lane & 1) == 0) kw_put(p, x, kvh, split, s_w + 32 * kt + 8 * (i >> 2) + 4 * hf + (i & 3), [&] { return total[kt]; });
  }
}

// fp32: four waves of 32 keys on 16x16x4 products; lane (c, i) holds chunk 4 s + c of key
// i, and of row i of the staged rows, as in dense_attn_f32_kernel.  Bound by the fp32 matrix
// rate: 8192 tokens of 32 heads on 8, D = 128, 2.5 ms, 110 TFLOP/s.
template <int D>
__global__ __launch_bounds__(256, 2) void key_weights_f32_kernel(KwKP p) {
  constexpr int NW = 4, KT = 32 * NW, BS = 32, BLK = BS * D, CH = D / 4, RP = 64 / CH, NX = BS / RP / NW;
  constexpr int NS = D / 16;
  __shared__ __align__(16) float smem[2 * BLK];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane >> 4, ri = lane & 15, G = p.s.G;
  uint32_t stream, tix;
  da_stream(blockIdx.x, (uint32_t)p.Hkv * p.splits, stream, tix);
  const int kvh = (int)(stream / (uint32_t)p.splits), split = (int)(stream % (uint32_t)p.splits);
  const KwTile x = kw_tile<KT, BS>(p, (int)tix, split);
  kw_rest(p, x, kvh, split, (int)tix);
  if (x.t.b < 0) return;
  const int s_w = x.s0 + 32 * w, diag = x.t.lk - x.t.lq;
  f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
  f32x4 total[2] = {acc[0], acc[1]};
  const int n = x.n, qs = 5 - p.ms, qpt = 1 << qs;
  if (n > 0) {
    f32x4 kf[2][NS];
    const float *kbh = (const float *)p.k + (p.s.cu_q ? x.t.k0 * p.k_st : x.t.b * p.k_sb) + kvh * p.k_sh;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const int64_t key = min(s_w + 16 * kt + ri, x.t.lk - 1);
#pragma unroll
      for (int s = 0; s < NS; ++s) kf[kt][s] = *(const f32x4 *)(kbh + key * p.k_st + 16 * s + 4 * c);
    }
    const float *qbh = (const float *)p.q + (p.s.cu_q ? x.t.q0 * p.q_st : x.t.b * p.q_sb) + kvh * G * p.q_sh;
    const float *lbh = p.lse + (p.s.cu_q ? x.t.q0 : x.t.b * p.l_sb) + kvh * G * p.l_sh;
    auto swz = [](int r) { return 2 * (r & 7); };
    int d_tb = x.tb, d_g = x.g, tb = x.tb, g = x.g;
    auto dma = [&](int slot) {  // the next tile
#pragma unroll
      for (int i = 0; i < NX; ++i) {
        const int u = NW * i + w, rr = RP * u + lane / CH;
        const int t = min(d_tb + (rr & (qpt - 1)), x.t.lq - 1);
        dma16(qbh + t * p.q_st + (d_g + (rr >> qs)) * p.q_sh + 4 * ((lane % CH) ^ swz(rr)), smem + slot * BLK + u * 256);
      }
      kw_next(p, x, qpt, d_tb, d_g);
    };
    dma(0);
    for (int j = 0; j < n; ++j, kw_next(p, x, qpt, tb, g)) {
      float nl[2];
      int seen[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int rr = 16 * h + ri, t = tb + (rr & (qpt - 1));
        nl[h] = lbh[min(t, x.t.lq - 1) + (g + (rr >> qs)) * p.l_sh];
        seen[h] = t >= x.t.lq ? -1 : p.causal ? diag + t : x.t.lk - 1;
      }
      wait_vmcnt<0>();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        settle(nl[h]);
        if (nl[h] == __int_as_float(0xff800000)) seen[h] = -1;
        else nl[h] *= -1.44269504088896340736f;
      }
      lds_barrier();
      if (j + 1 < n) dma((j + 1) & 1);
      if (j % KW_RUN == KW_RUN - 1) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          total[kt] += acc[kt];
          acc[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
      }
      const float *sq = smem + (j & 1) * BLK;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int rl = 16 * h + ri;
        f32x4 st[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          const f32x4 b = *(const f32x4 *)&sq[rl * D + 4 * ((4 * s + c) ^ swz(rl))];
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              st[kt] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[kt][s][e], b[e], st[kt], 0, 0, 0);
        }
        // register e: key 4 c + e
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          const int d = seen[h] - (s_w + 16 * kt + 4 * c);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float pr = fast_exp2(__builtin_fmaf(st[kt][e], p.qscale, nl[h]));
            acc[kt][e] += e <= d ? pr : 0.f;
          }
        }
      }
    }
  }
#pragma unroll
  for (int kt = 0; kt < 2; ++kt)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float v = group_sum<16>(total[kt][e] + acc[kt][e]);
      if (ri == e) kw_put(p, x, kvh, split, s_w + 16 * kt + 4 * c + e, [&] { return v; });
    }
}

// Adds the parts of a key in their order (5 us, its launch).  Packed keys of no sequence have no parts.
__global__ __launch_bounds__(256) void key_weights_sum_kernel(KwKP p) {
  const int64_t s = (int64_t)blockIdx.x * 256 + threadIdx.x, bh = blockIdx.y;
  if (s >= p.s.Tk) return;
  if (p.s.cu_q) {
    const int32_t *ck = p.s.cu_k ? p.s.cu_k : p.s.cu_q;
    if (s < da_cu(ck, 0, p.s.Tk) || s >= da_cu(ck, p.s.B, p.s.Tk)) return;
  }
  const float *part = p.ws + bh * p.s.Tk + s;
  float v = 0.f;
  for (int i = 0; i < p.splits; ++i) v += part[i * p.ws_split];
  float *o = p.out + (p.s.cu_q ? 0 : bh / p.Hkv * p.w_sb) + bh % p.Hkv * p.w_sh + s;
  *o = p.accumulate ? *o + v : v;
}

// ------------------------------------------------------------------ host ----
struct KwPlan {
  int keys = 256;
  int64_t ntile = 0, splits = 1;
  size_t bytes = 0;
};

static KwPlan kw_plan(const la_key_weights_args *a) {
  KwPlan pl;
  const bool packed = a->cu_q != nullptr;
  pl.keys = a->dtype == LA_F32 ? 128 : 256;
  pl.ntile = da_tiles(packed, a->B, a->Tk, 1, pl.keys);
  // Rows are split until there are four workgroups a CU (causal tiles differ in length by
  // far; 14567 packed tokens took 262 us unsplit, 167 with four, 180 with eight), down to
  // four staged tiles each.
  const int64_t wgs = pl.ntile * a->Hkv, G = a->Hq / a->Hkv;
  int64_t rows = (packed ? ceil_div(a->Tq, a->B) : a->Tq) * G;
  if (a->last > 0) rows = std::min(rows, a->last * G);
  pl.splits = std::max<int64_t>(1, std::min<int64_t>({ceil_div((int64_t)4 * num_cus(), wgs), rows / 256, 64}));
  if (pl.splits > 1) pl.bytes = (size_t)((packed ? 1 : a->B) * a->Hkv * a->Tk * pl.splits) * sizeof(float);
  return pl;
}

static int kw_check(const la_key_weights_args *a) {
  LA_REQUIRE(a != nullptr, "la_key_weights: null args");
  LA_REQUIRE(a->B > 0 && a->Hq > 0 && a->Hkv > 0 && a->Tq >= 0 && a->Tk >= 0, "la_key_weights: sizes must be positive");
  LA_REQUIRE(a->Hq % a->Hkv == 0, "la_key_weights: Hq must be a multiple of Hkv");
  LA_REQUIRE(a->D == 64 || a->D == 128, "la_key_weights: head_dim %lld (64 or 128)", (long long)a->D);
  LA_REQUIRE(a->dtype == LA_F32 || a->dtype == LA_BF16 || a->dtype == LA_F16, "la_key_weights: dtype");
  LA_REQUIRE(a->scale > 0.f && a->scale < 1e30f, "la_key_weights: scale must be positive");
  LA_REQUIRE(a->last >= 0, "la_key_weights: last must not be negative");
  LA_REQUIRE(a->B < ((int64_t)1 << 24) && a->Tk < ((int64_t)1 << 30) && a->Tq * (a->Hq / a->Hkv) < ((int64_t)1 << 30),
             "la_key_weights: sizes past 2^30 rows");
  LA_REQUIRE(a->cu_q || !a->cu_k, "la_key_weights: cu_k without cu_q");
  LA_REQUIRE(!(a->cu_q && (a->q_len || a->k_len)), "la_key_weights: lengths are for batched calls");
  return LA_OK;
}

}  // namespace la

extern "C" size_t la_key_weights_workspace(const la_key_weights_args *a) {
  if (la::kw_check(a) != LA_OK || a->Tk == 0) return 0;
  return la::kw_plan(a).bytes;
}

extern "C" int la_key_weights(const la_key_weights_args *a, void *stream) {
  using namespace la;
  if (int rc = kw_check(a)) return rc;
  if (a->Tk == 0) return LA_OK;
  const int64_t n16 = a->dtype == LA_F32 ? 4 : 8;
  const bool packed = a->cu_q != nullptr;
  LA_REQUIRE(a->k && a->out && ((a->q && a->lse) || a->Tq == 0), "la_key_weights: null pointer");
  auto ok = [&](const void *x, int64_t sb, int64_t sh, int64_t st, int64_t heads, int64_t rows) {
    return (uintptr_t)x % 16 == 0 && (packed || a->B == 1 || sb % n16 == 0) && (heads == 1 || sh % n16 == 0) &&
           (rows == 1 || st % n16 == 0);
  };
  LA_REQUIRE(ok(a->k, a->k_sb, a->k_sh, a->k_st, a->Hkv, a->Tk) &&
                 (a->Tq == 0 || ok(a->q, a->q_sb, a->q_sh, a->q_st, a->Hq, a->Tq)),
             "la_key_weights: rows of q and k must be 16-byte aligned");
  LA_REQUIRE(a->Tq <= 1 || (a->q_st >= 0 && a->q_st < (1 << 24)), "la_key_weights: query rows 2^24 values apart or more");
  const int64_t nb = packed ? 1 : a->B, es = a->dtype == LA_F32 ? 4 : 2;
  const Cover out(a->out, 4 * a->Tk, {4 * a->w_sb, nb}, {4 * a->w_sh, a->Hkv});
  LA_REQUIRE(!overlap(out, Cover(a->q, a->D * es, {es * a->q_sb, nb}, {es * a->q_sh, a->Hq}, {es * a->q_st, a->Tq})) &&
                 !overlap(out, Cover(a->k, a->D * es, {es * a->k_sb, nb}, {es * a->k_sh, a->Hkv}, {es * a->k_st, a->Tk})) &&
                 !overlap(out, Cover(a->lse, 4 * a->Tq, {4 * a->l_sb, nb}, {4 * a->l_sh, a->Hq})),
             "la_key_weights: out shares memory with an input");
  const KwPlan pl = kw_plan(a);
  if (pl.bytes > 0 && (!a->workspace || a->ws_bytes < (int64_t)pl.bytes))
    return fail(LA_ERR_WORKSPACE, "la_key_weights: workspace %lld < %lld bytes", (long long)a->ws_bytes,
                (long long)pl.bytes);
  const int64_t wgs = pl.ntile * a->Hkv * pl.splits;
  const int64_t bh = (packed ? 1 : a->B) * a->Hkv;
  // (rows are only split, and key_weights_sum_kernel's gridDim.y only bh, of fewer workgroups)
  LA_REQUIRE(grid_fits(wgs, 256) && (pl.splits == 1 || bh < 65536), "la_key_weights: too many keys or heads");
  KwKP p{};
  p.s = DaSeqs{a->cu_q, a->cu_k, a->q_len, a->k_len, a->Tq, a->Tk, (int32_t)a->B, (int32_t)(a->Hq / a->Hkv)};
  p.q = a->q; p.k = a->k; p.lse = a->lse; p.out = a->out; p.ws = (float *)a->workspace;
  p.q_sb = a->q_sb; p.q_sh = a->q_sh; p.q_st = a->q_st;
  p.k_sb = a->k_sb; p.k_sh = a->k_sh; p.k_st = a->k_st;
  p.l_sb = a->l_sb; p.l_sh = a->l_sh; p.w_sb = a->w_sb; p.w_sh = a->w_sh;
  p.last = a->last; p.ws_split = bh * a->Tk;
  p.Hq = (int32_t)a->Hq; p.Hkv = (int32_t)a->Hkv;
  p.ntile = (int32_t)pl.ntile; p.splits = (int32_t)pl.splits;
  p.causal = a->causal != 0; p.accumulate = a->accumulate != 0; p.zero_rest = a->zero_rest != 0 && !a->accumulate;
  p.qscale = a->scale * 1.44269504088896340736f;
  // up to four heads a staged tile, so that short or causal ranges of queries fill it; where
  // the heads are too far apart for 32-bit offsets, one
  auto fits = [&](int64_t m) {
    return p.s.G % m == 0 && a->q_sh >= 0 && (64 / m - 1) * a->q_st + (m - 1) * a->q_sh < ((int64_t)1 << 30) &&
           a->l_sh >= 0 && (m - 1) * a->l_sh < ((int64_t)1 << 28);
  };
  p.ms = fits(4) ? 2 : fits(2) ? 1 : 0;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((uint32_t)wgs);
  if (a->dtype == LA_F32) {
    if (a->D == 128) key_weights_f32_kernel<128><<<grid, 256, 0, st>>>(p);
    else key_weights_f32_kernel<64><<<grid, 256, 0, st>>>(p);
  } else if (a->dtype == LA_BF16) {
    if (a->D == 128) key_weights_kernel<DaBf16, 128><<<grid, 256, 0, st>>>(p);
    else key_weights_kernel<DaBf16, 64><<<grid, 256, 0, st>>>(p);
  } else {
    if (a->D == 128) key_weights_kernel<DaF16, 128><<<grid, 256, 0, st>>>(p);
    else key_weights_kernel<DaF16, 64><<<grid, 256, 0, st>>>(p);
  }
  LA_LAUNCHED();
  if (pl.splits > 1) {
    key_weights_sum_kernel<<<dim3((uint32_t)ceil_div(a->Tk, 256), (uint32_t)bh), 256, 0, st>>>(p);
    LA_LAUNCHED();
  }
  return LA_OK;
}
