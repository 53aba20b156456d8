// Dense attention of new tokens over a paged cache (la_paged_attention): chunks of prompts and
// single tokens, in one call, over caches in the inputs' type or in fp8.  The attention of
// core.py:148-181 where the reference's cache is one contiguous tensor.
//
// S^T = K Q^T, P = exp2(c S - m), O^T += V^T P^T over staged blocks of keys with the running
// maximum and sum of a softmax (as in dense_attn.hip); rows, the sharing of the work and the
// parts of rows: paged_attn.h.
#include <algorithm>

#include "paged_attn.h"

namespace la {

constexpr float PA_LN2 = 0.69314718055994530942f;

__device__ __forceinline__ float pa_ninf() { return __int_as_float(0xff800000); }

// One value of K or V of the cache, as the definition has it.
template <class E, bool KV8>
struct PaCache {
  const void *pool;
  const float *scale;
  int64_t s_stride;
  int D;
  __device__ __forceinline__ float at(uint32_t row, int d) const {
    if constexpr (KV8) return fp8x2_to_f32<false>(((const uint8_t *)pool)[(uint64_t)row * D + d]).x * scale[row * s_stride];
    else return (float)((const E *)pool)[(uint64_t)row * D + d];
  }
};

// A part of a row: where it is kept until the parts are joined.
__device__ __forceinline__ int64_t pa_part(const PaKP &p, int wg, bool last) { return ((int64_t)wg * 2 + (last ? 1 : 0)) * p.part_rows; }

// Rows r_first + i of which bit i of `bad` is set, whose results are not finite: those with an
// infinity or NaN of V among what their blocks (keys a .. end - 1) held and they do not see are done
// again, key by key, in fp32; the others stand, but in fp16, where a weight below 2^-40 of the
// row's largest is 0 and its product with an infinity NaN: a dim's first keys with NaN and either
// infinity say what it is for each row.  (What a block holds past the last key is that key again.)
template <class E, int D, int NR, bool KV8, bool LOST>
__device__ void pa_again(const PaKP &p, int b, const PaSeq &sq, int kvh, int64_t part, int r_tile, int r_first, uint32_t bad, int a, int end) {
  const int lane = threadIdx.x & 63, G = p.G;
  const int32_t *pages = p.page_table + b * p.pt_sb;
  const PaCache<E, KV8> K{p.k, p.k_scale, p.s_stride, D}, V{p.v, p.v_scale, p.s_stride, D};
  auto row = [&](int key) { return pa_row(p, pages, min(key, sq.lk - 1), kvh); };
  constexpr int N = D / 64;
  const float inf = __int_as_float(0x7f800000);
  int32_t at[3][N];  // of dim lane + 64 x
#pragma unroll
  for (int x = 0; x < N; ++x) at[0][x] = at[1][x] = at[2][x] = INT32_MAX;
  if constexpr (LOST) {
    const int e = min(end, sq.lk);
    for (int key = a; key < e; ++key) {
      const uint32_t kr = row(key);
#pragma unroll
      for (int x = 0; x < N; ++x) {
        const float v = V.at(kr, lane + 64 * x);
        at[0][x] = min(at[0][x], v != v ? key : INT32_MAX);
        at[1][x] = min(at[1][x], v == inf ? key : INT32_MAX);
        at[2][x] = min(at[2][x], v == -inf ? key : INT32_MAX);
      }
    }
  }
  wait_vmcnt<0>();  // (stores over those)
#pragma unroll 1
  for (int i = 0; i < NR; ++i) {
    if (!((bad >> i) & 1u)) continue;
    const int r = r_first + i, t = r / G, h = kvh * G + r % G;
    const int lim = p.causal ? min(sq.lk - 1, sq.lk - sq.lq + t) : sq.lk - 1;
    bool met = false;
    for (int key = max(max(lim + 1, a), 0); key < end; ++key)
      for (int d = lane; d < D; d += 64) met = met || !(fabsf(V.at(row(key), d)) < inf);
    if (__ballot(met) == 0) {
#pragma unroll
      for (int x = 0; x < N; ++x) {
        const bool up = at[1][x] <= lim, down = at[2][x] <= lim, nan = at[0][x] <= lim || (up && down);
        if (!nan && !up && !down) continue;
        const float y = nan ? __int_as_float(0x7fc00000) : up ? inf : -inf;
        if (part >= 0) p.ws_acc[(part + r - r_tile) * D + lane + 64 * x] = y;
        else store_from_f32(p.out, pa_out_at(p, b, sq, t, h) + lane + 64 * x, p.out_dt, y);
      }
      continue;
    }
    const E *q = (const E *)p.q + pa_q_at(p, b, sq, t, h);
    const int e = min(end, lim + 1);
    float m = pa_ninf(), l = 0.f, acc[N];
#pragma unroll
    for (int x = 0; x < N; ++x) acc[x] = 0.f;
    for (int key0 = a; key0 < e; key0 += 64) {
      const uint32_t kr = row(min(key0 + lane, e - 1));
      float s = 0.f;
      for (int d = 0; d < D; ++d) s = __builtin_fmaf((float)q[d], K.at(kr, d), s);
      s = key0 + lane < e ? s * p.qscale : pa_ninf();
      float mx = s;
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
      const float mn = fmaxf(m, mx);
      const float alpha = m == pa_ninf() ? 0.f : fast_exp2(m - mn);
      const float pr = fast_exp2(s - (mn == pa_ninf() ? 0.f : mn));
      m = mn;
      l = l * alpha + group_sum<64>(pr);
#pragma unroll
      for (int x = 0; x < N; ++x) acc[x] *= alpha;
      const int n = min(64, e - key0);
      for (int j = 0; j < n; ++j) {
        const float w = __shfl(pr, j, 64);
        const uint32_t vr = __shfl((int)kr, j, 64);
#pragma unroll
        for (int x = 0; x < N; ++x) acc[x] = __builtin_fmaf(w, V.at(vr, lane + 64 * x), acc[x]);
      }
    }
    if (part >= 0) {
      const int64_t pi = part + r - r_tile;
      if (lane == 0) {
        p.ws_ml[2 * pi] = m;
        p.ws_ml[2 * pi + 1] = l;
      }
#pragma unroll
      for (int x = 0; x < N; ++x) p.ws_acc[pi * D + lane + 64 * x] = acc[x];
      continue;
    }
    const int64_t o = pa_out_at(p, b, sq, t, h);
#pragma unroll
    for (int x = 0; x < N; ++x) store_from_f32(p.out, o + lane + 64 * x, p.out_dt, l == 0.f ? 0.f : acc[x] / l);
    if (p.lse && lane == 0) p.lse[pa_lse_at(p, b, sq, t, h)] = l == 0.f ? pa_ninf() : (m + __log2f(l)) * PA_LN2;
  }
}

// What follows a piece: the next tile of the stretch, or the join's note of the tile that is left open.
struct PaWalk {
  PaStretch s;
  PaSeq seq;
  PaTiles tiles;
  int wg, w, kvh;
  template <int R>
  __device__ __forceinline__ bool begin(const PaKP &p) {
    wg = blockIdx.x;
    kvh = wg % p.Hkv;
    w = wg / p.Hkv;
    s = pa_stretch<R>(p, w);
    if (s.left == 0) {
      if (threadIdx.x == 0) p.ws_join[wg] = int4{0, 0, 0, 0};
      return false;
    }
    load<R>(p);
    return true;
  }
  template <int R>
  __device__ __forceinline__ void load(const PaKP &p) {
    seq = pa_seq(p, s.b);
    seq.lq = __builtin_amdgcn_readfirstlane(seq.lq);
    seq.lk = __builtin_amdgcn_readfirstlane(seq.lk);
    seq.q0 = pa_uniform(seq.q0);
    tiles = pa_tiles<R>(p, seq);
  }
  // (false: the stretch is done)
  template <int R>
  __device__ __forceinline__ bool next(const PaKP &p, int64_t cost, int64_t upto) {
    s.left -= upto - s.off;
    if (s.left <= 0) {
      const bool open = s.off == 0 && upto < cost;
      const int parts = open ? 1 + (int)((cost - upto + s.quota - 1) / s.quota) : 0;
      if (threadIdx.x == 0) p.ws_join[wg] = int4{s.b, s.i, parts, 0};
      return false;
    }
    s.off = 0;
    if (++s.i < tiles.n) return true;
    s.i = 0;
    do {
      ++s.b;
      load<R>(p);
    } while (tiles.n == 0 && s.b + 1 < p.B);
    return true;
  }
};

// bf16 / fp16 rows: four waves of 32 rows, three workgroups a CU, and the products and registers of
// dense_attn_kernel (S^T by 32x32x16 products leaves a lane 16 scores of one row; P goes into its
// product with V from the same registers, rounded to the inputs' type (bf16 with an fp8 cache);
// l is of the fp32 weights).
//
// A wave stages 16 keys of each block of 64.  Pages of whole sixteens (`EVEN`): these lie in one
// page, whose place for 64 blocks ahead is looked up at once, a lane a block, and the rows go
// global -> LDS from a scalar base.  Any other page size: a lane a key, four blocks ahead.  K is
// staged a block ahead into the other of two slots, V while its block is scored.
//
// fp8 caches (KV8) are loaded a block ahead into registers and widened on their way into LDS, once
// a workgroup (e4m3 is exact in bf16 and fp16); the scale of a key multiplies its scores, that of its
// value its weights, both in fp32.
template <class T, int D, bool KV8, bool EVEN>
__global__ __launch_bounds__(256, 3) void paged_attn_kernel(PaKP p) {
  typedef typename std::conditional<KV8, DaBf16, T>::type TP;  // of P and V
  constexpr int NW = 4, R = 32 * NW, BLK = DA_BS * D, CH = D / 8, RP = 64 / CH, NX = 16 / RP;
  constexpr int NS = D / 16, ND = D / 32, SPAN = EVEN ? 64 : 4;
  typedef typename T::x8 x8;
  typedef typename TP::x8 px8;
  typedef typename T::elem elem;
  typedef typename TP::elem pelem;
  __shared__ __align__(16) uint16_t smem[3 * BLK];  // K slots 0, 1, then V
  __shared__ __align__(16) float s_scale[KV8 ? 3 * DA_BS : 1];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hf = lane >> 5, r32 = lane & 31;
  const int G = p.G;
  PaWalk walk;
  pa_rest<D>(p, blockIdx.x % (uint32_t)p.Hkv);
  if (!walk.begin<R>(p)) return;
  const int kvh = walk.kvh;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void_t *)smem);
  // LDS-DMA: instruction x of wave w fills rows 16 w + RP x + lane / CH
  uint32_t ko[NX], vo[NX];
#pragma unroll
  for (int x = 0; x < NX; ++x) {
    const int rr = RP * x + lane / CH;
    ko[x] = (uint32_t)((rr * D + 8 * ((lane % CH) ^ da_swz_k<D>(16 * w + rr))) * 2);
    vo[x] = (uint32_t)((rr * D + 8 * ((lane % CH) ^ da_swz_v<D>(16 * w + rr))) * 2);
  }
  // Byte offsets of this lane's first reads of a slot (as in dense_attn_kernel).
  const uint32_t k_at = 2 * (r32 * D + 8 * (hf ^ da_swz_k<D>(r32)));
  const int v_row = 4 * hf + ((lane & 15) >> 2);
  const uint32_t v_at = 2 * (2 * BLK + v_row * D + 8 * ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ da_swz_v<D>(v_row)) +
                             4 * (lane & 1));
  const char *lds = (const char *)smem;

  while (true) {
    const PaSeq sq = walk.seq;
    const int b = walk.s.b, r0 = walk.s.i * R;
    const int nrow = sq.lq * G, diag = sq.lk - sq.lq;
    auto limit = [&](int t) { return p.causal ? diag + t : sq.lk - 1; };  // last key seen
    const int r_first = r0 + 32 * w;
    const int r_mine = min(r_first + r32, nrow - 1);
    const bool live = r_first + r32 < nrow, wave_live = r_first < nrow;
    const int t = r_mine / G, h = kvh * G + r_mine % G;
    const int lim = limit(t);
    const int lim_lo = __builtin_amdgcn_readfirstlane(limit(min(r_first, nrow - 1) / G));
    const int lim_hi = __builtin_amdgcn_readfirstlane(limit(min(r_first + 31, nrow - 1) / G));
    const int lim_tile = __builtin_amdgcn_readfirstlane(limit((min(r0 + R, nrow) - 1) / G));
    const int n_all = lim_tile < 0 ? 0 : lim_tile / DA_BS + 1;
    const int64_t cost = walk.tiles.cost(walk.s.i), upto = min(cost, walk.s.off + walk.s.left);
    const int j0 = __builtin_amdgcn_readfirstlane(pa_blocks(n_all, walk.s.off, cost));
    const int j1 = __builtin_amdgcn_readfirstlane(pa_blocks(n_all, upto, cost));
    const bool whole = walk.s.off == 0 && upto == cost;
    const int64_t part = whole ? -1 : pa_part(p, walk.wg, walk.s.off == 0);
    const int32_t *pages = p.page_table + b * p.pt_sb;

    // The cache's rows of this wave's keys: EVEN: of block jb + lane, the first of its sixteen;
    // else of block jb + lane / 16, key lane % 16 of them.
    uint32_t rows = 0;
    int jb = j0;
    auto look = [&](int j) __attribute__((always_inline)) {
      jb = j;
      const int key = EVEN ? (j + lane) * DA_BS + 16 * w : (j + lane / 16) * DA_BS + 16 * w + lane % 16;
      rows = pa_row(p, pages, min(key, sq.lk - 1), kvh);
    };
    // this lane's row for key `rr` of the wave's sixteen of block j
    auto row_of = [&](int j, int rr) __attribute__((always_inline)) -> uint32_t {
      if constexpr (EVEN) {
        const int past = sq.lk - 1 - min(j * DA_BS + 16 * w, sq.lk - 1);  // keys behind the first
        return (uint32_t)__builtin_amdgcn_readlane((int)rows, j - jb) + min(rr, past);
      } else {
        return (uint32_t)__shfl((int)rows, (j - jb) * 16 + rr, 64);
      }
    };
    auto dma = [&](const void *pool, const uint32_t (&off)[NX], int j, int slot) __attribute__((always_inline)) {
      if constexpr (EVEN) {
        const uint32_t row = (uint32_t)__builtin_amdgcn_readlane((int)rows, j - jb);
        const uint16_t *base = (const uint16_t *)pool + (uint64_t)row * D;
        const int last = sq.lk - 1 - min(j * DA_BS + 16 * w, sq.lk - 1);
        if (last >= 15) {
#pragma unroll
          for (int x = 0; x < NX; ++x)
            asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(off[x]), "s"(base),
                         "{m0}"(lds0 + 2 * (slot * BLK + 16 * w * D + x * 512)) : "memory");
        } else {
#pragma unroll
          for (int x = 0; x < NX; ++x) {
            const int past = max(RP * x + lane / CH - last, 0);  // rows back to the last key
            asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(off[x] - past * (uint32_t)(2 * D)), "s"(base),
                         "{m0}"(lds0 + 2 * (slot * BLK + 16 * w * D + x * 512)) : "memory");
          }
        }
      } else {
#pragma unroll
        for (int x = 0; x < NX; ++x) {
          const int rr = RP * x + lane / CH;
          const char *src = (const char *)pool + (uint64_t)row_of(j, rr) * (2 * D) + (off[x] - (uint32_t)(rr * 2 * D));
          asm volatile("global_load_lds_dwordx4 %0, off" ::"v"(src),
                       "{m0}"(lds0 + 2 * (slot * BLK + 16 * w * D + x * 512)) : "memory");
        }
      }
    };
    auto dma_k = [&](int j) __attribute__((always_inline)) { dma(p.k, ko, j, (j - j0) & 1); };
    auto dma_v = [&](int j) __attribute__((always_inline)) { dma(p.v, vo, j, 2); };

    // fp8: 16 codes a lane and load, and (lanes below 16) the keys' scales
    constexpr int N8 = D / 64, R8 = 64 / (D / 16);  // loads, rows of a load
    uint4 kr[N8], vr[N8];
    float ks = 0.f, vs = 0.f;
    auto fetch = [&](const void *pool, const float *scale, uint4 (&to)[N8], float &sc, int j) __attribute__((always_inline)) {
#pragma unroll
      for (int x = 0; x < N8; ++x)
        to[x] = *(const uint4 *)((const uint8_t *)pool + (uint64_t)row_of(j, R8 * x + lane / (D / 16)) * D + 16 * (lane % (D / 16)));
      sc = scale[row_of(j, lane & 15) * p.s_stride];
    };
    auto put = [&](const uint4 (&from)[N8], float sc, bool is_v, int slot) __attribute__((always_inline)) {
#pragma unroll
      for (int x = 0; x < N8; ++x) {
        const int row = 16 * w + R8 * x + lane / (D / 16), c = 2 * (lane % (D / 16));
        const int swz = is_v ? da_swz_v<D>(row) : da_swz_k<D>(row);
        const uint32_t word[4] = {from[x].x, from[x].y, from[x].z, from[x].w};
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          uint32_t u[4];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (is_v || std::is_same<T, DaBf16>::value) {
              u[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word[2 * y + i], 1.f, false));
              u[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word[2 * y + i], 1.f, true));
            } else {
              u[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word[2 * y + i], 1.f, false));
              u[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word[2 * y + i], 1.f, true));
            }
          }
          *(uint4 *)(smem + slot * BLK + row * D + 8 * ((c + y) ^ swz)) = uint4{u[0], u[1], u[2], u[3]};
        }
      }
      if (lane < 16) s_scale[(slot == 2 ? 2 : slot) * DA_BS + 16 * w + lane] = sc;
    };

    lds_barrier();  // (the piece before is read out of LDS)
    if (j0 < j1) {
      look(j0);
      if constexpr (KV8) {
        fetch(p.k, p.k_scale, kr, ks, j0);
        fetch(p.v, p.v_scale, vr, vs, j0);
        put(kr, ks, false, 0);
        if (j0 + 1 < j1) fetch(p.k, p.k_scale, kr, ks, j0 + 1);
      } else {
        settle(rows);
        dma_k(j0);
        dma_v(j0);
      }
    }
    x8 qf[NS];  // B operand: dims 16 s + 8 hf ..
    {
      const elem *qp = (const elem *)p.q + pa_q_at(p, b, sq, t, h) + 8 * hf;
#pragma unroll
      for (int s = 0; s < NS; ++s) qf[s] = *(const x8 *)(qp + 16 * s);
    }
#pragma unroll
    for (int s = 0; s < NS; ++s) settle(qf[s]);

    float m = pa_ninf(), thr = pa_ninf(), l = 0.f, nmu = 0.f;
    f32x16 acc[ND];
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[dt][i] = 0.f;

    // scores of block j; register i of a half holds key 8 (i / 4) + 4 hf + i % 4
    auto scores = [&](int j, f32x16 (&st)[2]) __attribute__((always_inline)) {
      const uint32_t at = k_at + 2 * ((j - j0) & 1) * BLK;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) st[kt][i] = 0.f;
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)  // (row r32 + 32 has the same swizzle)
          st[kt] = T::mfma(*(const x8 *)(lds + (at ^ (32 * s)) + 64 * kt * D), qf[s], st[kt]);
      if constexpr (KV8) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x4 sc = *(const f32x4 *)(s_scale + ((j - j0) & 1) * DA_BS + 32 * kt + 8 * g + 4 * hf);
#pragma unroll
            for (int i = 0; i < 4; ++i) st[kt][4 * g + i] *= sc[i];
          }
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
    // masks block j where it has to be, and raises the reference maximum only past its
    // headroom (GAP); both halves of a row keep the same one
    auto settle_max = [&](int j, f32x16 (&st)[2], float mx) __attribute__((always_inline)) {
      if (j * DA_BS + DA_BS - 1 > lim_lo) {
        const int d = lim - j * DA_BS - 4 * hf;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int i = 0; i < 16; ++i) st[kt][i] = 32 * kt + 8 * (i >> 2) + (i & 3) <= d ? st[kt][i] : pa_ninf();
        mx = largest(st);
      }
      if (__ballot(mx > thr) != 0) {
        const float mn = fmaxf(m, pair32_max(mx)), to = da_ref<TP>(mn, p.qscale);
        const float alpha = m == pa_ninf() ? 0.f : fast_exp2(to - nmu);  // (both as rounded in the weights)
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
    // weights of half kt of a block, added among themselves first
    auto weigh = [&](int kt, f32x16 &st, px8 (&pw)[2]) __attribute__((always_inline)) {
      float sum[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        st[i] = fast_exp2(__builtin_fmaf(st[i], p.qscale, nmu));
        sum[i & 1] = i < 2 ? st[i] : sum[i & 1] + st[i];
      }
      l += sum[0] + sum[1];
      if constexpr (!KV8) {
#pragma unroll
        for (int i = 0; i < 16; ++i) pw[i >> 3][i & 7] = (pelem)st[i];
      }
    };
    auto scaled = [&](int kt, const f32x16 &st, px8 (&pw)[2]) __attribute__((always_inline)) {  // (KV8)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 sc = *(const f32x4 *)(s_scale + 2 * DA_BS + 32 * kt + 8 * g + 4 * hf);
#pragma unroll
        for (int i = 0; i < 4; ++i) pw[g >> 1][4 * (g & 1) + i] = (pelem)(st[4 * g + i] * sc[i]);
      }
    };
    auto values = [&](int kt, const px8 (&pw)[2]) __attribute__((always_inline)) {
#pragma unroll
      for (int ks_ = 0; ks_ < 2; ++ks_)
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) {
          const char *v = lds + (v_at ^ (64 * dt)) + 2 * (32 * kt + 16 * ks_) * D;
          const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)v);
          const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(v + 16 * D));
          acc[dt] = TP::mfma(__builtin_bit_cast(px8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)), pw[ks_], acc[dt]);
        }
    };

    const int jw = wave_live && lim_hi >= 0 ? min(lim_hi / DA_BS, j1 - 1) : -1;  // this wave's last block
    for (int j = j0; j < j1; ++j) {
      if constexpr (KV8) {
        lds_barrier();  // K of block j is there for every wave, block j - 1 is read
        put(vr, vs, true, 2);
        if (j + 1 < j1) {
          put(kr, ks, false, (j + 1 - j0) & 1);
          fetch(p.v, p.v_scale, vr, vs, j + 1);
          if (j + 2 < j1) {
            if (j + 2 - jb == SPAN) look(j + 2);
            fetch(p.k, p.k_scale, kr, ks, j + 2);
          }
        }
      } else {
        wait_vmcnt<0>();
        lds_barrier();  // K of block j has landed for every wave, block j - 1 is read
        if (j > j0) dma_v(j);
        if (j + 1 < j1) {
          if (j + 1 - jb == SPAN) {
            look(j + 1);
            settle(rows);
          }
          dma_k(j + 1);
        }
      }
      f32x16 st[2];
      px8 pw[2];
      if (j <= jw) {
        scores(j, st);
        settle_max(j, st, largest(st));
        weigh(0, st[0], pw);
      }
      if constexpr (!KV8) {
        if (j + 1 < j1) wait_vmcnt<NX>();
        else wait_vmcnt<0>();
      }
      lds_barrier();  // V of block j has landed
      if (j <= jw) {
        if constexpr (KV8) scaled(0, st[0], pw);
        values(0, pw);
        weigh(1, st[1], pw);
        if constexpr (KV8) scaled(1, st[1], pw);
        values(1, pw);
      }
    }
    if (wave_live) {
      l = pair32_sum(l);
      // results that are not finite (with scores that are not numbers, l is not, and the row stands)
      float sum = 0.f;
#pragma unroll
      for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) sum = __builtin_fmaf(acc[dt][i], 0.f, sum);
      const uint64_t bad = __ballot(sum != 0.f && l < __int_as_float(0x7f800000));  // (sum: NaN)
      // register i of dim tile dt holds dim 32 dt + 8 (i / 4) + 4 hf + i % 4
      if (live && part >= 0) {
        const int64_t pi = part + r_mine - r0;
        if (hf == 0) {
          p.ws_ml[2 * pi] = m == pa_ninf() ? m : -nmu;
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
        const int64_t o = pa_out_at(p, b, sq, t, h);
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
        if (p.lse && hf == 0) p.lse[pa_lse_at(p, b, sq, t, h)] = none ? pa_ninf() : (__log2f(l) - nmu) * PA_LN2;  // (as rounded in the weights)
      }
      if (bad != 0)
        pa_again<elem, D, 32, KV8, (!KV8 && T::BIAS > 0.f)>(p, b, sq, kvh, part, r0, r_first, (uint32_t)(bad | (bad >> 32)) & (uint32_t)__ballot(live),
                                                           j0 * DA_BS, min(j1, lim_hi / DA_BS + 1) * DA_BS);
    }
    if (!walk.next<R>(p, cost, upto)) break;
  }
}

// fp32 rows: four waves of 16 rows on 16x16x4 products, blocks of 32 keys (dense_attn_f32_kernel's),
// over pages of any size, a lane a key, two blocks ahead.
template <int D>
__global__ __launch_bounds__(256, 2) void paged_attn_f32_kernel(PaKP p) {
  constexpr int NW = 4, R = 16 * NW, BS = 32, BLK = BS * D, CH = D / 4, RP = 64 / CH, NX = BS / RP / NW;
  constexpr int NS = D / 16;
  __shared__ __align__(16) float smem[4 * BLK];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane >> 4, ri = lane & 15;
  const int G = p.G;
  PaWalk walk;
  pa_rest<D>(p, blockIdx.x % (uint32_t)p.Hkv);
  if (!walk.begin<R>(p)) return;
  const int kvh = walk.kvh;
  auto swz_k = [](int r) { return 2 * (r & 7); };
  auto swz_v = [](int r) { return 4 * ((r >> 2) & 3); };
  while (true) {
    const PaSeq sq = walk.seq;
    const int b = walk.s.b, r0 = walk.s.i * R;
    const int nrow = sq.lq * G, diag = sq.lk - sq.lq;
    auto limit = [&](int t) { return p.causal ? diag + t : sq.lk - 1; };
    const int r_first = r0 + 16 * w;
    const int r_mine = min(r_first + ri, nrow - 1);
    const bool live = r_first + ri < nrow, wave_live = r_first < nrow;
    const int t = r_mine / G, h = kvh * G + r_mine % G;
    const int lim = limit(t);
    const int lim_lo = __builtin_amdgcn_readfirstlane(limit(min(r_first, nrow - 1) / G));
    const int lim_hi = __builtin_amdgcn_readfirstlane(limit(min(r_first + 15, nrow - 1) / G));
    const int lim_tile = __builtin_amdgcn_readfirstlane(limit((min(r0 + R, nrow) - 1) / G));
    const int n_all = lim_tile < 0 ? 0 : lim_tile / BS + 1;
    const int64_t cost = walk.tiles.cost(walk.s.i), upto = min(cost, walk.s.off + walk.s.left);
    const int j0 = __builtin_amdgcn_readfirstlane(pa_blocks(n_all, walk.s.off, cost));
    const int j1 = __builtin_amdgcn_readfirstlane(pa_blocks(n_all, upto, cost));
    const bool whole = walk.s.off == 0 && upto == cost;
    const int64_t part = whole ? -1 : pa_part(p, walk.wg, walk.s.off == 0);
    const int32_t *pages = p.page_table + b * p.pt_sb;
    // the cache's row of key lane % 32 of a block
    uint32_t rows = 0, rows_next = 0;
    auto look = [&](int j) -> uint32_t { return pa_row(p, pages, min(j * BS + (lane & 31), sq.lk - 1), kvh); };
    auto dma = [&](uint32_t at, int slot) {
#pragma unroll
      for (int x = 0; x < NX; ++x) {
        const int u = NW * x + w, rr = RP * u + lane / CH;
        const uint64_t row = (uint32_t)__shfl((int)at, rr, 64);
        dma16((const float *)p.k + row * D + 4 * ((lane % CH) ^ swz_k(rr)), smem + slot * BLK + u * 256);
        dma16((const float *)p.v + row * D + 4 * ((lane % CH) ^ swz_v(rr)), smem + (2 + slot) * BLK + u * 256);
      }
    };
    lds_barrier();
    if (j0 < j1) {
      rows = look(j0);
      rows_next = look(j0 + 1);
      settle(rows);
      settle(rows_next);
      dma(rows, 0);
    }
    f32x4 qf[NS];
    {
      const float *qp = (const float *)p.q + pa_q_at(p, b, sq, t, h) + 4 * c;
#pragma unroll
      for (int s = 0; s < NS; ++s) qf[s] = *(const f32x4 *)(qp + 16 * s);
    }
#pragma unroll
    for (int s = 0; s < NS; ++s) settle(qf[s]);
    float m = pa_ninf(), thr = pa_ninf(), l = 0.f, nmu = 0.f;
    // acc of 16 blocks at a time is added to total: one long chain of products' sums, four
    // keys a step, would round as often as there are steps
    f32x4 acc[NS], total[NS];
#pragma unroll
    for (int dt = 0; dt < NS; ++dt) acc[dt] = total[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int j = j0; j < j1; ++j) {
      const int par = (j - j0) & 1;
      wait_vmcnt<0>();
      settle(rows_next);
      lds_barrier();
      if (j + 1 < j1) {
        dma(rows_next, par ^ 1);
        rows_next = look(j + 2);
      }
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
      // register e of a half holds key 4 c + e
      if (j * BS + BS - 1 > lim_lo) {
        const int d = lim - j * BS - 4 * c;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int e = 0; e < 4; ++e) st[kt][e] = 16 * kt + e <= d ? st[kt][e] : pa_ninf();
      }
      float mx = pa_ninf();
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, st[kt][e]);
      if (__ballot(mx > thr) != 0) {
        const float mn = fmaxf(m, pair32_max(pair16_max(mx))), to = da_ref<DaF32>(mn, p.qscale);
        const float alpha = m == pa_ninf() ? 0.f : fast_exp2(to - nmu);
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
      float sum = 0.f;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float pr = fast_exp2(__builtin_fmaf(st[kt][e], p.qscale, nmu));
          sum += pr;
          const int kr = 16 * kt + 4 * c + e;
#pragma unroll
          for (int dt = 0; dt < NS; ++dt)
            acc[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                sv[kr * D + 4 * ((4 * dt + (ri >> 2)) ^ swz_v(kr)) + (ri & 3)], pr, acc[dt], 0, 0, 0);
        }
      l += sum;
      if ((j - j0) % 16 == 15) {
#pragma unroll
        for (int dt = 0; dt < NS; ++dt) {
          total[dt] += acc[dt];
          acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
      }
    }
    if (wave_live) {
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
      if (live && part >= 0) {
        const int64_t pi = part + r_mine - r0;
        if (c == 0) {
          p.ws_ml[2 * pi] = m == pa_ninf() ? m : -nmu;
          p.ws_ml[2 * pi + 1] = l;
        }
#pragma unroll
        for (int dt = 0; dt < NS; ++dt)
          *(float4 *)(p.ws_acc + pi * D + 16 * dt + 4 * c) = float4{acc[dt][0], acc[dt][1], acc[dt][2], acc[dt][3]};
      } else if (live) {
        const bool none = l == 0.f;
        const float inv = none ? 0.f : 1.f / l;
        float *o = (float *)p.out + pa_out_at(p, b, sq, t, h) + 4 * c;
#pragma unroll
        for (int dt = 0; dt < NS; ++dt)
          *(float4 *)(o + 16 * dt) = float4{acc[dt][0] * inv, acc[dt][1] * inv, acc[dt][2] * inv, acc[dt][3] * inv};
        if (p.lse && c == 0) p.lse[pa_lse_at(p, b, sq, t, h)] = none ? pa_ninf() : (__log2f(l) - nmu) * PA_LN2;
      }
      if (bad != 0) {
        bad |= bad >> 32;
        pa_again<float, D, 16, false, false>(p, b, sq, kvh, part, r0, r_first, (uint32_t)((bad | (bad >> 16)) & __ballot(live) & 0xffffu),
                                            j0 * BS, min(j1, lim_hi / BS + 1) * BS);
      }
    }
    if (!walk.next<R>(p, cost, upto)) break;
  }
}

// Joins the parts of the tile that began last in a workgroup's stretch: a row by D / 4 lanes.
template <int D, int R>
__global__ __launch_bounds__(256) void paged_join_kernel(PaKP p) {
  constexpr int LR = D / 4, RW = 256 / LR;  // lanes of a row, rows at a time
  const int wg = blockIdx.x;
  const int4 note = p.ws_join[wg];
  if (note.z == 0) return;
  const int kvh = wg % p.Hkv, b = note.x, G = p.G;
  const PaSeq sq = pa_seq(p, b);
  const int nrow = sq.lq * G, r0 = note.y * R, lane = threadIdx.x % LR;
  for (int r = r0 + blockIdx.y * RW + threadIdx.x / LR; r < min(nrow, r0 + R); r += gridDim.y * RW) {
    float m = pa_ninf(), l = 0.f;
    float4 acc{0.f, 0.f, 0.f, 0.f};
    // (parts in their order, four on their way at a time)
    for (int i0 = 0; i0 < note.z; i0 += 4) {
      float2 ml[4];
      float4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int x = min(i0 + i, note.z - 1);
        const int64_t pi = pa_part(p, wg + x * p.Hkv, x == 0) + r - r0;
        ml[i] = *(const float2 *)(p.ws_ml + 2 * pi);
        v[i] = *(const float4 *)(p.ws_acc + pi * D + 4 * lane);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i0 + i >= note.z || (ml[i].x == pa_ninf() && ml[i].y == 0.f)) continue;  // (empty: no key seen)
        const float mn = fmaxf(m, ml[i].x), from = mn == pa_ninf() ? 0.f : mn;
        const float f = m == pa_ninf() && l == 0.f ? 0.f : fast_exp2(m - from), g = fast_exp2(ml[i].x - from);
        m = mn;
        l = l * f + ml[i].y * g;
        acc.x = acc.x * f + v[i].x * g;
        acc.y = acc.y * f + v[i].y * g;
        acc.z = acc.z * f + v[i].z * g;
        acc.w = acc.w * f + v[i].w * g;
      }
    }
    const int t = r / G, h = kvh * G + r % G;
    const bool none = l == 0.f;
    const float inv = none ? 0.f : 1.f / l;
    const int64_t o = pa_out_at(p, b, sq, t, h) + 4 * lane;
    const float y[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
    if (p.out_dt == LA_F32) {
      *(float4 *)((float *)p.out + o) = float4{y[0], y[1], y[2], y[3]};
    } else if (p.out_dt == LA_BF16) {
      typedef __bf16 x4 __attribute__((ext_vector_type(4)));
      *(x4 *)((__bf16 *)p.out + o) = x4{(__bf16)y[0], (__bf16)y[1], (__bf16)y[2], (__bf16)y[3]};
    } else {
      typedef _Float16 x4 __attribute__((ext_vector_type(4)));
      *(x4 *)((_Float16 *)p.out + o) = x4{(_Float16)y[0], (_Float16)y[1], (_Float16)y[2], (_Float16)y[3]};
    }
    if (p.lse && lane == 0) p.lse[pa_lse_at(p, b, sq, t, h)] = none ? pa_ninf() : (m + __log2f(l)) * PA_LN2;
  }
}

// ------------------------------------------------------------------ host ----
struct PaPlan {
  int64_t W = 1, rows = 128, least = 0;
  size_t ml = 0, join = 0, bytes = 0;
};

static PaPlan pa_plan(const la_paged_attn_args *a) {
  PaPlan pl;
  const bool f32 = a->dtype == LA_F32;
  const int64_t G = a->Hq / a->Hkv, R = f32 ? 64 : 128;
  // workgroups that are there at once, shared among the KV heads; no stretch is shorter than four
  // blocks of keys and a tile's beginning and end
  pl.least = G * (4 * (f32 ? 32 : DA_BS) + PA_AHEAD);
  const int64_t rows = a->Tq * G, keys = a->pt_pages * a->page;  // (rows: of a sequence, at most)
  const int64_t tiles = a->cu_q ? std::min(rows, rows / R + a->B) : a->B * ceil_div(rows, R);  // at most
  const double most = (double)tiles * ((double)G * (keys + PA_AHEAD) + (a->causal ? R + 0.0 : 0.0));
  pl.W = std::max<int64_t>(1, (f32 ? 2 : 3) * num_cus() / a->Hkv);
  if (most / pl.least < (double)pl.W) pl.W = (int64_t)(most / pl.least) + 1;
  pl.rows = std::min(R, rows);
  const int64_t parts = pl.W * a->Hkv * 2 * pl.rows;
  pl.ml = ((size_t)parts * 2 * sizeof(float) + 255) / 256 * 256;
  pl.join = pl.ml + ((size_t)parts * a->D * sizeof(float) + 255) / 256 * 256;
  pl.bytes = pl.join + (size_t)(pl.W * a->Hkv) * sizeof(int4);
  return pl;
}

static int pa_check(const la_paged_attn_args *a) {
  LA_REQUIRE(a != nullptr, "la_paged_attention: null args");
  LA_REQUIRE(a->B > 0 && a->Hq > 0 && a->Hkv > 0 && a->Tq >= 0, "la_paged_attention: sizes must be positive");
  LA_REQUIRE(a->Hq % a->Hkv == 0, "la_paged_attention: Hq must be a multiple of Hkv");
  LA_REQUIRE(a->D == 64 || a->D == 128, "la_paged_attention: head_dim %lld (64 or 128)", (long long)a->D);
  LA_REQUIRE(a->dtype == LA_F32 || a->dtype == LA_BF16 || a->dtype == LA_F16, "la_paged_attention: dtype");
  LA_REQUIRE(a->kv_dtype == a->dtype || (a->kv_dtype == LA_FP8_E4M3 && a->dtype != LA_F32),
             "la_paged_attention: the cache has q's dtype, or fp8 codes with 16-bit q");
  LA_REQUIRE(a->out_dtype == a->dtype || a->out_dtype == LA_F32, "la_paged_attention: out_dtype is dtype or fp32");
  LA_REQUIRE(a->scale > 0.f && a->scale < 1e30f, "la_paged_attention: scale must be positive");
  LA_REQUIRE(a->n_phys > 0 && a->page > 0 && a->pt_pages > 0 && a->page < ((int64_t)1 << 30) / a->pt_pages,
             "la_paged_attention: bad cache");
  LA_REQUIRE(a->n_phys < ((int64_t)1 << 32) / a->page / a->Hkv, "la_paged_attention: a cache of 2^32 rows");
  LA_REQUIRE(a->B < ((int64_t)1 << 24) && a->Hq < ((int64_t)1 << 20) &&
                 (a->cu_q ? 1 : a->B) * std::max<int64_t>(1, a->Tq) < ((int64_t)1 << 30) / (a->Hq / a->Hkv),
             "la_paged_attention: sizes past 2^30 rows");
  LA_REQUIRE(!(a->cu_q && a->q_len), "la_paged_attention: q_len is for batched calls");
  return LA_OK;
}

template <class K>
static int pa_launch(K kernel, int64_t wgs, const PaKP &p, hipStream_t st) {
  kernel<<<dim3((uint32_t)wgs), dim3(256), 0, st>>>(p);
  LA_LAUNCHED();
  return LA_OK;
}
template <class T, int D>
static int pa_launch16(bool kv8, bool even, int64_t wgs, const PaKP &p, hipStream_t st) {
  if (kv8) return even ? pa_launch(paged_attn_kernel<T, D, true, true>, wgs, p, st) : pa_launch(paged_attn_kernel<T, D, true, false>, wgs, p, st);
  return even ? pa_launch(paged_attn_kernel<T, D, false, true>, wgs, p, st) : pa_launch(paged_attn_kernel<T, D, false, false>, wgs, p, st);
}

}  // namespace la

extern "C" size_t la_paged_attention_workspace(const la_paged_attn_args *a) {
  if (la::pa_check(a) != LA_OK || a->Tq == 0) return 0;
  return la::pa_plan(a).bytes;
}

extern "C" int la_paged_attention(const la_paged_attn_args *args, void *stream) {
  using namespace la;
  if (int rc = pa_check(args)) return rc;
  if (args->Tq == 0) return LA_OK;
  la_paged_attn_args x = *args;
  la_paged_attn_args *a = &x;
  const int64_t esz = a->dtype == LA_F32 ? 4 : 2, osz = a->out_dtype == LA_F32 ? 4 : 2;
  const bool packed = a->cu_q != nullptr, kv8 = a->kv_dtype == LA_FP8_E4M3;
  const int64_t nb = packed ? 1 : a->B;
  auto flat = [&](int64_t &b, int64_t &h, int64_t &t) {  // strides that nothing takes a step by
    if (nb == 1) b = 0;
    if (a->Hq == 1) h = 0;
    if (a->Tq == 1) t = 0;
  };
  flat(a->q_sb, a->q_sh, a->q_st);
  flat(a->o_sb, a->o_sh, a->o_st);
  auto rows_ok = [&](const void *y, int64_t es, int64_t b, int64_t h, int64_t t) {
    return y != nullptr && (uintptr_t)y % 16 == 0 && (b | h | t) % (16 / es) == 0;
  };
  LA_REQUIRE(rows_ok(a->q, esz, a->q_sb, a->q_sh, a->q_st), "la_paged_attention: rows of q must be 16-byte aligned");
  LA_REQUIRE(rows_ok(a->out, osz, a->o_sb, a->o_sh, a->o_st), "la_paged_attention: rows of out must be 16-byte aligned");
  LA_REQUIRE(rows_ok(a->k_pool, 1, 0, 0, 0) && rows_ok(a->v_pool, 1, 0, 0, 0), "la_paged_attention: the cache must be 16-byte aligned");
  LA_REQUIRE(a->page_table && a->lengths, "la_paged_attention: null page_table or lengths");
  LA_REQUIRE(!kv8 || (a->k_scale && a->v_scale && a->s_stride > 0), "la_paged_attention: fp8 cache needs scales");
  const int64_t pool = a->n_phys * a->Hkv * a->page * a->D * (kv8 ? 1 : esz);
  const Cover out(a->out, a->D * osz, {a->o_sb * osz, nb}, {a->o_sh * osz, a->Hq}, {a->o_st * osz, a->Tq});
  LA_REQUIRE(!overlap(out, Cover(a->q, a->D * esz, {a->q_sb * esz, nb}, {a->q_sh * esz, a->Hq}, {a->q_st * esz, a->Tq})) &&
                 !overlap(out, Cover(a->k_pool, pool)) && !overlap(out, Cover(a->v_pool, pool)),
             "la_paged_attention: out shares memory with an input");
  const PaPlan pl = pa_plan(a);
  if (!a->workspace || a->ws_bytes < (int64_t)pl.bytes)
    return fail(LA_ERR_WORKSPACE, "la_paged_attention: workspace %lld < %lld bytes", (long long)a->ws_bytes, (long long)pl.bytes);
  LA_REQUIRE((uintptr_t)a->workspace % 256 == 0, "la_paged_attention: workspace alignment");
  PaKP p{};
  p.q = a->q; p.k = a->k_pool; p.v = a->v_pool; p.out = a->out; p.lse = a->lse;
  p.k_scale = a->k_scale; p.v_scale = a->v_scale;
  p.page_table = a->page_table; p.lengths = a->lengths; p.cu_q = a->cu_q; p.q_len = a->q_len;
  p.ws_ml = (float *)a->workspace;
  p.ws_acc = (float *)((char *)a->workspace + pl.ml);
  p.ws_join = (int4 *)((char *)a->workspace + pl.join);
  p.Tq = a->Tq;
  p.q_sb = a->q_sb; p.q_sh = a->q_sh; p.q_st = a->q_st;
  p.o_sb = a->o_sb; p.o_sh = a->o_sh; p.o_st = a->o_st;
  p.l_sb = a->l_sb; p.l_sh = a->l_sh;
  p.pt_sb = a->pt_sb; p.s_stride = a->s_stride; p.n_phys = a->n_phys;
  p.least = pl.least;
  p.B = (int32_t)a->B; p.G = (int32_t)(a->Hq / a->Hkv); p.Hq = (int32_t)a->Hq; p.Hkv = (int32_t)a->Hkv;
  p.D = (int32_t)a->D; p.W = (int32_t)pl.W; p.part_rows = (int32_t)pl.rows;
  p.page = (int32_t)a->page; p.pt_pages = (int32_t)a->pt_pages;
  p.causal = a->causal != 0; p.out_dt = a->out_dtype; p.zero_rest = a->zero_rest != 0;
  p.qscale = a->scale * 1.44269504088896340736f;
  p.thr_gap = std::min((a->dtype == LA_F16 && !kv8 ? DaF16::GAP : DaBf16::GAP) / p.qscale, 3e38f);  // (finite: -inf + it stays)
  hipStream_t st = (hipStream_t)stream;
  const int64_t wgs = pl.W * a->Hkv;
  const bool even = a->page % 16 == 0, d128 = a->D == 128;
  int rc;
  if (a->dtype == LA_F32) rc = d128 ? pa_launch(paged_attn_f32_kernel<128>, wgs, p, st) : pa_launch(paged_attn_f32_kernel<64>, wgs, p, st);
  else if (a->dtype == LA_BF16) rc = d128 ? pa_launch16<DaBf16, 128>(kv8, even, wgs, p, st) : pa_launch16<DaBf16, 64>(kv8, even, wgs, p, st);
  else rc = d128 ? pa_launch16<DaF16, 128>(kv8, even, wgs, p, st) : pa_launch16<DaF16, 64>(kv8, even, wgs, p, st);
  if (rc != LA_OK) return rc;
  const dim3 grid((uint32_t)wgs, pl.rows > 32 ? 4 : 1);
  if (a->dtype == LA_F32) {
    if (d128) paged_join_kernel<128, 64><<<grid, 256, 0, st>>>(p);
    else paged_join_kernel<64, 64><<<grid, 256, 0, st>>>(p);
  } else {
    if (d128) paged_join_kernel<128, 128><<<grid, 256, 0, st>>>(p);
    else paged_join_kernel<64, 128><<<grid, 256, 0, st>>>(p);
  }
  LA_LAUNCHED();
  return LA_OK;
}
