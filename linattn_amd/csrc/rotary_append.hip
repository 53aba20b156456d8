// New keys turned by their positions and stored, with their values, in a paged cache, and the
// queries turned beside them (la_rotary_append): the KV concatenation of
// AttentionVariant.push_kv (core.py:219-220) with rotary positions on the way, the codec of
// kv/quant.py:76-93 where the cache is fp8, and Quest's page bounds
// (QuestAttention._refresh_pages, variants/selection.py:181-201) where it keeps them.
//
// Angles are counted once a token and workgroup and shared by its heads (rotary.h); each row is
// taken by as many lanes as it has units, four rows of a lane on their way at a time.  Bound by the
// rows' reads and writes: 14567 tokens of 32 + 8 + 8 heads of 128 bf16 values 76 us, 4.7 TB/s (a large
// copy has 4.9); 2048 into an fp8 cache 14 us (bytes 9.5; offsets, position and page are read one after the
// other, and the angles, which need the position alone, wait for the page too); 64 single tokens with page
// bounds 8 us, that chain alone.
#include <algorithm>

#include "rotary.h"

namespace la {

struct RaKP {
  RoAngles an;  // (pos null: a token's place in its sequence)
  const void *q, *k_new, *v_new;
  void *q_out, *k_pool, *v_pool, *mn, *mx;
  float *k_scale, *v_scale;
  const int32_t *page_table, *positions, *cu;
  int64_t B, T;  // batched: T tokens of each sequence; packed: T rows
  int64_t q_sb, q_sh, q_st, k_sb, k_sh, k_st, v_sb, v_sh, v_st, o_sb, o_sh, o_st;
  int64_t n_phys, pt_sb, m_sb, m_sh, m_sp, m_sd, n_pages, s_stride;
  int32_t Hq, Hkv, D, units, lanes, ts, hs;
  int32_t pool_page, pt_pages, meta_page, zero_rest, fp8;
  int64_t blocks;  // (with bounds)
};

// A token of a workgroup.
struct RaToken {
  int64_t row;   // of the cache, for head 0 (pool_page rows a head); -1: not stored
  int64_t at;    // its position in its sequence
  int32_t b, t;  // its indices in q, k_new, v_new (packed: 0 and the row); b < 0: of no sequence
};

// Token t of q's batch entry xb, in sequence b (< 0: none), `i` tokens behind the first new one.
__device__ __forceinline__ RaToken ra_token(const RaKP &p, int b, int64_t i, int xb, int t) {
  RaToken r;
  r.b = b < 0 ? -1 : xb;
  r.t = t;
  r.row = -1;
  r.at = 0;
  if (b < 0) return r;
  r.at = (int64_t)p.positions[b] + i;
  if (r.at < 0 || r.at >= (int64_t)p.pt_pages * p.pool_page) return r;
  const uint32_t page = (uint32_t)r.at / (uint32_t)p.pool_page;  // (pages times page size: below 2^31)
  const int64_t phys = p.page_table[b * p.pt_sb + page];
  if (phys >= 0 && phys < p.n_phys)
    r.row = phys * p.Hkv * p.pool_page + ((uint32_t)r.at - page * (uint32_t)p.pool_page);
  return r;
}

__device__ __forceinline__ int32_t ra_cu(const RaKP &p, int i) {
  return (int32_t)min(max((int64_t)p.cu[i], (int64_t)0), p.T);
}

// The angles of `count` tokens, by all threads, into LDS.
__device__ __forceinline__ void ra_angles(const RaKP &p, const RaToken *tok, int count, float2 *cs) {
  const int n = p.an.n;
  for (int e = threadIdx.x; e < count * n; e += RO_NT) {
    const int ti = e / n, f = e - ti * n;
    const RaToken t = tok[ti];
    if (t.b < 0) continue;
    const double pos = p.an.pos ? (double)p.an.pos[p.an.axis(f) * p.an.p_sa + t.b * p.an.p_sb + t.t * p.an.p_st]
                                : (double)t.at;
    cs[e] = p.an.turn(pos, f);
  }
}

// A row's values into the cache, at `row`; of fp8 the row's lanes (p.lanes of them, aligned) come
// together for the largest, and `unit.oa < 0` lanes take part with nothing.
template <class E, int V>
__device__ __forceinline__ void ra_store(const RaKP &p, const RoUnit<E, V> &unit, bool mine, void *pool, float *scales,
                                         int64_t row, float (&x)[2 * V]) {
  if (!p.fp8) {
    if (row >= 0) unit.store((E *)pool + row * p.D, x);
    return;
  }
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (mine) most = fmaxf(most, fabsf(x[i]));
    if (mine && unit.ob >= 0) most = fmaxf(most, fabsf(x[V + i]));
  }
  for (int o = 1; o < p.lanes; o <<= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
  // scale = max(absmax, 1e-8) / 448 and codes = e4m3(x / scale), in fp32 (IEEE divisions)
  const float scale = fmaxf(most, 1e-8f) / 448.f;
  if (row < 0 || !mine) return;
  uint8_t *to = (uint8_t *)pool + row * p.D;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int at = half ? unit.ob : unit.oa;
    if (at < 0) continue;
    if constexpr (V == 1) {
      to[at] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[half] / scale, 0.f, 0, false);
    } else {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[V * half + i] / scale, x[V * half + i + 1] / scale, 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(x[V * half + i + 2] / scale, x[V * half + i + 3] / scale, w, true);
        *(int *)(to + at + i) = w;
      }
    }
  }
  if (unit.oa == 0) scales[row * p.s_stride] = scale;
}

// Row r of a token: heads of q, then of k, then of v.
template <class E, int V>
__device__ __forceinline__ const E *ra_source(const RaKP &p, int b, int t, int r) {
  if (r < p.Hq) return (const E *)p.q + b * p.q_sb + t * p.q_st + r * p.q_sh;
  r -= p.Hq;
  if (r < p.Hkv) return (const E *)p.k_new + b * p.k_sb + t * p.k_st + r * p.k_sh;
  return (const E *)p.v_new + b * p.v_sb + t * p.v_st + (r - p.Hkv) * p.v_sh;
}

// Without page bounds: a workgroup takes `ts` tokens, packed or batched, as they lie, and each
// token's rows (heads of q, then of k, then of v), `hs` at a time.
template <class E, int V>
__global__ __launch_bounds__(RO_NT) void rotary_append_kernel(RaKP p) {
  typedef RoUnit<E, V> U;
  extern __shared__ float2 cs[];
  __shared__ RaToken s_tok[RO_NT];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, n = p.an.n;
  const int64_t tokens = p.cu ? p.T : p.B * p.T, tok0 = (int64_t)blockIdx.x * p.ts;
  const int count = (int)min((int64_t)p.ts, tokens - tok0);
  const int slot = tid / p.lanes, u = tid - slot * p.lanes;
  const int ti = slot / p.hs, r0 = slot % p.hs, R = p.Hq + 2 * p.Hkv;
  const bool mine = u < p.units;
  const U unit(mine ? u : 0, p.D, n, p.an.interleaved);
  // (rows do not wait for what their tokens are)
  constexpr int AHEAD = 4;
  typename U::vec xa[AHEAD], xb[AHEAD];
  const int64_t tok = tok0 + min(ti, count - 1);
  const int xb_ = p.cu ? 0 : (int)(tok / p.T), xt = (int)(tok - (int64_t)xb_ * p.T);
  const bool live = ti < count;
  if (live)
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (r0 + i * p.hs < R) unit.load(ra_source<E, V>(p, xb_, xt, r0 + i * p.hs), xa[i], xb[i]);
  if (p.cu) {
    // a wave a token: its sequence is the last that begins at or before it, looked for among every
    // `each`th, then from there on
    const int B = (int)p.B, each = (B + 63) / 64;
    for (int i = w; i < count; i += RO_NT / 64) {
      const int64_t x = tok0 + i;
      int b = __popcll(__ballot(lane * each < B && ra_cu(p, min(lane * each, B)) <= x)) - 1;
      if (each > 1 && b >= 0) {
        const int end = min((b + 1) * each, B);
        int n = 0;
        for (int b0 = b * each; b0 < end; b0 += 64) n += __popcll(__ballot(b0 + lane < end && ra_cu(p, min(b0 + lane, B)) <= x));
        b = b * each + max(n, 1) - 1;
      }
      const bool in = b >= 0 && x < ra_cu(p, b + 1) && x >= ra_cu(p, b);
      if (lane == 0) s_tok[i] = ra_token(p, in ? b : -1, in ? x - ra_cu(p, b) : 0, 0, (int)x);
    }
  } else if (tid < count) {
    const int64_t x = tok0 + tid;
    const int b = (int)(x / p.T), t = (int)(x - (int64_t)b * p.T);
    s_tok[tid] = ra_token(p, b, t, b, t);
  }
  __syncthreads();
  ra_angles(p, s_tok, count, cs);
  __syncthreads();
  if (!live) return;
  const RaToken token = s_tok[ti];
  RoTurns<V> turns;
  if (token.b >= 0) turns.load(cs + ti * n, unit.f0);
  for (int r = r0; r < R; r += AHEAD * p.hs) {
    if (r != r0)
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (r + i * p.hs < R) unit.load(ra_source<E, V>(p, xb_, xt, r + i * p.hs), xa[i], xb[i]);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int ri = r + i * p.hs;
      if (ri >= R) break;
      float x[2 * V];
      U::widen(xa[i], xb[i], x);
      if (ri < p.Hq + p.Hkv && unit.f0 >= 0 && token.b >= 0) turns.apply(x, p.an.interleaved);
      if (ri < p.Hq) {
        if (token.b < 0) {
          if (!p.zero_rest) continue;
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) x[j] = 0.f;
        }
        if (mine) unit.store((E *)p.q_out + xb_ * p.o_sb + xt * p.o_st + ri * p.o_sh, x);
      } else {
        const bool v = ri >= p.Hq + p.Hkv;
        const int h = ri - p.Hq - (v ? p.Hkv : 0);
        ra_store<E, V>(p, unit, mine, v ? p.v_pool : p.k_pool, v ? p.v_scale : p.k_scale,
                       token.row < 0 ? -1 : token.row + (int64_t)h * p.pool_page, x);
      }
    }
  }
}

__device__ __forceinline__ int64_t ra_floor(int64_t x, int64_t y) { return x / y - (x % y < 0); }

// Packed: which sequence the page of bounds is of that number blk of all that new tokens touch is (-1: of none),
// by all threads; blk becomes its place among the sequence's, or among those behind the last.
__device__ __forceinline__ int ra_page(const RaKP &p, int64_t &blk) {
  __shared__ int s_sum[RO_NT / 64];
  __shared__ int2 s_at;  // the sequence (or the first of some that hold it), the pages before it
  const int tid = threadIdx.x, lane = tid & 63, mp = p.meta_page;
  // pages that sequence x touches; a thread counts a sequence, or, of more than there are threads, as
  // many that lie one behind the other
  const int B = (int)p.B, each = (B + RO_NT - 1) / RO_NT;
  auto pages = [&](int x, int end) -> int {
    const int y = min(x, B - 1);
    const int64_t m = ra_cu(p, y + 1) - ra_cu(p, y), at = p.positions[y];
    return x < end && m > 0 ? (int)(ra_floor(at + m - 1, mp) - ra_floor(at, mp) + 1) : 0;
  };
  auto scan = [&](int sum) -> int {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(sum, o, 64);
      if (lane >= o) sum += y;
    }
    return sum;
  };
  int c = 0;
#pragma unroll 4
  for (int i = 0; i < each; ++i) c += pages(tid * each + i, B);
  int sum = scan(c), before = 0, all = 0;
  if (lane == 63) s_sum[tid >> 6] = sum;
  if (tid == 0) s_at = int2{-1, 0};
  __syncthreads();
#pragma unroll
  for (int w = 0; w < RO_NT / 64; ++w) {
    if (w < tid >> 6) before += s_sum[w];
    all += s_sum[w];
  }
  if (before + sum - c <= blk && blk < before + sum) s_at = int2{tid * each, before + sum - c};
  __syncthreads();
  int b = s_at.x;
  blk -= b < 0 ? all : s_at.y;
  if (b >= 0 && each > 1) {
    for (const int end = min(b + each, B);; b += 64) {
      c = pages(b + lane, end);
      sum = scan(c);
      const int here = __shfl(sum, 63, 64);
      if (blk < here || b + 64 >= end) break;
      blk -= here;
    }
    const int at = max(__ffsll((unsigned long long)__ballot(sum > blk)) - 1, 0);
    blk -= __shfl(sum - c, at, 64);
    b = min(b + at, B - 1);
  }
  return b;
}

// The least and largest of the slots' (V-value pairs `least`, `most` of each thread) into bounds of a page.
template <class E, int V>
__device__ __forceinline__ void ra_bounds(const RaKP &p, const float (&least)[2 * V],
                                          const float (&most)[2 * V], float *s_red, int b, int kvh, int64_t page, int64_t pos0,
                                          int64_t tokens) {
  typedef RoUnit<E, V> U;
  const int tid = threadIdx.x, n = p.an.n, mp = p.meta_page, slots = RO_NT / p.units, slot = tid / p.units, u = tid - slot * p.units;
  // a page that starts among the new tokens holds only them; else its old bounds cover the others
  const bool fresh = page * mp >= pos0;
  const int used = (int)min((int64_t)slots, tokens), cols = p.units * 2 * V;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    if (slot < used)
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) s_red[slot * cols + j * p.units + u] = side ? most[j] : least[j];
    __syncthreads();
    for (int e = tid; e < cols; e += RO_NT) {
      const int j = e / p.units;
      const U at(e - j * p.units, p.D, n, p.an.interleaved);
      if (j >= V && at.ob < 0) continue;
      float x = s_red[e];
      for (int s = 1; s < used; ++s) x = side ? fmaxf(x, s_red[s * cols + e]) : fminf(x, s_red[s * cols + e]);
      E *to = (E *)(side ? p.mx : p.mn) + b * p.m_sb + kvh * p.m_sh + page * p.m_sp + (j < V ? at.oa + j : at.ob + j - V) * p.m_sd;
      if (!fresh) x = side ? fmaxf(x, (float)*to) : fminf(x, (float)*to);
      *to = (E)x;
    }
    __syncthreads();
  }
}

// With page bounds: a workgroup takes the new tokens of one page of bounds of one sequence, and one KV
// head with its group of q, so that a page's least and largest keys are found without atomics.  Which
// page that is every workgroup finds by itself: in a batch of 4096 slots with 64 tokens in all that takes
// no time beside the rest (14 us, as without the empty slots).
template <class E, int V>
__global__ __launch_bounds__(RO_NT) void rotary_append_bounds_kernel(RaKP p) {
  typedef RoUnit<E, V> U;
  constexpr int TOK = 32;
  extern __shared__ float2 cs[];
  __shared__ RaToken s_tok[TOK];
  __shared__ float s_red[RO_NT * 2 * V];
  __shared__ int s_any;
  const int tid = threadIdx.x, n = p.an.n, mp = p.meta_page;
  const int kvh = (int)(blockIdx.x % (uint32_t)p.Hkv), G = p.Hq / p.Hkv;
  int64_t blk = blockIdx.x / (uint32_t)p.Hkv;
  int b = -1;
  int64_t pos0 = 0, first = 0, new_tokens = 0;  // its position, its first row (packed), its tokens
  if (p.cu) {
    b = ra_page(p, blk);
    if (b >= 0) {
      first = ra_cu(p, b);
      new_tokens = max(ra_cu(p, b + 1) - first, (int64_t)0);
    }
  } else {
    const int64_t per = p.blocks / p.B;
    b = (int)(blk / per);
    blk -= b * per;
    new_tokens = p.T;
  }
  if (b < 0) {  // (blk workgroups after the last: rows that no sequence holds)
    if (!p.zero_rest) return;
    const int64_t lo = ra_cu(p, 0), hi = max(lo, (int64_t)ra_cu(p, (int)p.B)), rest = lo + p.T - hi;
    const int64_t step = p.blocks - ((int64_t)(blockIdx.x / (uint32_t)p.Hkv) - blk);
    for (int64_t i = blk; i < rest; i += step)
      for (int e = tid; e < G * p.D; e += RO_NT)
        ((E *)p.q_out)[(i < lo ? i : hi + i - lo) * p.o_st + (kvh * G + e / p.D) * p.o_sh + e % p.D] = (E)0.f;
    return;
  }
  pos0 = p.positions[b];
  const int64_t page = ra_floor(pos0, mp) + blk;
  const int64_t lo = max(page * mp, pos0), hi = min((page + 1) * mp, pos0 + new_tokens);
  if (lo >= hi) return;  // (batched: fewer pages than there could be)
  const int xb = p.cu ? 0 : b;
  const int slots = RO_NT / p.units, slot = tid / p.units, u = tid - slot * p.units;
  const U unit(u, p.D, n, p.an.interleaved);
  float least[2 * V], most[2 * V];
#pragma unroll
  for (int i = 0; i < 2 * V; ++i) {
    least[i] = __int_as_float(0x7f800000);
    most[i] = __int_as_float(0xff800000);
  }
  if (tid == 0) s_any = 0;
  for (int64_t base = lo; base < hi; base += TOK) {
    const int count = (int)min((int64_t)TOK, hi - base);
    __syncthreads();
    if (tid < count) {
      const int64_t i = base + tid - pos0;
      const RaToken x = ra_token(p, b, i, xb, (int)(first + i));
      s_tok[tid] = x;
      if (x.row >= 0) s_any = 1;
    }
    __syncthreads();
    ra_angles(p, s_tok, count, cs);
    __syncthreads();
    if (slot >= slots) continue;
    // rows of the group's heads of q, k and v
    for (int i = slot; i < count * (G + 2); i += slots) {
      const int ti = i % count, g = i / count;  // (k first: its least and largest wait for the others)
      const RaToken x = s_tok[ti];
      const int r = g == 0 ? p.Hq + kvh : g == 1 ? p.Hq + p.Hkv + kvh : kvh * G + g - 2;
      typename U::vec a, c;
      unit.load(ra_source<E, V>(p, xb, x.t, r), a, c);
      float y[2 * V];
      U::widen(a, c, y);
      if (g != 1 && unit.f0 >= 0) {
        RoTurns<V> turns;
        turns.load(cs + ti * n, unit.f0);
        turns.apply(y, p.an.interleaved);
      }
      if (g >= 2) {
        unit.store((E *)p.q_out + xb * p.o_sb + x.t * p.o_st + r * p.o_sh, y);
      } else if (x.row >= 0) {
        unit.store((E *)(g == 0 ? p.k_pool : p.v_pool) + (x.row + (int64_t)kvh * p.pool_page) * p.D, y);
        if (g == 0)
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) {
            const float z = (float)(E)y[j];  // as stored
            least[j] = fminf(least[j], z);
            most[j] = fmaxf(most[j], z);
          }
      }
    }
  }
  __syncthreads();
  if (!s_any || page < 0 || page >= p.n_pages) return;  // (a token on no page counts in no bounds)
  ra_bounds<E, V>(p, least, most, s_red, b, kvh, page, pos0, hi - lo);
}

// The bounds alone, of the keys as rotary_append_kernel has stored them: a workgroup takes a page of bounds and
// `hs` KV heads, as many as leave four workgroups a CU (1024 single tokens 36 us, with a head each 66).
// Bound by the chain from the page's sequence to its keys, and by LDS, where the slots come together, once a head,
// one head after the other: 30 MB of keys of twelve prompts 40 us in pages of 16 tokens, of which half of the lanes
// have none, 25 in pages of 64.
template <class E, int V>
__global__ __launch_bounds__(RO_NT) void rotary_bounds_kernel(RaKP p) {
  typedef RoUnit<E, V> U;
  __shared__ int64_t s_row[RO_NT];
  __shared__ float s_red[RO_NT * 2 * V];
  __shared__ int s_any;
  const int tid = threadIdx.x, mp = p.meta_page, groups = p.Hkv / p.hs;
  const int h0 = (int)(blockIdx.x % (uint32_t)groups) * p.hs;
  int64_t blk = blockIdx.x / (uint32_t)groups, new_tokens = p.T;
  int b = 0;
  if (p.cu) {
    b = ra_page(p, blk);
    if (b < 0) return;  // (fewer pages than there could be)
    new_tokens = max(ra_cu(p, b + 1) - ra_cu(p, b), 0);
  } else {
    const int64_t per = p.blocks / p.B;
    b = (int)(blk / per);
    blk -= b * per;
  }
  const int64_t pos0 = p.positions[b], page = ra_floor(pos0, mp) + blk;
  const int64_t lo = max(page * mp, pos0), hi = min((page + 1) * mp, pos0 + new_tokens);
  if (lo >= hi || page < 0 || page >= p.n_pages) return;
  const int slots = RO_NT / p.units, slot = tid / p.units, u = tid - slot * p.units;
  const U unit(u, p.D, p.an.n, p.an.interleaved);
  if (tid == 0) s_any = 0;
  for (int kvh = h0; kvh < h0 + p.hs; ++kvh) {
    float least[2 * V], most[2 * V];
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) {
      least[i] = __int_as_float(0x7f800000);
      most[i] = __int_as_float(0xff800000);
    }
    for (int64_t base = lo; base < hi; base += RO_NT) {
      const int count = (int)min((int64_t)RO_NT, hi - base);
      if (kvh == h0 || hi - lo > RO_NT) {  // (else they are there)
        __syncthreads();
        if (tid < count) {
          const int64_t row = ra_token(p, b, base + tid - pos0, 0, 0).row;
          s_row[tid] = row;
          if (row >= 0) s_any = 1;
        }
        __syncthreads();
      }
      if (slot < slots)
#pragma unroll 4
        for (int i = slot; i < count; i += slots) {
          const int64_t row = s_row[i];
          if (row < 0) continue;
          typename U::vec a, c;
          unit.load((const E *)p.k_pool + (row + (int64_t)kvh * p.pool_page) * p.D, a, c);
          float y[2 * V];
          U::widen(a, c, y);
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) {
            least[j] = fminf(least[j], y[j]);
            most[j] = fmaxf(most[j], y[j]);
          }
        }
    }
    __syncthreads();
    if (!s_any) return;  // (a token on no page counts in no bounds)
    ra_bounds<E, V>(p, least, most, s_red, b, kvh, page, pos0, hi - lo);
  }
}

template <class E, int V>
static int ra_launch(RaKP p, hipStream_t st) {
  p.units = RoUnit<E, V>::count(p.D, p.an.n);
  p.lanes = p.units;
  if (p.fp8) {  // a row's lanes find its largest by swaps within a wave
    p.lanes = 1 << ilog2(p.units);
    if (p.lanes > 64) return fail(LA_ERR_UNSUPPORTED, "la_rotary_append: fp8 rows of %d values need aligned chunks", p.D);
  }
  const size_t turns = (size_t)p.an.n * sizeof(float2);
  const int64_t tokens = p.cu ? p.T : p.B * p.T;
  if (p.mn) {
    // (packed: no more than a token each, or than the tokens fill and one at either end of each sequence;
    // and one for the rest)
    p.blocks = p.cu ? std::min(p.T, p.T / p.meta_page + 2 * p.B) + 1 : p.B * (ceil_div(p.T - 1, p.meta_page) + 1);
    LA_REQUIRE(grid_fits(p.blocks * p.Hkv, RO_NT), "la_rotary_append: too many tokens");
    // few tokens in one launch; of more its angles, once a KV head, cost more than a launch (64 tokens 14.0 us,
    // in two 14.7; 128 of four sequences 17.6 and 14.9, 2048 31 and 23, twelve prompts into pages of 16
    // 141 and 110, 256 single ones 20.5 and 15.5)
    if (tokens < 128) {
      rotary_append_bounds_kernel<E, V><<<dim3((uint32_t)(p.blocks * p.Hkv)), RO_NT, 32 * turns, st>>>(p);
      LA_LAUNCHED();
      return LA_OK;
    }
  }
  const int slots = RO_NT / p.lanes, R = p.Hq + 2 * p.Hkv;
  // tokens of a workgroup: about eight rows a lane, where there are tokens for every CU (twelve prompts
  // into pages of 16 76 us, with four rows a lane 81, sixteen 77; into fp8 72, 82 and 70)
  p.ts = (int)std::min<int64_t>(std::max(1, 8 * slots / R), std::max<int64_t>(1, tokens / (2 * num_cus())));
  p.ts = std::min(p.ts, slots);
  p.hs = std::min(R, slots / p.ts);
  const int64_t wgs = ceil_div(tokens, p.ts);
  LA_REQUIRE(grid_fits(wgs, RO_NT), "la_rotary_append: too many tokens");
  rotary_append_kernel<E, V><<<dim3((uint32_t)wgs), RO_NT, p.ts * turns, st>>>(p);
  LA_LAUNCHED();
  if (p.mn) {
    p.hs = (int32_t)std::min<int64_t>(p.Hkv, std::max<int64_t>(1, p.blocks * p.Hkv / (4 * num_cus())));
    while (p.Hkv % p.hs) --p.hs;
    rotary_bounds_kernel<E, V><<<dim3((uint32_t)(p.blocks * (p.Hkv / p.hs))), RO_NT, 0, st>>>(p);
    LA_LAUNCHED();
  }
  return LA_OK;
}

}  // namespace la

extern "C" int la_rotary_append(const la_rotary_append_args *args, void *stream) {
  using namespace la;
  LA_REQUIRE(args != nullptr, "la_rotary_append: null args");
  la_rotary_append_args x = *args;
  la_rotary_append_args *a = &x;
  LA_REQUIRE(a->B > 0 && a->T >= 0 && a->Hq >= 0 && a->Hkv > 0 && a->D > 0 && a->n > 0 && a->A > 0,
             "la_rotary_append: sizes must be positive");
  LA_REQUIRE(a->Hq % a->Hkv == 0, "la_rotary_append: Hq must be a multiple of Hkv");
  LA_REQUIRE(a->D <= 512 && 2 * a->n <= a->D, "la_rotary_append: head_dim up to 512, at most half as many frequencies");
  LA_REQUIRE(a->Hq + 2 * a->Hkv < 65536 && a->A < 65536, "la_rotary_append: too many heads");
  LA_REQUIRE(a->dtype == LA_F32 || a->dtype == LA_BF16 || a->dtype == LA_F16, "la_rotary_append: dtype");
  const bool fp8 = a->pool_dtype == LA_FP8_E4M3;
  LA_REQUIRE(fp8 || a->pool_dtype == a->dtype, "la_rotary_append: the pool stores the input dtype (or fp8 codes)");
  LA_REQUIRE(a->n_phys > 0 && a->pool_page > 0 && a->pt_pages > 0 && a->pool_page < ((int64_t)1 << 31) / a->pt_pages,
             "la_rotary_append: bad pool");
  const bool meta = a->page_min != nullptr || a->page_max != nullptr;
  if (meta) {
    LA_REQUIRE(a->page_min && a->page_max, "la_rotary_append: both bounds tensors");
    if (fp8) return fail(LA_ERR_UNSUPPORTED, "la_rotary_append: page bounds of an fp8 pool");
    LA_REQUIRE(a->meta_page > 0 && a->meta_page < ((int64_t)1 << 30) && a->n_pages > 0, "la_rotary_append: bad page bounds shape");
  }
  if (a->T == 0) return LA_OK;
  const bool packed = a->cu != nullptr;
  LA_REQUIRE(a->B < ((int64_t)1 << 24) && a->T < ((int64_t)1 << 30) && (packed || a->B < ((int64_t)1 << 30) / a->T),
             "la_rotary_append: too many tokens");
  LA_REQUIRE(a->k_new && a->v_new && a->k_pool && a->v_pool && a->page_table && a->positions && (a->Hq == 0 || (a->q && a->q_out)),
             "la_rotary_append: null pointer");
  LA_REQUIRE(a->inv_freq && (a->axes || a->A == 1) && (a->rot_positions || a->A == 1),
             "la_rotary_append: null frequencies, axes or positions");
  LA_REQUIRE(!fp8 || (a->k_scale && a->v_scale && a->s_stride > 0), "la_rotary_append: fp8 pool needs scales");
  const int64_t nb = packed ? 1 : a->B, esz = a->dtype == LA_F32 ? 4 : 2, psz = fp8 ? 1 : esz;
  auto flat = [&](int64_t &b, int64_t &h, int64_t &t, int64_t heads) {  // strides that nothing takes a step by
    if (nb == 1) b = 0;
    if (heads <= 1) h = 0;
    if (a->T == 1) t = 0;
  };
  flat(a->q_sb, a->q_sh, a->q_st, a->Hq);
  flat(a->o_sb, a->o_sh, a->o_st, a->Hq);
  flat(a->kn_sb, a->kn_sh, a->kn_st, a->Hkv);
  flat(a->vn_sb, a->vn_sh, a->vn_st, a->Hkv);
  auto cover = [&](const void *y, int64_t b, int64_t h, int64_t t, int64_t heads) {
    return Cover(y, a->D * esz, {b * esz, nb}, {h * esz, heads}, {t * esz, a->T});
  };
  const int64_t pool = a->n_phys * a->Hkv * a->pool_page, m_run = a->m_sd == 1 ? a->D : 1;
  auto page_bounds = [&](const void *y) {
    return Cover(meta ? y : nullptr, m_run * esz, {a->m_sb * esz, a->B}, {a->m_sh * esz, a->Hkv}, {a->m_sp * esz, a->n_pages},
                 {a->m_sd * esz, a->D / m_run});
  };
  const Cover::Dim each{a->s_stride * 4, pool};
  const Cover written[] = {cover(a->Hq ? a->q_out : nullptr, a->o_sb, a->o_sh, a->o_st, a->Hq),
                           Cover(a->k_pool, pool * a->D * psz),
                           Cover(a->v_pool, pool * a->D * psz),
                           Cover(fp8 ? a->k_scale : nullptr, 4, each),
                           Cover(fp8 ? a->v_scale : nullptr, 4, each),
                           page_bounds(a->page_min),
                           page_bounds(a->page_max)};
  // (in place: the same rows, each of which the lanes that write it have read)
  const bool in = a->q_out == a->q && a->o_sb == a->q_sb && a->o_sh == a->q_sh && a->o_st == a->q_st;
  const Cover read[] = {cover(a->Hq && !in ? a->q : nullptr, a->q_sb, a->q_sh, a->q_st, a->Hq),
                        cover(a->k_new, a->kn_sb, a->kn_sh, a->kn_st, a->Hkv),
                        cover(a->v_new, a->vn_sb, a->vn_sh, a->vn_st, a->Hkv),
                        Cover(a->page_table, a->pt_pages * 4, {a->pt_sb * 4, a->B}),
                        Cover(a->positions, a->B * 4),
                        Cover(a->cu, (a->B + 1) * 4),
                        Cover(a->rot_positions, 4, {a->p_sa * 4, a->A}, {a->p_sb * 4, nb}, {a->p_st * 4, a->T}),
                        Cover(a->inv_freq, a->n * 4),
                        Cover(a->axes, a->n * 4)};
  LA_REQUIRE(!overlap_any(written, read), "la_rotary_append: what is written shares memory with another argument");
  RaKP p{};
  p.an = RoAngles{a->rot_positions, a->axes, a->inv_freq, a->p_sa, a->p_sb, a->p_st, (int32_t)a->n, (int32_t)a->A,
                  a->interleaved != 0, 0};
  p.q = a->q; p.k_new = a->k_new; p.v_new = a->v_new;
  p.q_out = a->q_out; p.k_pool = a->k_pool; p.v_pool = a->v_pool;
  p.mn = a->page_min; p.mx = a->page_max;
  p.k_scale = a->k_scale; p.v_scale = a->v_scale;
  p.page_table = a->page_table; p.positions = a->positions; p.cu = a->cu;
  p.B = a->B; p.T = a->T;
  p.q_sb = a->q_sb; p.q_sh = a->q_sh; p.q_st = a->q_st;
  p.k_sb = a->kn_sb; p.k_sh = a->kn_sh; p.k_st = a->kn_st;
  p.v_sb = a->vn_sb; p.v_sh = a->vn_sh; p.v_st = a->vn_st;
  p.o_sb = a->o_sb; p.o_sh = a->o_sh; p.o_st = a->o_st;
  p.n_phys = a->n_phys; p.pt_sb = a->pt_sb;
  p.m_sb = a->m_sb; p.m_sh = a->m_sh; p.m_sp = a->m_sp; p.m_sd = a->m_sd;
  p.n_pages = a->n_pages; p.s_stride = a->s_stride;
  p.Hq = (int32_t)a->Hq; p.Hkv = (int32_t)a->Hkv; p.D = (int32_t)a->D;
  p.pool_page = (int32_t)a->pool_page; p.pt_pages = (int32_t)a->pt_pages; p.meta_page = (int32_t)a->meta_page;
  p.zero_rest = packed && a->zero_rest != 0; p.fp8 = fp8;
  uint64_t at = (uint64_t)(uintptr_t)a->k_new | (uint64_t)(uintptr_t)a->v_new;
  uint64_t by = (uint64_t)(a->kn_sb | a->kn_sh | a->kn_st | a->vn_sb | a->vn_sh | a->vn_st);
  if (a->Hq) {
    at |= (uint64_t)(uintptr_t)a->q | (uint64_t)(uintptr_t)a->q_out;
    by |= (uint64_t)(a->q_sb | a->q_sh | a->q_st | a->o_sb | a->o_sh | a->o_st);
  }
  const uint64_t pools = (uint64_t)(uintptr_t)a->k_pool | (uint64_t)(uintptr_t)a->v_pool;
  if (!fp8) at |= pools;
  hipStream_t st = (hipStream_t)stream;
  // codes are written four at a time, of chunks of any size but one
  const int v = fp8 && pools % 4 != 0 ? 1 : ro_vector((int)esz, a->D, a->n, at, by);
  LA_REQUIRE(at % esz == 0, "la_rotary_append: unaligned tensors");
  if (a->dtype == LA_F32) return v == 4 ? ra_launch<float, 4>(p, st) : ra_launch<float, 1>(p, st);
  if (a->dtype == LA_BF16)
    return v == 8 ? ra_launch<__bf16, 8>(p, st) : v == 4 ? ra_launch<__bf16, 4>(p, st) : ra_launch<__bf16, 1>(p, st);
  return v == 8 ? ra_launch<_Float16, 8>(p, st) : v == 4 ? ra_launch<_Float16, 4>(p, st) : ra_launch<_Float16, 1>(p, st);
}
