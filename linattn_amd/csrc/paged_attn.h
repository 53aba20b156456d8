// Dense attention over a paged cache: which keys of which rows a workgroup takes, where they
// lie, and how parts of rows are joined.  Used by paged_attn.hip.
//
// Rows: row r of a sequence and KV head is query r / G of head r % G of its group (so the heads of
// a group share every staged key); R of them are a tile, which walks the keys its last row sees.
//
// The lengths are known on the device only, and a batch holds single tokens beside long chunks, so
// the work is shared out there: all tiles of a KV head in a line, sequence after sequence, each
// as long as its keys (and a little, for its beginning and end); of that line every workgroup
// takes a stretch, across the ends of tiles.  A tile that lies in one stretch is finished by
// its workgroup; of one that does not, each workgroup leaves its part (unnormalised sums,
// reference and weight sum of each row) and the join, a second launch, adds them up.
// Sequences of few rows (at most 16: single tokens, bound by the reads) have a line of their own.
// There are as many stretches as there are places for workgroups: with three times as many, the
// last of which would fill the places of workgroups that are done early, beginnings and ends
// cost more than that gains (tokens of 48 sequences 333 us in place of 312, tokens and chunks
// together 293 in place of 254).
#pragma once

#include "few_rows.h"

namespace la {

struct PaKP {
  const void *q, *k, *v;
  void *out;
  float *lse;
  const float *k_scale, *v_scale;
  const int32_t *page_table, *lengths, *cu_q, *q_len;
  float *ws_ml, *ws_acc;  // parts (pa_part): (reference, sum) and D values (pa_in_part) of each row
  int4 *ws_join;          // [workgroup]: of the tile that begins last there: sequence, tile, parts (0: none), and
                          // 1 + the stretch's number where rows are few, else 0
  int64_t Tq, q_sb, q_sh, q_st, o_sb, o_sh, o_st, l_sb, l_sh, pt_sb, s_stride, n_phys;
  int64_t least, least_few, few_parts;  // of a stretch, of few rows; where the parts of few rows begin
  int32_t B, G, Hq, Hkv, D, W, part_rows;  // W: workgroups of a KV head
  int32_t page, pt_pages, causal, out_dt, zero_rest;
  float qscale, thr_gap;
};

// What a tile's beginning and end cost, in keys (twelve prompts 264, 256 and 263 us at 160, 256, 600).
constexpr int PA_AHEAD = 256;

struct PaSeq {
  int32_t lq, lk;
  int64_t q0;  // packed: its first row
};

__device__ __forceinline__ PaSeq pa_seq(const PaKP &p, int b) {
  PaSeq s;
  if (p.cu_q) {
    const int32_t a = da_cu(p.cu_q, b, p.Tq), e = da_cu(p.cu_q, b + 1, p.Tq);
    s.q0 = a;
    s.lq = max(e - a, 0);
  } else {
    s.q0 = 0;
    s.lq = (int32_t)(p.q_len ? min(max((int64_t)p.q_len[b], (int64_t)0), p.Tq) : p.Tq);
  }
  s.lk = min(max(p.lengths[b], 0), p.pt_pages * p.page);  // (below 2^31)
  return s;
}

// A sequence's tiles: tile i costs a + step (i + 1), in keys times G.
struct PaTiles {
  int64_t a, step;
  int32_t n;
  __device__ __forceinline__ int64_t upto(int64_t i) const { return i * a + step * (i * (i + 1) / 2); }
  __device__ __forceinline__ int64_t cost(int64_t i) const { return a + step * (i + 1); }
};
constexpr int PA_FEW = 16;  // rows of a sequence that are few
// (n 0: no tiles in that line; FEW: whether there are two)
template <int R, bool FEW>
__device__ __forceinline__ PaTiles pa_tiles(const PaKP &p, const PaSeq &s, bool few) {
  PaTiles t;
  const int64_t rows = (int64_t)s.lq * p.G;
  t.n = FEW && (rows <= PA_FEW) != few ? 0 : (int32_t)((rows + R - 1) / R);
  t.a = (int64_t)p.G * ((p.causal ? max(s.lk - s.lq, 0) : s.lk) + PA_AHEAD);
  t.step = p.causal ? R : 0;
  return t;
}

__device__ __forceinline__ int64_t pa_uniform(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x), hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)x >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ int64_t pa_lane_value(int64_t x, int lane) {  // (the same lane for all)
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)x, lane), hi = __builtin_amdgcn_readlane((uint32_t)((uint64_t)x >> 32), lane);
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
// Sum over the lanes up to this one, on the vector unit (shuffles go through LDS: a call's first
// microsecond is such sums).
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t pa_dpp(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)((uint64_t)x >> 32), CTRL, ROWS, 0xf, false);
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ int64_t pa_scan(int64_t x) {
  x += pa_dpp<0x111, 0xf>(x);  // 1, 2, 4, 8 lanes up within rows of 16
  x += pa_dpp<0x112, 0xf>(x);
  x += pa_dpp<0x114, 0xf>(x);
  x += pa_dpp<0x118, 0xf>(x);
  x += pa_dpp<0x142, 0xa>(x);  // lane 15 of a row to the next, then lane 31 to the upper half
  x += pa_dpp<0x143, 0xc>(x);
  return x;
}
// a / b, both below 2^53, a >= 0, b > 0
__device__ __forceinline__ int64_t pa_div(int64_t a, int64_t b) {
  int64_t q = (int64_t)((double)a / (double)b);
  const int64_t r = a - q * b;
  return r < 0 ? q - 1 : r >= b ? q + 1 : q;
}

// A line: its length, that of a stretch (but of the last), its first workgroup.
struct PaLine {
  int64_t all, quota;
  int32_t first;
};

// The stretch of workgroup w of a KV head: sequence b, tile i, `off` into the tile, which begins at
// `pos` of the line; `left` is the stretch's length (0: none).
struct PaStretch {
  PaLine line;
  int64_t off, left, pos;
  int32_t b, i, few, mixed;  // mixed: there are both lines
};
template <int R, bool FEW>
__device__ __forceinline__ PaStretch pa_stretch(const PaKP &p, int w, PaSeq &seq, PaTiles &tiles) {
  const int lane = threadIdx.x & 63;
  auto cost = [&](const PaSeq &q, int b, bool few) -> int64_t {
    const PaTiles t = pa_tiles<R, FEW>(p, q, few);
    return b < p.B ? t.upto(t.n) : 0;
  };
  // a lane counts a sequence, or, of more than 64, as many that lie one behind the other
  const int each = (p.B + 63) / 64;
  PaSeq mine = pa_seq(p, min(lane * each, p.B - 1));
  int64_t sum_many = cost(mine, lane * each, false), sum_few = FEW ? cost(mine, lane * each, true) : 0;
#pragma unroll 4
  for (int i = 1; i < each; ++i) {
    const int b = lane * each + i;
    const PaSeq q = pa_seq(p, min(b, p.B - 1));
    sum_many += cost(q, b, false);
    if (FEW) sum_few += cost(q, b, true);
  }
  sum_many = pa_scan(sum_many);
  if (FEW) sum_few = pa_scan(sum_few);
  const int64_t many = pa_lane_value(sum_many, 63), few = pa_lane_value(sum_few, 63);
  PaStretch s;
  s.left = 0;
  s.b = s.i = 0;
  // places for tiles of many rows, by the share of the time (beside them, a block of few rows takes a
  // little less than one of many: three mixed batches 707, 697, 702, 709 and 747 us together at 0.5,
  // 0.65, 0.8, 1 and 1.3)
  const int wm = few == 0 ? p.W : many == 0 ? 0 : max(1, min(p.W - 1, (int)((double)p.W * (double)many / ((double)many + 0.7 * (double)few) + 0.5)));
  s.few = w >= wm && few > 0;
  s.mixed = few > 0 && many > 0;
  s.line.all = s.few ? few : many;
  s.line.first = s.few ? wm : 0;
  const int places = s.few ? p.W - wm : max(wm, 1);
  s.line.quota = max(pa_div(s.line.all + places - 1, places), s.few ? p.least_few : p.least);
  s.off = (w - s.line.first) * s.line.quota;
  if (s.off >= s.line.all) return s;
  s.left = min(s.line.quota, s.line.all - s.off);
  s.pos = s.off;
  int64_t sum = s.few ? sum_few : sum_many;
  int at = __ffsll((unsigned long long)__ballot(sum > s.off)) - 1;  // (off is below the line's end)
  if (at > 0) s.off -= pa_lane_value(sum, at - 1);
  int first = at * each;
  if (each == 1) {
    first = 0;
  } else {
    for (const int end = min(first + each, p.B);; first += 64) {
      const int b = first + lane;
      mine = pa_seq(p, min(b, p.B - 1));
      sum = pa_scan(b < end ? cost(mine, b, s.few) : 0);
      const int64_t here = pa_lane_value(sum, 63);
      if (s.off < here || first + 64 >= end) break;
      s.off -= here;
    }
    at = __ffsll((unsigned long long)__ballot(sum > s.off)) - 1;
    if (at > 0) s.off -= pa_lane_value(sum, at - 1);
  }
  s.b = __builtin_amdgcn_readfirstlane(first + at);
  seq.lq = __builtin_amdgcn_readlane(mine.lq, at);
  seq.lk = __builtin_amdgcn_readlane(mine.lk, at);
  seq.q0 = pa_lane_value(mine.q0, at);
  tiles = pa_tiles<R, FEW>(p, seq, s.few);
  if (tiles.n > 1) {
    // upto(i) <= off < upto(i + 1): the quadratic's root, and what its rounding may have missed
    int64_t i;
    if (tiles.step == 0) {
      i = pa_div(s.off, tiles.a);
    } else {
      const double h = (double)tiles.a + 0.5 * (double)tiles.step;
      i = (int64_t)((sqrt(h * h + 2.0 * (double)tiles.step * (double)s.off) - h) / (double)tiles.step);
    }
    i = min(max(i, (int64_t)0), (int64_t)tiles.n - 1);
    while (i > 0 && tiles.upto(i) > s.off) --i;
    while (i + 1 < tiles.n && tiles.upto(i + 1) <= s.off) ++i;
    s.i = __builtin_amdgcn_readfirstlane((int32_t)i);
    s.off = pa_uniform(s.off - tiles.upto(i));
  }
  s.left = pa_uniform(s.left);
  s.pos -= s.off;
  return s;
}

// A part of a row of stretch x of a KV head: where it is kept until the parts are joined.
__device__ __forceinline__ int64_t pa_part(const PaKP &p, int64_t x, int kvh, bool last, bool few) {
  const int64_t at = (x * p.Hkv + kvh) * 2 + (last ? 1 : 0);
  return few ? p.few_parts + at * PA_FEW : at * p.part_rows;
}

// Where value d of row r of a tile of D-value rows lies in its part, in 16-bit types: the 32 rows of a wave as
// its lanes hold them (register i of dim tile dt of lane l: dim 32 dt + 8 (i / 4) + 4 (l / 32) + i % 4 of row
// l % 32), so that a wave writes and reads 1 KB at a time.
template <int D>
__device__ __forceinline__ int64_t pa_in_part(int r, int d) {
  return (int64_t)(r >> 5) * 32 * D + ((d >> 5) * 4 + ((d >> 3) & 3)) * 256 + ((((d >> 2) & 1) << 5) | (r & 31)) * 4 + (d & 3);
}

// Of a tile of `n` staged blocks of keys and cost C, those before place c.
__device__ __forceinline__ int pa_blocks(int n, int64_t c, int64_t C) {
  if (c <= 0) return 0;
  if (c >= C) return n;
  return min((int)((double)n * ((double)c / (double)C)), n);
}

// The cache's row of (page entry of key, KV head): its place among the pool's rows.
__device__ __forceinline__ uint32_t pa_row(const PaKP &p, const int32_t *pages, int key, int kvh) {
  const uint32_t at = (uint32_t)key / (uint32_t)p.page;
  const int64_t phys = min(max((int64_t)pages[at], (int64_t)0), p.n_phys - 1);
  return (uint32_t)((phys * p.Hkv + kvh) * p.page + ((uint32_t)key - at * (uint32_t)p.page));
}

__device__ __forceinline__ int64_t pa_q_at(const PaKP &p, int b, const PaSeq &s, int t, int h) {
  return (p.cu_q ? (s.q0 + t) * p.q_st : b * p.q_sb + t * p.q_st) + h * p.q_sh;
}
__device__ __forceinline__ int64_t pa_out_at(const PaKP &p, int b, const PaSeq &s, int t, int h) {
  return (p.cu_q ? (s.q0 + t) * p.o_st : b * p.o_sb + t * p.o_st) + h * p.o_sh;
}
__device__ __forceinline__ int64_t pa_lse_at(const PaKP &p, int b, const PaSeq &s, int t, int h) {
  return (p.cu_q ? s.q0 + t : b * p.l_sb + t) + h * p.l_sh;
}

// Rows of the call that no sequence holds: zeros, lse -inf; shared out over the workgroups.
template <int D>
__device__ __forceinline__ void pa_rest(const PaKP &p, int kvh) {
  const float ninf = __int_as_float(0xff800000);
  auto zero = [&](int64_t o, int64_t l) {
    for (int e = threadIdx.x; e < p.G * D; e += blockDim.x)
      store_from_f32(p.out, o + (kvh * p.G + e / D) * p.o_sh + e % D, p.out_dt, 0.f);
    if (p.lse)
      for (int g = threadIdx.x; g < p.G; g += blockDim.x) p.lse[l + (kvh * p.G + g) * p.l_sh] = ninf;
  };
  const int64_t first = blockIdx.x / (uint32_t)p.Hkv, step = p.W;
  if (p.cu_q) {
    if (!p.zero_rest) return;
    const int64_t lo = da_cu(p.cu_q, 0, p.Tq), hi = max(lo, (int64_t)da_cu(p.cu_q, p.B, p.Tq));
    for (int64_t i = first; i < lo + p.Tq - hi; i += step) {
      const int64_t t = i < lo ? i : hi + i - lo;
      zero(t * p.o_st, t);
    }
  } else if (p.q_len) {
    for (int64_t i = first; i < (int64_t)p.B * p.Tq; i += step) {
      const int64_t b = i / p.Tq, t = i % p.Tq;
      if (t >= p.q_len[b]) zero(b * p.o_sb + t * p.o_st, b * p.l_sb + t);
    }
  }
}

}  // namespace la
