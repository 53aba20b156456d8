// Eviction from a cache by the weights its entries gathered (la_evict_kv): the entries a
// sequence keeps, and their rows copied to a cache of their own.
//
// The smallest kept key of a (sequence, KV head) is found by a radix select, digit by
// digit over histograms in LDS; then every wave lists what it keeps of its own stretch of
// the entries, in order.  Without positions the protected entries are the first and the
// last ones and are never looked at; else they are keys above all others.
// Up to EV_SMALL entries: one kernel, whose workgroups each select (keys in registers,
// 8-bit digits) and copy 64 of the row's slots: repeating the selection costs less than a
// second launch.  Up to EV_MID: evict_select_kernel, a workgroup a row, writes the list,
// evict_copy_kernel copies the rows.  Longer ones would be bound by the instructions that
// their keys cost on one CU (100 000 cycles for 65536, measured), so slices of a row have
// workgroups of their own, and each digit a launch (evict_digit_kernel): the histograms
// of a row's slices are added by whoever needs the sum, in place of atomics.
// Slots that are not chosen by weight (the newest tokens, mostly half of the cache) wait
// for no selection: the selecting launches, which leave the memory idle, copy them in
// workgroups of their own (four caches of 6572 to 66473 entries of 8 heads cut to 4096: 61
// us without, 55.7 with; passes 7, 11, 11 and 11 us, the rest of the rows 12, of which 28
// would move all bytes at the rate of a large copy).
#include <algorithm>

#include "evict.h"

namespace la {

struct EvKP {
  const char *k, *v;
  const float *weights;
  const int32_t *positions, *pos, *lengths, *cu;
  char *k_out, *v_out;
  float *w_out;
  int32_t *pos_out, *len_out;
  int32_t *list;  // [row][budget]: by slot, the kept entries that are chosen by weight
  int64_t T, k_sb, k_sh, k_st, v_sb, v_sh, v_st;  // (k, v: bytes)
  int64_t w_sb, w_sh, ps_sb, ps_sh, budget, capacity, recent, sink;
  uint2 *state;           // [pass][row]: the smallest kept key so far, how many are wanted of its bin
  uint32_t *ahead;        // [pass][row][slice]: keys of earlier slices that the pass found above
  uint16_t *hist;         // [pass][row][slice][bin]
  int32_t B, Hkv, row16, slices;  // row16: 16-byte chunks of a row
  int32_t sel;                    // workgroups of a launch that select
  int32_t open, early;            // blocks of EV_SLOTS slots that wait for the lists, and after them that do not
};

typedef float ev_f4 __attribute__((ext_vector_type(4), aligned(4)));
typedef int32_t ev_i4 __attribute__((ext_vector_type(4), aligned(4)));

// One row of a call: sequence b, KV head h.  Slot s of the kept entries is entry s below
// `lead`, entry n - kept + s from slot kept - tail on, and else chosen by weight.
struct EvRow {
  int64_t first;
  int32_t n, kept, lead, tail;
  int32_t lo, hi;  // positions lo .. hi - 1 are not protected
  const float *w;
  const int32_t *ps;
};
__device__ __forceinline__ EvRow ev_row(const EvKP &p, int b, int h) {
  EvRow r;
  if (p.cu) {
    const int64_t a = min(max((int64_t)p.cu[b], (int64_t)0), p.T), e = min(max((int64_t)p.cu[b + 1], (int64_t)0), p.T);
    r.first = a;
    r.n = (int32_t)max(e - a, (int64_t)0);
  } else {
    r.first = 0;
    r.n = (int32_t)(p.lengths ? min(max((int64_t)p.lengths[b], (int64_t)0), p.T) : p.T);
  }
  r.kept = (int32_t)min((int64_t)r.n, p.budget);
  r.w = p.weights + (p.cu ? r.first : b * p.w_sb) + h * p.w_sh;
  r.ps = p.positions ? p.positions + b * p.ps_sb + h * p.ps_sh : nullptr;
  // (recent + sink <= budget, so that of n > budget entries the protected ones are apart)
  r.lead = r.n <= r.kept ? r.kept : r.ps ? 0 : (int32_t)p.sink;
  r.tail = r.n <= r.kept || r.ps ? 0 : (int32_t)p.recent;
  r.lo = (int32_t)min(p.sink, (int64_t)INT32_MAX);
  r.hi = r.ps ? (int32_t)max((int64_t)p.pos[b] - p.recent, (int64_t)INT32_MIN) : 0;
  return r;
}
// Entry of slot s where it is not chosen by weight; -1: none.
__device__ __forceinline__ int32_t ev_slot(const EvRow &r, int32_t s) {
  return s < r.lead ? s : s >= r.kept - r.tail && s < r.kept ? r.n - r.kept + s : -1;
}

constexpr int EV_SMALL = 2048, EV_MID = 16384, EV_SLOTS = 64;

// Slots s0 .. s0 + ns - 1 of a row, at most EV_SLOTS, by a workgroup of NT: entries at[]
// (-1: none) of k and v, 16 bytes a lane, four of each in flight; weights and positions.
template <int NT>
__device__ __forceinline__ void ev_copy(const EvKP &p, const EvRow &r, int b, int h, const int32_t *at, int32_t s0,
                                        int32_t ns) {
  const int64_t bh = (int64_t)b * p.Hkv + h;
  if ((int)threadIdx.x < ns) {
    const int32_t i = at[threadIdx.x];
    const int64_t o = bh * p.capacity + s0 + threadIdx.x;
    p.w_out[o] = i < 0 ? 0.f : r.w[i];
    p.pos_out[o] = i < 0 || !r.ps ? i : r.ps[i];
  }
  const char *kb = p.k + (p.cu ? r.first * p.k_st : b * p.k_sb) + h * p.k_sh;
  const char *vb = p.v + (p.cu ? r.first * p.v_st : b * p.v_sb) + h * p.v_sh;
  const int64_t o0 = 16 * (bh * p.capacity + s0) * p.row16;
  const uint32_t r16 = (uint32_t)p.row16, end = (uint32_t)ns * r16;
  for (uint32_t x0 = threadIdx.x; x0 < end; x0 += 4 * NT) {
    uint4 kk[4], vv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t x = x0 + NT * j;
      const int32_t i = x < end ? at[x / r16] : -1;
      const uint32_t ch = x % r16;
      kk[j] = vv[j] = uint4{0, 0, 0, 0};
      if (i >= 0) {
        kk[j] = *(const uint4 *)(kb + i * p.k_st + 16 * ch);
        vv[j] = *(const uint4 *)(vb + i * p.v_st + 16 * ch);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t x = x0 + NT * j;
      if (x < end) {
        *(uint4 *)(p.k_out + o0 + 16 * (int64_t)x) = kk[j];
        *(uint4 *)(p.v_out + o0 + 16 * (int64_t)x) = vv[j];
      }
    }
  }
}

// Block x (row by row) of those that wait for no list.
template <int NT>
__device__ __forceinline__ void ev_early(const EvKP &p, uint32_t x) {
  __shared__ int32_t at[EV_SLOTS];
  const int bh = x / (uint32_t)p.early, blk = p.open + x % (uint32_t)p.early, b = bh / p.Hkv, h = bh % p.Hkv;
  if (bh >= p.B * p.Hkv) return;
  const EvRow r = ev_row(p, b, h);
  const int32_t s0 = blk * EV_SLOTS, ns = (int32_t)min((int64_t)EV_SLOTS, p.capacity - s0);
  if (threadIdx.x < EV_SLOTS) at[threadIdx.x] = ev_slot(r, s0 + threadIdx.x);
  __syncthreads();
  ev_copy<NT>(p, r, b, h, at, s0, ns);
}

__device__ __forceinline__ uint32_t ev_below(uint64_t m) {  // set bits of lanes before this one
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u));
}

// The entries of a row (at most MOST) kept for their weight, in order: list(slot, entry) for
// the slots from `lead` on.  By a workgroup of NT threads, whose wave w holds the keys of up
// to 256 NJ entries from w * seg on: 4 lane .. 4 lane + 3 of each 256.
template <int NT, int MOST, int BITS, bool POS, class List>
__device__ __forceinline__ void ev_choose(const EvRow &r, List list) {
  constexpr int NW = NT / 64, NJ = MOST / (4 * NT), BINS = 1 << BITS, PER = BINS / NT;
  static_assert(PER >= 1 && 4 * NT * NJ == MOST, "a thread has a bin, and the workgroup all keys");
  // a bin's count in COPIES parts, by lane: weights crowd into a few exponents, and lanes
  // that meet in one LDS word wait for each other
  constexpr int COPIES = 4;
  __shared__ __align__(16) uint32_t hist[BINS * COPIES];
  __shared__ uint32_t part[NW][2];
  // after the first digit, the keys of the bin that holds the smallest kept one, where
  // they are this few: what the other digits are of
  constexpr int CAND = 4 * NT;
  __shared__ uint32_t cand[CAND];
  __shared__ uint32_t ncand;
  __shared__ uint32_t found[3];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t n = r.n - r.lead - r.tail;  // entries to choose from: r.lead on
  uint32_t want = (uint32_t)(r.kept - r.lead - r.tail);
  if (want == 0) return;
  const float *wr = r.w + r.lead;
  const int32_t seg = ((n + NT * 4 - 1) / (NT * 4)) * 256;
  const int32_t s0 = w * seg, s1 = min(s0 + seg, n);
  uint32_t key[NJ][4];  // 0: no entry
#pragma unroll
  for (int j = 0; j < NJ; ++j) {  // (every load in flight before the first is used)
    const int32_t c0 = s0 + 256 * j, i = c0 + 4 * lane;
    if (c0 + 256 <= s1) {
      const ev_i4 v = *(const ev_i4 *)(wr + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) key[j][e] = (uint32_t)v[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) key[j][e] = __float_as_uint(wr[min(i + e, n - 1)]);
    }
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int32_t c0 = s0 + 256 * j, i = c0 + 4 * lane;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t k = ev_key(__uint_as_float(key[j][e]));
      if constexpr (POS) {
        const int32_t at = r.ps[min(i + e, n - 1)];
        k = at >= r.lo && at < r.hi ? k : EV_SAFE;
      }
      key[j][e] = k;
    }
    if (c0 + 256 > s1) {
#pragma unroll
      for (int e = 0; e < 4; ++e) key[j][e] = i + e < s1 ? key[j][e] : 0u;
    }
  }
  // kept: keys above thr, and the first `want` of those equal to it
  uint32_t thr = 0;
  int shift = 32;
  uint32_t few = 0;
#pragma unroll 1
  while (shift > 0) {
    const int bits = min(BITS, shift), up = shift;
    shift -= bits;
    for (int i = tid; i < BINS * COPIES / 4; i += NT) ((uint4 *)hist)[i] = uint4{0, 0, 0, 0};
    __syncthreads();
    const uint32_t mask = (1u << bits) - 1u;
    auto count = [&](uint32_t k) {
      atomicAdd(&hist[((k >> shift) & mask) * COPIES + (lane & (COPIES - 1))], 1u);
    };
    if (few > 0) {
      for (uint32_t i = tid; i < few; i += NT)
        if (((cand[i] ^ thr) >> up) == 0u) count(cand[i]);
    } else {
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t k = key[j][e];
          if (k != 0u && (up == 32 || ((k ^ thr) >> (up & 31)) == 0u)) count(k);
        }
    }
    __syncthreads();
    // from the highest bin down, PER bins a thread: where the count reaches `want`
    uint32_t c[PER], incl = 0;
#pragma unroll
    for (int x = 0; x < PER; ++x) {
      const uint4 y = ((const uint4 *)hist)[BINS - 1 - (PER * tid + x)];
      c[x] = y.x + y.y + y.z + y.w;
      incl += c[x];
    }
    const uint32_t mine = incl;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t y = (uint32_t)__shfl_up((int)incl, o, 64);
      if (lane >= o) incl += y;
    }
    if (lane == 63) part[w][0] = incl;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < NW; ++x) incl += x < w ? part[x][0] : 0u;
    uint32_t before = incl - mine;
    if (before < want && want <= incl) {  // (one thread: there are more entries than are wanted)
      int x = 0;
#pragma unroll
      for (int y = 0; y < PER - 1; ++y)
        if (x == y && before + c[y] < want) {
          before += c[y];
          ++x;
        }
      found[0] = (uint32_t)(BINS - 1 - (PER * tid + x));
      found[1] = before;
      found[2] = c[0];
#pragma unroll
      for (int y = 1; y < PER; ++y)
        if (x == y) found[2] = c[y];
      ncand = 0u;
    }
    __syncthreads();
    thr |= found[0] << shift;
    want -= found[1];
    if (up == 32 && found[2] <= (uint32_t)CAND) {
      few = found[2];
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (((key[j][e] ^ thr) >> shift) == 0u && key[j][e] != 0u)
            cand[atomicAdd(&ncand, 1u)] = key[j][e];
      // (in any order: only their number in each bin counts)
      __syncthreads();
    }
    // (part and found are written again after further barriers)
  }
  // what each wave keeps, and from where on
  uint32_t gt = 0, eq = 0;
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      gt += (uint32_t)__popcll(__ballot(key[j][e] > thr));  // (thr is 1 or more)
      eq += (uint32_t)__popcll(__ballot(key[j][e] == thr));
    }
  __syncthreads();
  if (lane == 0) {
    part[w][0] = gt;
    part[w][1] = eq;
  }
  __syncthreads();
  uint32_t g = 0, q = 0;  // above thr, and equal to it, in the waves before
#pragma unroll
  for (int y = 0; y < NW; ++y) {
    g += y < w ? part[y][0] : 0u;
    q += y < w ? part[y][1] : 0u;
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    uint64_t any = 0;
    uint32_t gl = g;  // above thr, of earlier lanes (and, below, of this lane's earlier entries)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint64_t m = __ballot(key[j][e] > thr);
      gl += ev_below(m);
      g += (uint32_t)__popcll(m);
      any |= __ballot(key[j][e] == thr);
    }
    const int32_t i = s0 + 4 * lane + r.lead + 256 * j;
    if (any == 0) {
      int32_t slot = r.lead + (int32_t)(gl + min(q, want));
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (key[j][e] > thr) list(slot++, i + e);
      continue;
    }
    uint32_t ql = q;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint64_t m = __ballot(key[j][e] == thr);
      ql += ev_below(m);
      q += (uint32_t)__popcll(m);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool above = key[j][e] > thr, same = key[j][e] == thr;
      if (above || (same && ql < want)) list(r.lead + (int32_t)(gl + min(ql, want)), i + e);
      gl += above ? 1u : 0u;
      ql += same ? 1u : 0u;
    }
  }
}

// (Two caches of 660 and 740 entries of 8 heads cut to 256: 9.4 us, the search's barriers.)
template <bool POS>
__global__ __launch_bounds__(256) void evict_small_kernel(EvKP p, int32_t parts) {
  __shared__ int32_t at[EV_SLOTS];
  const int part = blockIdx.x % parts, bh = blockIdx.x / parts, b = bh / p.Hkv, h = bh % p.Hkv;
  const EvRow r = ev_row(p, b, h);
  const int32_t s0 = part * EV_SLOTS, ns = (int32_t)min((int64_t)EV_SLOTS, p.capacity - s0);
  if (threadIdx.x == 0 && h == 0 && part == 0) p.len_out[b] = r.kept;
  if (threadIdx.x < EV_SLOTS) at[threadIdx.x] = ev_slot(r, s0 + threadIdx.x);
  __syncthreads();
  if (s0 + ns > r.lead && s0 < r.kept - r.tail)  // (some slot is chosen by weight)
    ev_choose<256, EV_SMALL, 8, POS>(r, [&](int32_t s, int32_t i) {
      if (s >= s0 && s < s0 + ns) at[s - s0] = i;
    });
  __syncthreads();
  ev_copy<256>(p, r, b, h, at, s0, ns);
}

// (One cache of 16000 entries of 8 heads cut to 4096, with the copies: 20 us.)
template <bool POS>
__global__ __launch_bounds__(1024) void evict_select_kernel(EvKP p) {
  if ((int)blockIdx.x >= p.sel) {
    ev_early<1024>(p, blockIdx.x - p.sel);
    return;
  }
  const int b = blockIdx.x / p.Hkv, h = blockIdx.x % p.Hkv;
  const EvRow r = ev_row(p, b, h);
  if (h == 0 && threadIdx.x == 0) p.len_out[b] = r.kept;
  if (r.n <= r.kept) return;
  int32_t *list = p.list + (int64_t)blockIdx.x * p.budget;
  ev_choose<1024, EV_MID, 11, POS>(r, [&](int32_t s, int32_t i) { list[s] = i; });
}

// A slice of a row of a long cache: pass 0 counts the first digits; passes 1 and 2 find the
// bin of the smallest kept key in the counts of the pass before and count the next digit
// of the keys in it; pass 3 finds the key and lists what is kept of the slice.
constexpr int EV_BINS = 2048;
template <int PASS, bool POS>
__global__ __launch_bounds__(256) void evict_digit_kernel(EvKP p) {
  if ((int)blockIdx.x >= p.sel) {  // (this launch's share of them)
    ev_early<256>(p, blockIdx.x - p.sel + PASS * (gridDim.x - p.sel));
    return;
  }
  constexpr int COPIES = 4;  // (see ev_choose)
  __shared__ __align__(16) uint32_t hist[PASS < 3 ? EV_BINS * COPIES : 4];
  __shared__ uint32_t part[4][2];
  __shared__ uint32_t found[2];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int row = blockIdx.x / p.slices, slice = blockIdx.x % p.slices, b = row / p.Hkv, h = row % p.Hkv;
  const int64_t rows = (int64_t)p.B * p.Hkv;
  const EvRow r = ev_row(p, b, h);
  if (PASS == 0 && h == 0 && slice == 0 && tid == 0) p.len_out[b] = r.kept;
  const int32_t n = r.n - r.lead - r.tail;  // entries to choose from: r.lead on
  uint32_t want = (uint32_t)(r.kept - r.lead - r.tail);
  if (want == 0) return;
  const int32_t per = ((n + p.slices * 256 - 1) / (p.slices * 256)) * 256;
  const int32_t i0 = min(slice * per, n), i1 = min(i0 + per, n);
  const float *wr = r.w + r.lead;
  // the first 4096 weights of the slice (all of it, mostly) are on their way meanwhile
  float pre[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int32_t i = i0 + 1024 * j + 4 * tid;
    if (i + 4 <= i1) {
      const ev_f4 x = *(const ev_f4 *)(wr + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) pre[j][e] = x[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) pre[j][e] = i + e < i1 ? wr[i + e] : 0.f;
    }
  }
  uint32_t thr = 0, ahead = 0, same_ahead = 0;  // ahead: kept keys of earlier slices
  if constexpr (PASS > 0) {
    if constexpr (PASS > 1) {
      const uint2 st = p.state[(PASS - 1) * rows + row];
      thr = st.x;
      want = st.y;
    }
    // eight bins a thread, from the highest down, over all slices and over the earlier ones
    const uint16_t *hp = p.hist + (((PASS - 1) * rows + row) * p.slices) * EV_BINS + EV_BINS - 8 * (tid + 1);
    uint32_t all[8], bef[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) all[x] = bef[x] = 0u;
    for (int sl0 = 0; sl0 < p.slices; sl0 += 16) {
      uint4 v[16];
#pragma unroll
      for (int y = 0; y < 16; ++y) v[y] = *(const uint4 *)(hp + (int64_t)min(sl0 + y, p.slices - 1) * EV_BINS);
#pragma unroll
      for (int y = 0; y < 16; ++y) {
        const uint32_t u[4] = {v[y].x, v[y].y, v[y].z, v[y].w};
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const uint32_t c = x & 1 ? u[x >> 1] >> 16 : u[x >> 1] & 0xffffu;
          all[x] += sl0 + y < p.slices ? c : 0u;
          bef[x] += sl0 + y < slice ? c : 0u;
        }
      }
    }
    uint32_t mine = 0;
#pragma unroll
    for (int x = 0; x < 8; ++x) mine += all[x];
    uint32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t y = (uint32_t)__shfl_up((int)incl, o, 64);
      if (lane >= o) incl += y;
    }
    if (lane == 63) part[w][0] = incl;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 4; ++x) incl += x < w ? part[x][0] : 0u;
    uint32_t before = incl - mine;
    if (before < want && want <= incl) {  // (one thread: there are more entries than are wanted)
      int bin = 8 * (tid + 1);  // counted from the top
#pragma unroll
      for (int x = 0; x < 8; ++x) {  // lowest bin of the eight last
        const int y = 7 - x;
        if (bin == 8 * (tid + 1) && before + all[y] >= want) bin = 8 * tid + x;
        if (bin == 8 * (tid + 1)) before += all[y];
      }
      found[0] = (uint32_t)bin;
      found[1] = before;
    }
    __syncthreads();
    const int top = (int)found[0];  // bins above it: 0 .. top - 1 from the top
    uint32_t up = 0, eq = 0;
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int at = 8 * tid + 7 - x;  // bin x of the thread, from the top
      up += at < top ? bef[x] : 0u;
      eq += at == top ? bef[x] : 0u;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      up += (uint32_t)__shfl_xor((int)up, o, 64);
      eq += (uint32_t)__shfl_xor((int)eq, o, 64);
    }
    if (lane == 0) {
      part[w][0] = up;
      part[w][1] = eq;
    }
    __syncthreads();
    ahead = part[0][0] + part[1][0] + part[2][0] + part[3][0];
    same_ahead = part[0][1] + part[1][1] + part[2][1] + part[3][1];
    constexpr int SHIFT = PASS == 1 ? 21 : PASS == 2 ? 10 : 0;
    thr |= (uint32_t)(EV_BINS - 1 - top) << SHIFT;
    want -= found[1];
    if constexpr (PASS < 3) {
      if (tid == 0) p.ahead[(PASS * rows + row) * p.slices + slice] = ahead;
      if (tid == 0 && slice == 0) p.state[PASS * rows + row] = uint2{thr, want};
    } else {
      for (int x = 1; x < 3; ++x) ahead += p.ahead[(x * rows + row) * p.slices + slice];
    }
  }
  auto keys = [&](int j, uint32_t (&k)[4]) {  // of the entries of step j; 0: none
    const int32_t i = i0 + 1024 * j + 4 * tid;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = j == 0 ? pre[0][e] : j == 1 ? pre[1][e] : j == 2 ? pre[2][e] : j == 3 ? pre[3][e]
                      : i + e < i1 ? wr[i + e] : 0.f;
      k[e] = i + e < i1 ? ev_key(x) : 0u;
      if constexpr (POS) {
        const int32_t at = i + e < i1 ? r.ps[i + e] : 0;
        if (i + e < i1 && !(at >= r.lo && at < r.hi)) k[e] = EV_SAFE;
      }
    }
  };
  const int steps = (i1 - i0 + 1023) / 1024;
  if constexpr (PASS < 3) {
    constexpr int SHIFT = PASS == 0 ? 21 : PASS == 1 ? 10 : 0;  // of the digit counted
    for (int i = tid; i < EV_BINS * COPIES / 4; i += 256) ((uint4 *)hist)[i] = uint4{0, 0, 0, 0};
    __syncthreads();
    auto add = [&](int j) {
      uint32_t k[4];
      keys(j, k);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (k[e] != 0u && (PASS == 0 || ((k[e] ^ thr) >> (PASS == 1 ? 21 : 10)) == 0u))
          atomicAdd(&hist[((k[e] >> SHIFT) & (PASS == 2 ? 1023u : 2047u)) * COPIES + (lane & (COPIES - 1))], 1u);
    };
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < steps) add(j);
    for (int j = 4; j < steps; ++j) add(j);
    __syncthreads();
    uint16_t *o = p.hist + ((PASS * rows + row) * p.slices + slice) * EV_BINS + 8 * tid;
    uint32_t c[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const uint4 v = ((const uint4 *)hist)[8 * tid + x];
      c[x] = v.x + v.y + v.z + v.w;
    }
    *(uint4 *)o = uint4{c[0] | c[1] << 16, c[2] | c[3] << 16, c[4] | c[5] << 16, c[6] | c[7] << 16};
  } else {
    int32_t *list = p.list + (int64_t)row * p.budget;
    uint32_t g = ahead, q = same_ahead;  // above thr, and equal to it, up to here
    __syncthreads();                     // (part is read)
    auto put = [&](int j) {
      const int32_t i = i0 + 1024 * j + 4 * tid;
      uint32_t k[4];
      keys(j, k);
      uint32_t gt = 0, eq = 0;  // the wave's
      uint32_t gl = 0, ql = 0;  // of earlier lanes
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t mg = __ballot(k[e] > thr), me = __ballot(k[e] == thr);
        gt += (uint32_t)__popcll(mg);
        eq += (uint32_t)__popcll(me);
        gl += ev_below(mg);
        ql += ev_below(me);
      }
      if (lane == 0) {
        part[w][0] = gt;
        part[w][1] = eq;
      }
      __syncthreads();
      gl += g;
      ql += q;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t a = part[x][0], c = part[x][1];
        gl += x < w ? a : 0u;
        ql += x < w ? c : 0u;
        g += a;
        q += c;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool above = k[e] > thr, same = k[e] == thr;
        if (above || (same && ql < want)) list[r.lead + (int32_t)(gl + min(ql, want))] = r.lead + i + e;
        gl += above ? 1u : 0u;
        ql += same ? 1u : 0u;
      }
      __syncthreads();
    };
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < steps) put(j);
    for (int j = 4; j < steps; ++j) put(j);
  }
}

__global__ __launch_bounds__(256) void evict_copy_kernel(EvKP p) {
  __shared__ int32_t at[EV_SLOTS];
  const int bh = blockIdx.x / (uint32_t)p.open, blk = blockIdx.x % (uint32_t)p.open, b = bh / p.Hkv, h = bh % p.Hkv;
  const EvRow r = ev_row(p, b, h);
  const int32_t s0 = blk * EV_SLOTS, ns = (int32_t)min((int64_t)EV_SLOTS, p.capacity - s0);
  if (threadIdx.x < EV_SLOTS) {
    const int32_t s = s0 + threadIdx.x;
    at[threadIdx.x] = s >= r.lead && s < r.kept - r.tail ? p.list[(int64_t)bh * p.budget + s] : ev_slot(r, s);
  }
  __syncthreads();
  ev_copy<256>(p, r, b, h, at, s0, ns);
}

static int ev_check(const la_evict_args *a) {
  LA_REQUIRE(a != nullptr, "la_evict_kv: null args");
  LA_REQUIRE(a->B > 0 && a->Hkv > 0 && a->T >= 0 && a->D > 0, "la_evict_kv: sizes must be positive");
  LA_REQUIRE(a->esize == 1 || a->esize == 2 || a->esize == 4, "la_evict_kv: esize");
  LA_REQUIRE(a->D * a->esize % 16 == 0, "la_evict_kv: rows must be whole 16-byte chunks");
  LA_REQUIRE(a->budget > 0 && a->recent >= 0 && a->sink >= 0 && a->recent + a->sink <= a->budget,
             "la_evict_kv: sink + recent must fit a positive budget");
  LA_REQUIRE(a->capacity >= a->budget, "la_evict_kv: capacity must be at least budget");
  LA_REQUIRE(a->T < ((int64_t)1 << 30) && a->capacity < ((int64_t)1 << 30) && a->B * a->Hkv < ((int64_t)1 << 24) &&
                 a->B * a->Hkv * ceil_div(a->capacity, EV_SLOTS) < ((int64_t)1 << 31),
             "la_evict_kv: too many entries");
  LA_REQUIRE(!(a->cu && a->lengths), "la_evict_kv: lengths are for batched calls");
  LA_REQUIRE(!(a->cu && a->positions), "la_evict_kv: positions are for batched calls");
  LA_REQUIRE(!a->positions || a->pos, "la_evict_kv: positions need pos");
  return LA_OK;
}

}  // namespace la

namespace la {

// Workspace: the lists, and for long caches what the passes hand on.
struct EvPlan {
  int64_t slices = 0;
  size_t list = 0, state = 0, ahead = 0, hist = 0, bytes = 0;
};
static EvPlan ev_plan(const la_evict_args *a) {
  EvPlan pl;
  if (a->T <= EV_SMALL) return pl;
  const size_t rows = (size_t)(a->B * a->Hkv);
  size_t at = 0;
  auto take = [&](size_t n) { const size_t o = at; at += (n + 255) / 256 * 256; return o; };
  pl.list = take(rows * (size_t)a->budget * sizeof(int32_t));
  if (a->T > EV_MID) {
    // slices of 4096 entries, 16 of them at most (each reads all their counts), and none
    // of more than a 16-bit count holds
    pl.slices = std::max(std::min(ceil_div(a->T, 4096), (int64_t)16), ceil_div(a->T, 65024));
    pl.state = take(3 * rows * sizeof(uint2));
    pl.ahead = take(3 * rows * (size_t)pl.slices * sizeof(uint32_t));
    pl.hist = take(3 * rows * (size_t)pl.slices * EV_BINS * sizeof(uint16_t));
  }
  pl.bytes = at;
  return pl;
}

}  // namespace la

extern "C" size_t la_evict_kv_workspace(const la_evict_args *a) {
  if (la::ev_check(a) != LA_OK) return 0;
  return la::ev_plan(a).bytes;
}

extern "C" int la_evict_kv(const la_evict_args *a, void *stream) {
  using namespace la;
  if (int rc = ev_check(a)) return rc;
  LA_REQUIRE(a->k_out && a->v_out && a->w_out && a->pos_out && a->len_out &&
                 (a->T == 0 || (a->k && a->v && a->weights)),
             "la_evict_kv: null pointer");
  const int64_t es = a->esize;
  auto ok = [&](const void *x, int64_t sb, int64_t sh, int64_t st) {
    return (uintptr_t)x % 16 == 0 && (a->cu || a->B == 1 || sb * es % 16 == 0) && (a->Hkv == 1 || sh * es % 16 == 0) &&
           (a->T <= 1 || st * es % 16 == 0);
  };
  LA_REQUIRE(ok(a->k, a->k_sb, a->k_sh, a->k_st) && ok(a->v, a->v_sb, a->v_sh, a->v_st) &&
                 (uintptr_t)a->k_out % 16 == 0 && (uintptr_t)a->v_out % 16 == 0,
             "la_evict_kv: rows of k and v must be 16-byte aligned");
  const EvPlan pl = ev_plan(a);
  if (pl.bytes > 0 && (!a->workspace || a->ws_bytes < (int64_t)pl.bytes))
    return fail(LA_ERR_WORKSPACE, "la_evict_kv: workspace %lld < %lld bytes", (long long)a->ws_bytes,
                (long long)pl.bytes);
  LA_REQUIRE(pl.bytes == 0 || (uintptr_t)a->workspace % 256 == 0, "la_evict_kv: workspace alignment");
  EvKP p{};
  p.k = (const char *)a->k; p.v = (const char *)a->v; p.weights = a->weights;
  p.positions = a->positions; p.pos = a->pos; p.lengths = a->lengths; p.cu = a->cu;
  p.k_out = (char *)a->k_out; p.v_out = (char *)a->v_out;
  p.w_out = a->w_out; p.pos_out = a->pos_out; p.len_out = a->len_out;
  char *ws = (char *)a->workspace;
  p.list = (int32_t *)(ws + pl.list); p.state = (uint2 *)(ws + pl.state);
  p.ahead = (uint32_t *)(ws + pl.ahead); p.hist = (uint16_t *)(ws + pl.hist); p.slices = (int32_t)pl.slices;
  p.T = a->T;
  p.k_sb = a->k_sb * es; p.k_sh = a->k_sh * es; p.k_st = a->k_st * es;
  p.v_sb = a->v_sb * es; p.v_sh = a->v_sh * es; p.v_st = a->v_st * es;
  p.w_sb = a->w_sb; p.w_sh = a->w_sh; p.ps_sb = a->ps_sb; p.ps_sh = a->ps_sh;
  p.budget = a->budget; p.capacity = a->capacity; p.recent = a->recent; p.sink = a->sink;
  p.B = (int32_t)a->B; p.Hkv = (int32_t)a->Hkv; p.row16 = (int32_t)(a->D * es / 16);
  hipStream_t st = (hipStream_t)stream;
  const uint32_t rows = (uint32_t)(a->B * a->Hkv);
  const int32_t parts = (int32_t)ceil_div(a->capacity, EV_SLOTS);
  if (a->T <= EV_SMALL) {
    LA_REQUIRE(grid_fits((int64_t)rows * parts, 256), "la_evict_kv: too many slots");
    if (a->positions) evict_small_kernel<true><<<rows * (uint32_t)parts, 256, 0, st>>>(p, parts);
    else evict_small_kernel<false><<<rows * (uint32_t)parts, 256, 0, st>>>(p, parts);
    LA_LAUNCHED();
    return LA_OK;
  }
  // (of a row of more than budget entries; one of fewer has no chosen slots at all)
  p.open = (int32_t)ceil_div(a->budget - (a->positions ? 0 : a->recent), EV_SLOTS);
  p.early = parts - p.open;
  const uint32_t early = rows * (uint32_t)p.early;
  LA_REQUIRE(grid_fits((int64_t)rows * p.open, 256), "la_evict_kv: too many slots");
  if (a->T <= EV_MID) {
    LA_REQUIRE(grid_fits((int64_t)rows + early, 1024), "la_evict_kv: too many slots");
    p.sel = (int32_t)rows;
    if (a->positions) evict_select_kernel<true><<<rows + early, 1024, 0, st>>>(p);
    else evict_select_kernel<false><<<rows + early, 1024, 0, st>>>(p);
  } else {
    p.sel = (int32_t)(rows * (uint32_t)pl.slices);
    const uint32_t grid = (uint32_t)p.sel + (early + 3) / 4;
    LA_REQUIRE(grid_fits(grid, 256), "la_evict_kv: too many entries");
    if (a->positions) {
      evict_digit_kernel<0, true><<<grid, 256, 0, st>>>(p);
      evict_digit_kernel<1, true><<<grid, 256, 0, st>>>(p);
      evict_digit_kernel<2, true><<<grid, 256, 0, st>>>(p);
      evict_digit_kernel<3, true><<<grid, 256, 0, st>>>(p);
    } else {
      evict_digit_kernel<0, false><<<grid, 256, 0, st>>>(p);
      evict_digit_kernel<1, false><<<grid, 256, 0, st>>>(p);
      evict_digit_kernel<2, false><<<grid, 256, 0, st>>>(p);
      evict_digit_kernel<3, false><<<grid, 256, 0, st>>>(p);
    }
  }
  LA_LAUNCHED();
  if (p.open > 0) {
    evict_copy_kernel<<<rows * (uint32_t)p.open, 256, 0, st>>>(p);
    LA_LAUNCHED();
  }
  return LA_OK;
}
