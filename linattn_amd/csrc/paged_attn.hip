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

// The blocks of a piece: number i of j0 .. j1 - 1 is block i + turn of the tile, and behind its last of
// n_all comes its first.  A tile's blocks begin where the workgroups of its KV head are at that time, if
// all take equally long for a block: they read the same keys at about the same time, of which
// L2 then has what another has read (8192 tokens behind 24576: 67 % of the reads in place of 28,
// 3.67 ms in place of 3.87).
struct PaBlocks {
  int32_t j0, j1, turn, n_all;
  __device__ __forceinline__ int at(int i) const { return i + turn < n_all ? i + turn : i + turn - n_all; }
};

// Rows r_first + i of which bit i of `bad` is set, whose results are not finite: those with an
// infinity or NaN of V among what their blocks of BS keys (up to the tile's block `top`) held and they do
// not see are done again, key by key, in fp32 (ALL: and the others); the others stand, but in
// fp16 (LOST), where a weight below 2^-40 of the row's largest is 0 and its product with an
// infinity NaN: a dim's first keys with NaN and either infinity say what it is for each row.
// (What a block holds past the last key is that key again.)
template <class E, int D, int BS, int NR, bool KV8, bool ALL, bool LOST, bool WAVES>
__device__ void pa_again(const PaKP &p, int b, const PaSeq &sq, int kvh, int64_t part, int r_tile, int r_first, uint32_t bad,
                         const PaBlocks &blocks, int top) {
  const int lane = threadIdx.x & 63, G = p.G;
  const int32_t *pages = p.page_table + b * p.pt_sb;
  const PaCache<E, KV8> K{p.k, p.k_scale, p.s_stride, D}, V{p.v, p.v_scale, p.s_stride, D};
  auto row = [&](int key) { return pa_row(p, pages, min(key, sq.lk - 1), kvh); };
  constexpr int N = D / 64;
  const float inf = __int_as_float(0x7f800000);
  auto in_part = [&](int r, int d) { return part * D + (WAVES ? pa_in_part<D>(r - r_tile, d) : (int64_t)(r - r_tile) * D + d); };
  int32_t at[3][N];  // of dim lane + 64 x
#pragma unroll
  for (int x = 0; x < N; ++x) at[0][x] = at[1][x] = at[2][x] = INT32_MAX;
  if constexpr (LOST) {
    for (int i = blocks.j0; i < blocks.j1; ++i) {
      const int j = blocks.at(i);
      if (j > top) continue;
      for (int key = j * BS; key < min(j * BS + BS, sq.lk); ++key) {
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
  }
  wait_vmcnt<0>();  // (stores over those)
#pragma unroll 1
  for (int r = r_first; r < r_first + NR; ++r) {
    if (!((bad >> (r - r_first)) & 1u)) continue;
    const int t = r / G, h = kvh * G + r % G;
    const int lim = p.causal ? min(sq.lk - 1, sq.lk - sq.lq + t) : sq.lk - 1;
    bool met = ALL;
    for (int i = blocks.j0; i < blocks.j1 && !ALL; ++i) {
      const int j = blocks.at(i);
      if (j > top || j * BS + BS - 1 <= lim) continue;
      for (int key = max(j * BS, lim + 1); key < j * BS + BS; ++key)
        for (int d = lane; d < D; d += 64) met = met || !(fabsf(V.at(row(key), d)) < inf);
    }
    if (__ballot(met) == 0) {
#pragma unroll
      for (int x = 0; x < N; ++x) {
        const bool up = at[1][x] <= lim, down = at[2][x] <= lim, nan = at[0][x] <= lim || (up && down);
        if (!nan && !up && !down) continue;
        const float y = nan ? __int_as_float(0x7fc00000) : up ? inf : -inf;
        if (part >= 0) p.ws_acc[in_part(r, lane + 64 * x)] = y;
        else store_from_f32(p.out, pa_out_at(p, b, sq, t, h) + lane + 64 * x, p.out_dt, y);
      }
      continue;
    }
    const E *q = (const E *)p.q + pa_q_at(p, b, sq, t, h);
    float m = pa_ninf(), l = 0.f, acc[N];
#pragma unroll
    for (int x = 0; x < N; ++x) acc[x] = 0.f;
    for (int i = blocks.j0; i < blocks.j1; ++i) {
      const int key0 = blocks.at(i) * BS, n = min(BS, lim + 1 - key0);  // keys of the block that it sees
      if (n <= 0) continue;
      const uint32_t kr = row(key0 + min(lane, n - 1));
      float s = 0.f;
      for (int d = 0; d < D; ++d) s = __builtin_fmaf((float)q[d], K.at(kr, d), s);
      s = lane < n ? s * p.qscale : pa_ninf();
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
      for (int y = 0; y < n; ++y) {
        const float w = __shfl(pr, y, 64);
        const uint32_t vr = __shfl((int)kr, y, 64);
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
      for (int x = 0; x < N; ++x) p.ws_acc[in_part(r, lane + 64 * x)] = acc[x];
      continue;
    }
    const int64_t o = pa_out_at(p, b, sq, t, h);
#pragma unroll
    for (int x = 0; x < N; ++x) store_from_f32(p.out, o + lane + 64 * x, p.out_dt, l == 0.f ? 0.f : acc[x] / l);
    if (p.lse && lane == 0) p.lse[pa_lse_at(p, b, sq, t, h)] = l == 0.f ? pa_ninf() : (m + __log2f(l)) * PA_LN2;
  }
}

// A workgroup's way along its stretch.  It lies in LDS, and the call's arguments are read anew
// (pa_args) at either end of a piece, so that nothing of it takes registers in between.
struct PaWalk {
  PaStretch s;
  PaSeq seq;
  int64_t a, step;  // (of the sequence's tiles)
  int64_t since;    // where the tile begins, from where its first workgroup's stretch does
  int32_t n;
};

// The lane's number, of which nothing is worked out ahead (it would take registers, or memory, from
// there on).
__device__ __forceinline__ int pa_lane() {
  int x = threadIdx.x & 63;
  asm volatile("" : "+v"(x));
  return x;
}

typedef const __attribute__((address_space(4))) PaKP PaArgs;
__device__ __forceinline__ const PaKP &pa_args() {
  PaArgs *x = (PaArgs *)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(x));
  return *(const PaKP *)x;
}

// The stretch's beginning, by every wave; false: there is none.
template <int R, bool FEW>
__device__ __forceinline__ bool pa_begin(PaWalk *walk) {
  const PaKP &p = pa_args();
  PaWalk w;
  PaTiles t;
  w.s = pa_stretch<R, FEW>(p, blockIdx.x / (uint32_t)p.Hkv, w.seq, t);
  if (w.s.left == 0) {
    if (threadIdx.x == 0) p.ws_join[blockIdx.x] = int4{0, 0, 0, 0};
    return false;
  }
  w.a = t.a;
  w.step = t.step;
  w.n = t.n;
  w.since = w.s.off == 0 ? 0 : w.s.pos - pa_div(w.s.pos, w.s.line.quota) * w.s.line.quota;
  if (threadIdx.x == 0) *walk = w;
  __syncthreads();
  return true;
}

// The next tile of the stretch, or the join's note of the tile that is left open (false: the stretch
// is done).  By every wave.
template <int R, bool FEW>
__device__ __forceinline__ bool pa_next(PaWalk *walk) {
  const PaKP &p = pa_args();
  PaWalk w = *walk;
  lds_barrier();  // (every wave has read it)
  const int64_t cost = w.a + w.step * (w.s.i + 1), upto = min(cost, w.s.off + w.s.left);
  w.s.left -= upto - w.s.off;
  const bool more = __builtin_amdgcn_readfirstlane(w.s.left > 0);
  if (threadIdx.x < 64) {
    const int64_t own = blockIdx.x / (uint32_t)p.Hkv - w.s.line.first;
    if (!more) {
      const int parts = w.s.off == 0 && upto < cost ? (int)(pa_div(w.s.pos + cost - 1, w.s.line.quota) - own) + 1 : 0;
      if (threadIdx.x == 0) p.ws_join[blockIdx.x] = int4{w.s.b, w.s.i, parts, w.s.few ? 1 + (int)own : 0};
    } else {
      w.s.off = 0;
      w.s.pos += cost;
      w.since = w.s.pos - own * w.s.line.quota;
      if (++w.s.i >= w.n) {  // the next sequence that has tiles in the line (of a padded batch most may have none)
        w.s.i = 0;
        for (int b0 = w.s.b + 1; b0 < p.B; b0 += 64) {
          const int b = b0 + (int)threadIdx.x;
          const PaSeq seq = pa_seq(p, min(b, p.B - 1));
          const PaTiles t = pa_tiles<R, FEW>(p, seq, w.s.few);
          const uint64_t there = __ballot(b < p.B && t.n > 0);
          if (there == 0) continue;
          const int at = __ffsll((unsigned long long)there) - 1;
          w.s.b = b0 + at;
          w.seq.lq = __builtin_amdgcn_readlane(seq.lq, at);
          w.seq.lk = __builtin_amdgcn_readlane(seq.lk, at);
          w.seq.q0 = pa_lane_value(seq.q0, at);
          w.a = pa_lane_value(t.a, at);
          w.n = __builtin_amdgcn_readlane(t.n, at);
          break;
        }
      }
      if (threadIdx.x == 0) *walk = w;
    }
  }
  __syncthreads();
  return more;
}

// The piece that the walk is at, in scalar registers: rows r0 .. of a sequence, and which of its
// blocks of BS keys.
struct PaPiece {
  PaSeq sq;
  int32_t b, r0, kvh, mixed;
  PaBlocks blocks;
  int64_t part;  // (-1: the whole tile)
};
template <int R, int BS, bool TURN>
__device__ __forceinline__ PaPiece pa_piece(const PaKP &p, const PaWalk *walk) {
  asm volatile("" ::: "memory");
  PaWalk w = *walk;
  PaPiece x;
  x.sq.lq = __builtin_amdgcn_readfirstlane(w.seq.lq);
  x.sq.lk = __builtin_amdgcn_readfirstlane(w.seq.lk);
  x.sq.q0 = pa_uniform(w.seq.q0);
  x.b = __builtin_amdgcn_readfirstlane(w.s.b);
  x.r0 = __builtin_amdgcn_readfirstlane(w.s.i) * R;
  x.kvh = (int)(blockIdx.x % (uint32_t)p.Hkv);
  x.mixed = __builtin_amdgcn_readfirstlane(w.s.mixed);
  const int last = (min(x.r0 + R, x.sq.lq * p.G) - 1) / p.G;  // its last query
  const int lim = p.causal ? x.sq.lk - x.sq.lq + last : x.sq.lk - 1;
  const int n_all = lim < 0 ? 0 : lim / BS + 1;
  const int64_t cost = w.a + w.step * (w.s.i + 1), upto = min(cost, w.s.off + w.s.left);
  x.blocks.n_all = __builtin_amdgcn_readfirstlane(n_all);
  x.blocks.j0 = x.blocks.turn = 0;
  x.blocks.j1 = x.blocks.n_all;
  if (w.s.off > 0) x.blocks.j0 = __builtin_amdgcn_readfirstlane(pa_blocks(n_all, w.s.off, cost));
  if (upto < cost) x.blocks.j1 = __builtin_amdgcn_readfirstlane(pa_blocks(n_all, upto, cost));
  if (TURN && w.since > 0) {
    const double turns = (double)w.since / (double)cost;
    x.blocks.turn = __builtin_amdgcn_readfirstlane(max(0, min((int)((turns - floor(turns)) * n_all), n_all - 1)));
  }
  x.part = pa_uniform(w.s.off == 0 && upto == cost ? -1 : pa_part(p, blockIdx.x / (uint32_t)p.Hkv - w.s.line.first, x.kvh, w.s.off == 0, w.s.few));
  return x;
}

// The cache's rows of a wave's sixteen keys of each block of 64: pages of whole sixteens (EVEN):
// of block jb + lane, the first of the sixteen; else of block jb + lane / 16, key lane % 16 of them.
template <bool EVEN>
struct PaRows {
  static constexpr int SPAN = EVEN ? 64 : 4;
  const int32_t *pages;
  uint32_t rows;
  int jb, key0, last;  // first key of the wave's sixteen in a block; the sequence's last
  __device__ __forceinline__ void look(const PaKP &p, int kvh, int j) {
    jb = j;
    const int lane = pa_lane();
    const int key = EVEN ? (j + lane) * DA_BS + key0 : (j + lane / 16) * DA_BS + key0 + lane % 16;
    rows = pa_row(p, pages, min(key, last), kvh);
    settle(rows);
  }
  // EVEN: the first row of block j's sixteen, and how many keys there are behind it
  __device__ __forceinline__ uint32_t first(int j) const { return (uint32_t)__builtin_amdgcn_readlane((int)rows, j - jb); }
  __device__ __forceinline__ int behind(int j) const { return last - min(j * DA_BS + key0, last); }
  // this lane's row for key rr (keys past the last: that again)
  __device__ __forceinline__ uint32_t of(int j, int rr) const {
    if constexpr (EVEN) return first(j) + min(rr, behind(j));
    else return (uint32_t)__shfl((int)rows, (j - jb) * 16 + rr, 64);
  }
  // Sixteen rows of RB bytes each of block j into LDS at `to`, 16-byte chunk c of row r at c ^ swz(r)
  // (swz takes the same values for rows PER apart): 64 lanes x 16 bytes a load.
  template <int RB, int PER, class Swz>
  __device__ __forceinline__ void load(const void *pool, int j, uint32_t to, int lane, Swz swz) const {
    constexpr int CH = RB / 16, RP = 64 / CH, NX = 16 / RP;
    if constexpr (EVEN) {
      const int n = behind(j);
      const char *base = (const char *)pool + (uint64_t)first(j) * RB;
      if (n >= 15) {
#pragma unroll
        for (int x = 0; x < NX; ++x) {
          constexpr int STEP = PER / RP > 0 ? PER / RP : 1;  // loads after which the offsets come again
          const int rr = RP * (x % STEP) + lane / CH;
          asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"((uint32_t)(rr * RB + 16 * ((lane % CH) ^ swz(rr)))),
                       "s"(base + RP * (x - x % STEP) * RB), "{m0}"(to + x * 1024) : "memory");
        }
      } else {
        lane = pa_lane();
#pragma unroll
        for (int x = 0; x < NX; ++x) {
          const int rr = RP * x + lane / CH;
          asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"((uint32_t)(min(rr, n) * RB + 16 * ((lane % CH) ^ swz(rr)))),
                       "s"(base), "{m0}"(to + x * 1024) : "memory");
        }
      }
    } else {
#pragma unroll
      for (int x = 0; x < NX; ++x) {
        const int rr = RP * x + lane / CH;
        const char *src = (const char *)pool + (uint64_t)of(j, rr) * RB + 16 * ((lane % CH) ^ swz(rr));
        asm volatile("global_load_lds_dwordx4 %0, off" ::"v"(src), "{m0}"(to + x * 1024) : "memory");
      }
    }
  }
};

// Four codes as two pairs of bf16 or fp16 (exactly).
template <class T>
__device__ __forceinline__ uint2 pa_widen(uint32_t codes) {
  if constexpr (std::is_same<T, DaBf16>::value)
    return uint2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.f, true))};
  else
    return uint2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.f, true))};
}

// 16 x 16 += (16 x 16) (16 x 16)
template <class T>
__device__ __forceinline__ f32x4 pa_mfma16(s16x4 a, s16x4 b, f32x4 c) {
  typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
  if constexpr (std::is_same<T, DaBf16>::value) return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
}

// Of a CU's three workgroups each is preferred for a block in turn: else the one that came first is, and
// they end one after the other (8192 tokens behind 24576, equal stretches: after 2.87, 3.23 and
// 3.81 ms).  In six blocks the first is preferred to both others once, the second twice and the third
// three times, for which all three end at the same time (3.32, 3.33 and 3.33 ms on the mean, as often as one
// another 3.24, 3.33, 3.43): that call 3.34 ms (3.37), chunks of four prompts 225 us (227), tokens over fp8
// caches 136 (139).  Where single tokens lie beside chunks the third holds the tokens, which would come
// first: as often as one another there (243 us, 250 otherwise).
struct PaTurns {
  uint32_t order;  // two bits a block
  __device__ __forceinline__ PaTurns(int third, bool mixed, int i) {
    constexpr uint32_t A = 0x112, B = 0x648, C = 0x8a5, X = 0x924, Y = 0x249, Z = 0x492;
    order = third == 0 ? (mixed ? X : A) : third == 1 ? (mixed ? Y : B) : (mixed ? Z : C);
    i %= 6;
    order = (order >> 2 * i | order << (12 - 2 * i)) & 0xfff;
  }
  __device__ __forceinline__ void next() {
    const uint32_t now = order & 3;
    order = order >> 2 | now << 10;
    if (now == 0) __builtin_amdgcn_s_setprio(0);
    else if (now == 1) __builtin_amdgcn_s_setprio(1);
    else __builtin_amdgcn_s_setprio(2);
  }
};

constexpr int PA_WAVE_LDS = 12288;  // of a wave, where the waves of a workgroup go their own ways

// At most 16 rows of a sequence and KV head (single tokens): the waves take a quarter of each block's
// keys each, without barriers, and join in LDS.  Bound by the reads: a wave has three pieces of
// sixteen rows of K or V on their way into LDS of its own (fp8: four), of which one is used.
// S^T = K Q^T by 16x16x32 products, O^T += V^T P^T by 16x16x16, P as the sum of two
// terms of the type (16 bits of each weight), which the matrix cores have room for here.
// One token each behind 48 caches of up to 16384 keys 307 us, 5.6 TB/s of the 6.0 that plain reads have;
// behind 8 fp8 caches of up to 65537 136 us, 5.1 TB/s, the beginning and end of one wave of workgroups
// among them.
template <class T, int D, bool KV8, bool EVEN>
__device__ __forceinline__ void pa_few(PaWalk *walk, char *smem, float *s_scale, uint32_t *s_bad) {
  typedef typename std::conditional<KV8, DaBf16, T>::type TP;  // of P and V
  typedef typename T::x8 x8;
  typedef typename T::elem elem;
  typedef typename TP::elem pelem;
  typedef pelem px4 __attribute__((ext_vector_type(4)));
  constexpr int NW = 4, NK = D / 32, RB = KV8 ? D : 2 * D, UNIT = 16 * RB, NU = KV8 ? 4 : 3, NX = UNIT / 1024;
  constexpr int CH = D / 8;
  const int lane = pa_lane(), w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane >> 4, ri = lane & 15;
  char *mine = smem + w * PA_WAVE_LDS;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void_t *)mine);
  const uint32_t sc0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void_t *)((char *)s_scale + w * 768));
  // 16-byte chunk swizzles.  K: the sixteen rows of one chunk lie in all banks; V (two bytes a
  // value): eight rows' pairs of chunks (FewRows).
  auto swz_k = [](int r) { return D == 128 && !KV8 ? r & 15 : D == 128 || !KV8 ? (r >> 1) & 7 : (r >> 2) & 3; };
  auto swz_v = [](int r) { return D == 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3); };
  x8 qf[NK];
  f32x4 acc[D / 16];
  float m = pa_ninf(), thr = pa_ninf(), l = 0.f, nmu = 0.f;
  {
    const PaKP &p = pa_args();
    const PaPiece x = pa_piece<128, DA_BS, false>(p, walk);
    const int nrow = x.sq.lq * p.G, row = min(ri, nrow - 1), t = row / p.G;
    const int lim = p.causal ? x.sq.lk - x.sq.lq + t : x.sq.lk - 1;  // last key seen
    const float qscale = p.qscale, thr_gap = p.thr_gap;
    const int64_t s_stride = p.s_stride;
    const void *kp = p.k, *vp = p.v;
    const float *k_scale = p.k_scale, *v_scale = p.v_scale;
    PaRows<EVEN> rows;
    rows.pages = p.page_table + x.b * p.pt_sb;
    rows.key0 = 16 * w;
    rows.last = x.sq.lk - 1;
    const int n = x.blocks.j1 - x.blocks.j0;
    // piece u of K or V rows: K of block j0 + u / 2, then V
    auto load = [&](int u) {
      const int j = x.blocks.j0 + (u >> 1);
      if ((u & 1) == 0 && j - rows.jb == PaRows<EVEN>::SPAN) rows.look(p, x.kvh, j);
      const uint32_t to = lds0 + (uint32_t)(u % NU) * UNIT;
      if (u & 1) {
        if constexpr (KV8) rows.template load<RB, 16>(vp, j, to, lane, [](int) { return 0; });
        else rows.template load<RB, 8>(vp, j, to, lane, swz_v);
      } else {
        rows.template load<RB, 16>(kp, j, to, lane, swz_k);
        if constexpr (KV8) {  // the keys' scales and their values', 16 each (and again)
          const float *src = (lane & 16 ? v_scale : k_scale) + rows.of(j, ri) * (uint64_t)s_stride;
          const uint32_t m0 = sc0 + (uint32_t)((u >> 1) % 3) * 256;
          asm volatile("global_load_lds_dword %0, off" ::"v"(src), "{m0}"(m0) : "memory");
        }
      }
    };
    const elem *qp = (const elem *)p.q + pa_q_at(p, x.b, x.sq, t, x.kvh * p.G + row % p.G);
#pragma unroll
    for (int s = 0; s < NK; ++s) qf[s] = *(const x8 *)(qp + 32 * s + 8 * c);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (n > 0) {
      rows.look(p, x.kvh, x.blocks.j0);
#pragma unroll
      for (int u = 0; u < NU; ++u)
        if (u < 2 * n) load(u);
    }
#pragma unroll
    for (int s = 0; s < NK; ++s) settle(qf[s]);
    PaTurns turns((int)(blockIdx.x / (uint32_t)(p.W * p.Hkv / 3 + 1)), x.mixed, 0);
    for (int i = 0; i < n; ++i) {
      const int j = x.blocks.j0 + i;
      turns.next();
      // newer pieces on their way: V of this block, and K (fp8: and V) of the next
      if (i + 1 < n) wait_vmcnt<(NU - 1) * NX + (KV8 ? 1 : 0)>();
      else wait_vmcnt<NX>();
      const float *sc = (const float *)((const char *)s_scale + w * 768 + (i % 3) * 256);
      f32x4 st = f32x4{0.f, 0.f, 0.f, 0.f};
      const char *sk = mine + ((2 * i) % NU) * UNIT;
#pragma unroll
      for (int s = 0; s < NK; ++s) {
        if constexpr (KV8) {
          const uint2 codes = *(const uint2 *)(sk + ri * RB + 16 * ((2 * s + (c >> 1)) ^ swz_k(ri)) + 8 * (c & 1));
          const uint2 a = pa_widen<T>(codes.x), b = pa_widen<T>(codes.y);
          st = T::mfma16(__builtin_bit_cast(x8, uint4{a.x, a.y, b.x, b.y}), qf[s], st);
        } else {
          st = T::mfma16(*(const x8 *)(sk + ri * RB + 16 * ((4 * s + c) ^ swz_k(ri))), qf[s], st);
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K is read: its place is free
      if (2 * i + NU < 2 * n) load(2 * i + NU);
      if constexpr (KV8) {
        // register e: key 4 c + e
#pragma unroll
        for (int e = 0; e < 4; ++e) st[e] *= sc[4 * c + e];
      }
      const int d = lim - j * DA_BS - 16 * w - 4 * c;
      float mx = pa_ninf();
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        st[e] = e <= d ? st[e] : pa_ninf();
        mx = fmaxf(mx, st[e]);
      }
      if (__ballot(mx > thr) != 0) {
        const float mn = fmaxf(m, pair32_max(pair16_max(mx))), to = da_ref<TP>(mn, qscale);
        const float alpha = m == pa_ninf() ? 0.f : fast_exp2(to - nmu);
        m = mn;
        thr = mn + thr_gap;
        nmu = to;
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) acc[dt] *= alpha;
      }
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        st[e] = fast_exp2(__builtin_fmaf(st[e], qscale, nmu));
        sum += st[e];
      }
      l += sum;
      if constexpr (KV8) {
#pragma unroll
        for (int e = 0; e < 4; ++e) st[e] *= sc[16 + 4 * c + e];
      }
      px4 hi, lo;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        hi[e] = (pelem)st[e];
        lo[e] = (pelem)(st[e] - (float)hi[e]);
      }
      // newer: K and V of the next block, and (fp8) K of the one behind it
      if (KV8 && i + 2 < n) wait_vmcnt<3 * NX + 2>();
      else if (i + 1 < n) wait_vmcnt<2 * NX + (KV8 ? 1 : 0)>();
      else wait_vmcnt<0>();
      const uint16_t *sv = (const uint16_t *)(mine + ((2 * i + 1) % NU) * UNIT);
      if constexpr (KV8) {  // widened into a place of its own
        sv = (const uint16_t *)(mine + NU * UNIT);
#pragma unroll
        for (int y = 0; y < NX; ++y) {
          const int at = 64 * y + lane, r = at / (RB / 16), ch = at % (RB / 16);
          const uint4 codes = *(const uint4 *)(mine + ((2 * i + 1) % NU) * UNIT + 16 * at);
          const uint2 a = pa_widen<TP>(codes.x), b = pa_widen<TP>(codes.y), e = pa_widen<TP>(codes.z), f = pa_widen<TP>(codes.w);
          *(uint4 *)((char *)sv + 2 * r * D + 16 * ((2 * ch) ^ swz_v(r))) = uint4{a.x, a.y, b.x, b.y};
          *(uint4 *)((char *)sv + 2 * r * D + 16 * ((2 * ch + 1) ^ swz_v(r))) = uint4{e.x, e.y, f.x, f.y};
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      const int kr = 4 * c + (ri >> 2);
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) {
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_s16x4 *)(sv + kr * D + 8 * ((2 * dt + ((ri & 3) >> 1)) ^ swz_v(kr)) + 4 * (ri & 1)));
        acc[dt] = pa_mfma16<TP>(a, __builtin_bit_cast(s16x4, hi), acc[dt]);
        acc[dt] = pa_mfma16<TP>(a, __builtin_bit_cast(s16x4, lo), acc[dt]);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // V is read
      if (2 * i + 1 + NU < 2 * n) load(2 * i + 1 + NU);
    }
    l = pair32_sum(pair16_sum(l));
  }
  // the waves' states into LDS, and together
  float *ml = (float *)mine, *vals = ml + 32;
  if (c == 0) {
    ml[2 * ri] = m == pa_ninf() ? m : -nmu;
    ml[2 * ri + 1] = l;
  }
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt) *(f32x4 *)&vals[ri * (D + 4) + 16 * dt + 4 * c] = acc[dt];
  if (threadIdx.x == 0) *s_bad = 0u;
  lds_barrier();
  const PaKP &p = pa_args();
  const PaPiece x = pa_piece<128, DA_BS, false>(p, walk);
  const int nrow = x.sq.lq * p.G;
  for (int e = threadIdx.x; e < nrow * D; e += 64 * NW) {
    const int g = e / D, dim = e % D;
    float mm = pa_ninf();
#pragma unroll
    for (int y = 0; y < NW; ++y) mm = fmaxf(mm, ((const float *)(smem + y * PA_WAVE_LDS))[2 * g]);
    float ll = 0.f, a = 0.f;
#pragma unroll
    for (int y = 0; y < NW; ++y) {
      const float *of = (const float *)(smem + y * PA_WAVE_LDS);
      const float f = fast_exp2(of[2 * g] - (mm == pa_ninf() ? 0.f : mm));
      ll = __builtin_fmaf(of[2 * g + 1], f, ll);
      a = __builtin_fmaf(of[32 + g * (D + 4) + dim], f, a);
    }
    // (with scores that are not numbers, l is not, and the row stands)
    if (!(fabsf(a) < __int_as_float(0x7f800000)) && ll > 0.f && ll < __int_as_float(0x7f800000)) atomicOr(s_bad, 1u << g);
    if (ll == 0.f) a = 0.f;  // (no key seen)
    const int t = g / p.G, h = x.kvh * p.G + g % p.G;
    if (x.part >= 0) {
      p.ws_acc[(x.part + g) * D + dim] = a;
      if (dim == 0) {
        p.ws_ml[2 * (x.part + g)] = mm;
        p.ws_ml[2 * (x.part + g) + 1] = ll;
      }
    } else {
      store_from_f32(p.out, pa_out_at(p, x.b, x.sq, t, h) + dim, p.out_dt, ll == 0.f ? 0.f : a / ll);
      if (p.lse && dim == 0) p.lse[pa_lse_at(p, x.b, x.sq, t, h)] = ll == 0.f ? pa_ninf() : (mm + __log2f(ll)) * PA_LN2;
    }
  }
  __syncthreads();
  // (an infinity that a row sees meets weights of both signs in the second terms, so all are done
  // again; every wave's stores are done, which those replace)
  if (*s_bad != 0u) {
    const uint32_t bad = *s_bad;
    wait_vmcnt<0>();
    __syncthreads();
    for (int g = w; g < nrow; g += NW)
      pa_again<elem, D, DA_BS, 16, KV8, true, false, false>(p, x.b, x.sq, x.kvh, x.part, 0, 0, bad & (1u << g), x.blocks, x.blocks.n_all);
  }
}

// A row as two lanes hold it (pa_in_part), times inv, to out; the two (hf 0 and 1) trade fours, so that each
// stores eight values of 16 bits.
template <class E, int D>
__device__ __forceinline__ void pa_rows_out(const PaKP &p, int64_t o, const f32x16 (&acc)[D / 32], float inv, int hf) {
  if (p.out_dt == LA_F32) {
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(float4 *)((float *)p.out + o + 32 * dt + 8 * i + 4 * hf) =
            float4{acc[dt][4 * i] * inv, acc[dt][4 * i + 1] * inv, acc[dt][4 * i + 2] * inv, acc[dt][4 * i + 3] * inv};
    return;
  }
  typedef E x4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      uint2 y[2];
#pragma unroll
      for (int z = 0; z < 2; ++z)
        y[z] = __builtin_bit_cast(uint2, x4{(E)(acc[dt][4 * (i + z)] * inv), (E)(acc[dt][4 * (i + z) + 1] * inv),
                                            (E)(acc[dt][4 * (i + z) + 2] * inv), (E)(acc[dt][4 * (i + z) + 3] * inv)});
      const auto a = __builtin_amdgcn_permlane32_swap(y[0].x, y[1].x, false, false);
      const auto c = __builtin_amdgcn_permlane32_swap(y[0].y, y[1].y, false, false);
      *(uint4 *)((E *)p.out + o + 32 * dt + 8 * (i + hf)) = uint4{a[0], c[0], a[1], c[1]};
    }
}

// bf16 / fp16 rows: four waves of 32 rows, three workgroups a CU, and the products and registers of
// dense_attn_kernel (S^T by 32x32x16 products leaves a lane 16 scores of one row; P goes into its
// product with V from the same registers, rounded to the inputs' type; l is of the fp32 weights).
// With an fp8 cache weights take the values' scales, whose range is fp32's, and are rounded to bf16; of
// fp16 queries, whose bits that would lose, to two terms of bf16 (16 bits): chunks of four prompts
// 325 us, with one term 271, and 2.1e-4 of the norm off in place of 1.7e-3.
//
// A wave stages 16 keys of each block of 64 (PaRows).  K and V of the blocks take three slots in turn,
// so that each is on its way while the block before is scored and weighed.  fp8 caches
// (KV8): codes of K and V go into LDS a block ahead, and are widened there once a workgroup (e4m3 is exact
// in bf16 and fp16); the scale of a key multiplies its scores, that of its value its weights, both in fp32.
//
// Bound by matrix and vector unit in turn: 8192 tokens behind 24576 3.34 to 3.49 ms, 1.15 to 1.10 PFLOP/s
// (a large product has 1.36), the matrix unit busy for 57 to 65 % of the cycles
// at 1.75 to 1.53 GHz.  Products of the next block beside a block's weights (32 keys at a time, for the
// registers) take 3.77 to 3.90 ms, two workgroups a CU with them 4.16.
// Over fp8 caches a block is widened between two barriers, and nothing else of the workgroup goes on
// meanwhile: chunks of four prompts 255 us, over bf16 205.
template <class T, int D, bool KV8, bool EVEN>
__device__ __forceinline__ void pa_many(PaWalk *walk, uint16_t *smem, float *s_scale) {
  typedef typename std::conditional<KV8, DaBf16, T>::type TP;  // of P and V
  constexpr bool TWO = KV8 && !std::is_same<T, TP>::value;     // P in two terms
  constexpr int NW = 4, R = 32 * NW, BLK = DA_BS * D, NX = D / 32;
  constexpr int NS = D / 16, ND = D / 32;
  constexpr int SLOT = 2 * BLK;  // bytes; KV8: K, V, then codes of K and of V
  typedef typename T::x8 x8;
  typedef typename TP::x8 px8;
  typedef typename T::elem elem;
  typedef typename TP::elem pelem;
  const int lane = pa_lane(), w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hf = lane >> 5, r32 = lane & 31;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void_t *)smem);
  // Byte offsets of this lane's first reads of a slot (as in dense_attn_kernel).
  const uint32_t k_at = 2 * (r32 * D + 8 * (hf ^ da_swz_k<D>(r32)));
  const int v_row = 4 * hf + ((lane & 15) >> 2);
  const uint32_t v_at = 2 * (v_row * D + 8 * ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ da_swz_v<D>(v_row)) +
                             4 * (lane & 1));
  const char *lds = (const char *)smem;
  float m = pa_ninf(), thr = pa_ninf(), l = 0.f, nmu = 0.f;
  f32x16 acc[ND];
  {
    const PaKP &p = pa_args();
    const PaPiece x = pa_piece<R, DA_BS, true>(p, walk);
    const int G = p.G, nrow = x.sq.lq * G, diag = x.sq.lk - x.sq.lq, causal = p.causal;
    auto limit = [&](int t) { return causal ? diag + t : x.sq.lk - 1; };  // last key seen
    const int r_first = x.r0 + 32 * w, r_mine = min(r_first + r32, nrow - 1);
    const int t = r_mine / G, lim = limit(t);
    const int lim_lo = __builtin_amdgcn_readfirstlane(limit(min(r_first, nrow - 1) / G));
    const int lim_hi = __builtin_amdgcn_readfirstlane(limit(min(r_first + 31, nrow - 1) / G));
    const PaBlocks blocks = x.blocks;
    const int j0 = blocks.j0, j1 = blocks.j1;
    const float qscale = p.qscale, thr_gap = p.thr_gap;
    const void *kp = p.k, *vp = p.v;
    const float *k_scale = p.k_scale, *v_scale = p.v_scale;
    const int64_t s_stride = p.s_stride;
    PaRows<EVEN> rows;
    rows.pages = p.page_table + x.b * p.pt_sb;
    rows.key0 = 16 * w;
    rows.last = x.sq.lk - 1;
    const int sw = 16 * w;
    auto dma_k = [&](int j, int slot) __attribute__((always_inline)) {
      if ((uint32_t)(j - rows.jb) >= (uint32_t)PaRows<EVEN>::SPAN) rows.look(p, x.kvh, j);
      rows.template load<2 * D, 8>(kp, j, lds0 + (uint32_t)(slot * SLOT + 2 * sw * D), lane, [&](int r) { return da_swz_k<D>(sw + r); });
    };
    auto dma_v = [&](int j, int slot) __attribute__((always_inline)) {
      rows.template load<2 * D, 4>(vp, j, lds0 + (uint32_t)(slot * SLOT + 2 * sw * D), lane, [&](int r) { return da_swz_v<D>(sw + r); });
    };
    // fp8: codes of a block, a wave's own rows, and (lanes below 16) the keys' scales
    float ks = 0.f, vs = 0.f;
    auto dma_codes = [&](int j) __attribute__((always_inline)) {
      const int lane = pa_lane();
      if ((uint32_t)(j - rows.jb) >= (uint32_t)PaRows<EVEN>::SPAN) rows.look(p, x.kvh, j);
      rows.template load<D, 1>(kp, j, lds0 + 4 * BLK + sw * D, lane, [](int) { return 0; });
      rows.template load<D, 1>(vp, j, lds0 + 5 * BLK + sw * D, lane, [](int) { return 0; });
      const uint64_t at = (uint64_t)rows.of(j, lane & 15) * s_stride;
      ks = k_scale[at];
      vs = v_scale[at];
    };
    auto widen = [&]() __attribute__((always_inline)) {
      const int lane = pa_lane();
#pragma unroll
      for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int y = 0; y < D / 64; ++y) {
          const int at = 64 * y + lane, row = sw + at / (D / 16), ch = 2 * (at % (D / 16));
          const uint4 u = *(const uint4 *)(lds + (4 + v) * BLK + sw * D + 16 * at);
          const int swz = v ? da_swz_v<D>(row) : da_swz_k<D>(row);
          uint2 z[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) z[i] = v ? pa_widen<TP>((&u.x)[i]) : pa_widen<T>((&u.x)[i]);
          char *to = (char *)smem + 2 * (v * BLK + row * D);
          *(uint4 *)(to + 16 * (ch ^ swz)) = uint4{z[0].x, z[0].y, z[1].x, z[1].y};
          *(uint4 *)(to + 16 * ((ch + 1) ^ swz)) = uint4{z[2].x, z[2].y, z[3].x, z[3].y};
        }
      if (lane < 16) {
        s_scale[sw + lane] = ks;
        s_scale[DA_BS + sw + lane] = vs;
      }
    };
    int j = blocks.at(j0);
    if (j0 < j1) {
      rows.look(p, x.kvh, j);
      if constexpr (KV8) {
        dma_codes(j);
      } else {
        dma_k(j, 0);
        dma_v(j, 1);
      }
    }
    x8 qf[NS];  // B operand: dims 16 s + 8 hf ..
    {
      const elem *qp = (const elem *)p.q + pa_q_at(p, x.b, x.sq, t, x.kvh * G + r_mine % G) + 8 * hf;
#pragma unroll
      for (int s = 0; s < NS; ++s) qf[s] = *(const x8 *)(qp + 16 * s);
    }
#pragma unroll
    for (int s = 0; s < NS; ++s) settle(qf[s]);
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[dt][i] = 0.f;

    // scores of block j; register i of a half holds key 8 (i / 4) + 4 hf + i % 4
    auto scores = [&](int slot, f32x16 (&st)[2]) __attribute__((always_inline)) {
      const uint32_t at = k_at + slot * SLOT;
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
            const f32x4 sc = *(const f32x4 *)(s_scale + 32 * kt + 8 * g + 4 * hf);
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
        const float mn = fmaxf(m, pair32_max(mx)), to = da_ref<TP>(mn, qscale);
        const float alpha = m == pa_ninf() ? 0.f : fast_exp2(to - nmu);  // (both as rounded in the weights)
        m = mn;
        thr = mn + thr_gap;
        nmu = to;
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[dt][i] *= alpha;
      }
    };
    // weights of half kt of a block, added among themselves first
    auto weigh = [&](int kt, f32x16 &st, px8 (&pw)[TWO ? 4 : 2]) __attribute__((always_inline)) {
      float sum[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        st[i] = fast_exp2(__builtin_fmaf(st[i], qscale, nmu));
        sum[i & 1] = i < 2 ? st[i] : sum[i & 1] + st[i];
        if constexpr (!KV8) pw[i >> 3][i & 7] = (pelem)st[i];
      }
      l += sum[0] + sum[1];
      if constexpr (KV8) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 sc = *(const f32x4 *)(s_scale + DA_BS + 32 * kt + 8 * g + 4 * hf);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = st[4 * g + i] * sc[i];
            const pelem hi = (pelem)x;
            pw[g >> 1][4 * (g & 1) + i] = hi;
            if constexpr (TWO) pw[2 + (g >> 1)][4 * (g & 1) + i] = (pelem)(x - (float)hi);
          }
        }
      }
    };
    auto values = [&](int slot, int kt, const px8 (&pw)[TWO ? 4 : 2]) __attribute__((always_inline)) {
      const uint32_t at = v_at + slot * SLOT;
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) {
          const char *v = lds + (at ^ (64 * dt)) + 2 * (32 * kt + 16 * y) * D;
          const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)v);
          const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(v + 16 * D));
          const px8 vt = __builtin_bit_cast(px8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
          acc[dt] = TP::mfma(vt, pw[y], acc[dt]);
          if constexpr (TWO) acc[dt] = TP::mfma(vt, pw[2 + y], acc[dt]);
        }
    };

    const int jw = r_first < nrow && lim_hi >= 0 ? lim_hi / DA_BS : -1;  // this wave's last block
    PaTurns turns((int)(blockIdx.x / (uint32_t)(p.W * p.Hkv / 3 + 1)), x.mixed, j0);
    int sk = 0, sv = 1;  // this block's slots
    for (int i = j0; i < j1; ++i) {
      const int next = j + 1 < blocks.n_all ? j + 1 : 0, free = 3 - sk - sv;
      turns.next();
      f32x16 st[2];
      px8 pw[TWO ? 4 : 2];
      if constexpr (KV8) {
        wait_vmcnt<0>();
        lds_barrier();  // the block before is read
        widen();
        lds_barrier();  // this one is there, and its codes are read
      } else {
        wait_vmcnt<NX>();
        lds_barrier();  // K of this block has landed for every wave, V of the one before is read
        if (i + 1 < j1) dma_k(next, free);
      }
      if (j <= jw) {
        scores(sk, st);
        settle_max(j, st, largest(st));
        weigh(0, st[0], pw);
      }
      if constexpr (KV8) {
        // (here: registers are short before, and a reload of one waits for loads issued before it: chunks of
        // four prompts over fp8 caches take 260 us, and 290 with these at the block's beginning)
        if (i + 1 < j1) dma_codes(next);
      } else {
        if (i + 1 < j1) wait_vmcnt<NX>();
        else wait_vmcnt<0>();
        lds_barrier();  // V of this block has landed, its K is read
        if (i + 1 < j1) dma_v(next, sk);
      }
      if (j <= jw) {
        values(sv, 0, pw);
        weigh(1, st[1], pw);
        values(sv, 1, pw);
      }
      if constexpr (!KV8) {
        sv = sk;
        sk = free;
      }
      j = next;
    }
  }
  const PaKP &p = pa_args();
  const PaPiece x = pa_piece<R, DA_BS, true>(p, walk);
  const int G = p.G, nrow = x.sq.lq * G, r_first = x.r0 + 32 * w, r_mine = min(r_first + r32, nrow - 1);
  if (r_first >= nrow) return;
  const bool live = r_first + r32 < nrow;
  const int t = r_mine / G, h = x.kvh * G + r_mine % G;
  l = pair32_sum(l);
  // results that are not finite (with scores that are not numbers, l is not, and the row stands)
  float sum = 0.f;
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) sum = __builtin_fmaf(acc[dt][i], 0.f, sum);
  const uint64_t bad = __ballot(sum != 0.f && l < __int_as_float(0x7f800000));  // (sum: NaN)
  // register i of dim tile dt holds dim 32 dt + 8 (i / 4) + 4 hf + i % 4
  if (x.part >= 0) {
    const int64_t pi = x.part + r_first - x.r0;  // (room for whole waves)
    if (hf == 0) {
      p.ws_ml[2 * (pi + r32)] = m == pa_ninf() ? m : -nmu;
      p.ws_ml[2 * (pi + r32) + 1] = l;
    }
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(float4 *)(p.ws_acc + pi * D + (dt * 4 + i) * 256 + 4 * lane) =
            float4{acc[dt][4 * i], acc[dt][4 * i + 1], acc[dt][4 * i + 2], acc[dt][4 * i + 3]};
  } else if (live) {
    const bool none = l == 0.f;  // no key seen
    pa_rows_out<elem, D>(p, pa_out_at(p, x.b, x.sq, t, h), acc, none ? 0.f : 1.f / l, hf);
    if (p.lse && hf == 0) p.lse[pa_lse_at(p, x.b, x.sq, t, h)] = none ? pa_ninf() : (__log2f(l) - nmu) * PA_LN2;  // (as rounded in the weights)
  }
  if (bad != 0) {
    const int lim_hi = p.causal ? x.sq.lk - x.sq.lq + min(r_first + 31, nrow - 1) / G : x.sq.lk - 1;
    // (in two terms: as in pa_few)
    pa_again<elem, D, DA_BS, 32, KV8, TWO, (!KV8 && T::BIAS > 0.f), true>(p, x.b, x.sq, x.kvh, x.part, x.r0, r_first,
                                                                     (uint32_t)(bad | (bad >> 32)) & (uint32_t)__ballot(live),
                                                                     x.blocks, lim_hi / DA_BS);
  }
}

template <class T, int D, bool KV8, bool EVEN>
__global__ __launch_bounds__(256, 3) void paged_attn_kernel(PaKP) {
  __shared__ __align__(16) uint16_t smem[PA_WAVE_LDS * 4 / 2];
  __shared__ __align__(16) float s_scale[KV8 ? 768 : 4];  // few: 3 blocks' of each wave; many: a block's
  __shared__ PaWalk s_walk;
  __shared__ uint32_t s_bad;
  static_assert(sizeof(uint16_t) * 3 * DA_BS * D <= sizeof(smem), "K and V");
  if (pa_begin<128, true>(&s_walk)) {
    do {
      if (__builtin_amdgcn_readfirstlane(s_walk.s.few)) pa_few<T, D, KV8, EVEN>(&s_walk, (char *)smem, s_scale, &s_bad);
      else pa_many<T, D, KV8, EVEN>(&s_walk, smem, s_scale);
    } while (pa_next<128, true>(&s_walk));
  }
  const PaKP &p = pa_args();
  pa_rest<D>(p, (int)(blockIdx.x % (uint32_t)p.Hkv));
}

// fp32 rows: four waves of 16 rows on 16x16x4 products, blocks of 32 keys (dense_attn_f32_kernel's),
// over pages of any size, a lane a key, pages two blocks ahead and keys one.  Bound by the fp32 products (two
// chunks of 256 tokens behind 4096, 16 heads on 8, 177 us, of which the products alone would take 110; the matrix
// unit is busy for 62 % of the cycles).  Of single tokens the rows fill one wave, which does all products while
// the other three only stage, and a block's keys are on their way for as long as one block's products take:
// 32 tokens behind up to 8192 290 us, 4.5 TB/s of the 6.0 that plain reads have, waves waiting 75 % of the time.
template <int D>
__global__ __launch_bounds__(256, 2) void paged_attn_f32_kernel(PaKP p) {
  constexpr int NW = 4, R = 16 * NW, BS = 32, BLK = BS * D, CH = D / 4, RP = 64 / CH, NX = BS / RP / NW;
  constexpr int NS = D / 16;
  __shared__ __align__(16) float smem[4 * BLK];
  __shared__ PaWalk s_walk;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane >> 4, ri = lane & 15;
  const int G = p.G;
  bool more = pa_begin<R, false>(&s_walk);
  auto swz_k = [](int r) { return 2 * (r & 7); };
  auto swz_v = [](int r) { return 4 * ((r >> 2) & 3); };
  for (; more; more = pa_next<R, false>(&s_walk)) {
    const PaPiece x = pa_piece<R, BS, true>(p, &s_walk);
    const PaSeq sq = x.sq;
    const PaBlocks blocks = x.blocks;
    const int b = x.b, r0 = x.r0, kvh = x.kvh, j0 = blocks.j0, j1 = blocks.j1;
    const int64_t part = x.part;
    const int nrow = sq.lq * G, diag = sq.lk - sq.lq;
    auto limit = [&](int t) { return p.causal ? diag + t : sq.lk - 1; };
    const int r_first = r0 + 16 * w;
    const int r_mine = min(r_first + ri, nrow - 1);
    const bool live = r_first + ri < nrow, wave_live = r_first < nrow;
    const int t = r_mine / G, h = kvh * G + r_mine % G;
    const int lim = limit(t);
    const int lim_lo = __builtin_amdgcn_readfirstlane(limit(min(r_first, nrow - 1) / G));
    const int lim_hi = __builtin_amdgcn_readfirstlane(limit(min(r_first + 15, nrow - 1) / G));
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
    if (j0 < j1) {
      rows = look(blocks.at(j0));
      rows_next = look(blocks.at(min(j0 + 1, j1 - 1)));
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
    for (int i = j0; i < j1; ++i) {
      const int par = (i - j0) & 1, j = blocks.at(i);
      wait_vmcnt<0>();
      settle(rows_next);
      lds_barrier();
      if (i + 1 < j1) {
        dma(rows_next, par ^ 1);
        rows_next = look(blocks.at(min(i + 2, j1 - 1)));
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
      if ((i - j0) % 16 == 15) {
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
        pa_again<float, D, BS, 16, false, false, false, false>(p, b, sq, kvh, part, r0, r_first, (uint32_t)((bad | (bad >> 16)) & __ballot(live) & 0xffffu),
                                                       blocks, lim_hi / BS);
      }
    }
  }
  pa_rest<D>(p, (int)(blockIdx.x % (uint32_t)p.Hkv));
}

// What D / 4 lanes hold of a row: the reference, the weights' sum and four values each.
struct PaState {
  float m, l;
  float4 acc;
  __device__ __forceinline__ PaState() : m(pa_ninf()), l(0.f), acc{0.f, 0.f, 0.f, 0.f} {}
  __device__ __forceinline__ void add(float2 ml, const float4 &v) {
    if (ml.x == pa_ninf() && ml.y == 0.f) return;  // (empty: no key seen)
    const float mn = fmaxf(m, ml.x), from = mn == pa_ninf() ? 0.f : mn;
    const float f = m == pa_ninf() && l == 0.f ? 0.f : fast_exp2(m - from), g = fast_exp2(ml.x - from);
    m = mn;
    l = l * f + ml.y * g;
    acc.x = acc.x * f + v.x * g;
    acc.y = acc.y * f + v.y * g;
    acc.z = acc.z * f + v.z * g;
    acc.w = acc.w * f + v.w * g;
  }
};

// Joins the parts of tiles that lie row by row: a row by D / 4 lanes, or, of more than 16 parts
// (few tiles, each shared by many workgroups), by all, which take the parts in turn and join in LDS (with
// more than 4 by all, fp32 chunks of 8 parts take 202 us, not 177).
template <int D, int R>
__device__ __forceinline__ void pa_join_rows(const PaKP &p, const int4 &note, int own, int kvh) {
  constexpr int LR = D / 4, RW = 256 / LR, AHEAD = 8;  // lanes of a row, rows at a time, parts on their way
  __shared__ float s_ml[2 * RW];
  __shared__ float4 s_acc[256];
  const int b = note.x, G = p.G;
  const PaSeq sq = pa_seq(p, b);
  const int nrow = sq.lq * G, r0 = note.y * R, lane = threadIdx.x % LR, group = threadIdx.x / LR;
  auto parts = [&](PaState &x, int r, int first, int step) {
    for (int i0 = first; i0 < note.z; i0 += AHEAD * step) {
      float2 ml[AHEAD];
      float4 v[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int y = min(i0 + i * step, note.z - 1);
        const int64_t pi = pa_part(p, own + y, kvh, y == 0, note.w != 0) + r - r0;
        ml[i] = *(const float2 *)(p.ws_ml + 2 * pi);
        v[i] = *(const float4 *)(p.ws_acc + pi * D + 4 * lane);
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (i0 + i * step < note.z) x.add(ml[i], v[i]);
    }
  };
  auto store = [&](const PaState &x, int r) {
    const int t = r / G, h = kvh * G + r % G;
    const bool none = x.l == 0.f;
    const float inv = none ? 0.f : 1.f / x.l;
    const int64_t o = pa_out_at(p, b, sq, t, h) + 4 * lane;
    const float y[4] = {x.acc.x * inv, x.acc.y * inv, x.acc.z * inv, x.acc.w * inv};
    if (p.out_dt == LA_F32) {
      *(float4 *)((float *)p.out + o) = float4{y[0], y[1], y[2], y[3]};
    } else if (p.out_dt == LA_BF16) {
      typedef __bf16 x4 __attribute__((ext_vector_type(4)));
      *(x4 *)((__bf16 *)p.out + o) = x4{(__bf16)y[0], (__bf16)y[1], (__bf16)y[2], (__bf16)y[3]};
    } else {
      typedef _Float16 x4 __attribute__((ext_vector_type(4)));
      *(x4 *)((_Float16 *)p.out + o) = x4{(_Float16)y[0], (_Float16)y[1], (_Float16)y[2], (_Float16)y[3]};
    }
    if (p.lse && lane == 0) p.lse[pa_lse_at(p, b, sq, t, h)] = none ? pa_ninf() : (x.m + __log2f(x.l)) * PA_LN2;
  };
  const int end = min(nrow, r0 + R);
  if (note.z <= 2 * AHEAD) {
    for (int r = r0 + blockIdx.y * RW + group; r < end; r += gridDim.y * RW) {
      PaState x;
      parts(x, r, 0, 1);
      store(x, r);
    }
    return;
  }
  for (int r = r0 + blockIdx.y; r < end; r += gridDim.y) {
    PaState x;
    parts(x, r, group, RW);
    if (lane == 0) {
      s_ml[2 * group] = x.m;
      s_ml[2 * group + 1] = x.l;
    }
    s_acc[threadIdx.x] = x.acc;
    __syncthreads();
    if (group == 0) {
      for (int g = 1; g < RW; ++g) x.add(float2{s_ml[2 * g], s_ml[2 * g + 1]}, s_acc[g * LR + lane]);
      store(x, r);
    }
    __syncthreads();
  }
}

// The same where parts lie as waves hold them: four waves of 32 rows.
template <class E, int D>
__device__ __forceinline__ void pa_join_many(const PaKP &p, const int4 &note, int own, int kvh) {
  constexpr int ND = D / 32;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hf = lane >> 5, r32 = lane & 31;
  const PaSeq sq = pa_seq(p, note.x);
  const int nrow = sq.lq * p.G, r_first = note.y * 128 + 32 * w;
  if (r_first >= nrow) return;
  const int r = min(r_first + r32, nrow - 1);
  f32x16 acc[ND];
  float m = pa_ninf(), l = 0.f;
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[dt][i] = 0.f;
  for (int x = 0; x < note.z; ++x) {  // (parts in their order)
    const int64_t pi = pa_part(p, own + x, kvh, x == 0, false) + 32 * w;
    const float2 ml = *(const float2 *)(p.ws_ml + 2 * (pi + r32));
    float4 v[ND * 4];
#pragma unroll
    for (int i = 0; i < ND * 4; ++i) v[i] = *(const float4 *)(p.ws_acc + pi * D + i * 256 + 4 * lane);
    const bool empty = ml.x == pa_ninf() && ml.y == 0.f;  // (no key seen)
    const float mn = fmaxf(m, ml.x), from = mn == pa_ninf() ? 0.f : mn;
    const float f = m == pa_ninf() && l == 0.f ? 0.f : fast_exp2(m - from), g = empty ? 0.f : fast_exp2(ml.x - from);
    m = mn;
    l = l * f + (empty ? 0.f : ml.y * g);
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float y[4] = {v[4 * dt + i].x, v[4 * dt + i].y, v[4 * dt + i].z, v[4 * dt + i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[dt][4 * i + e] = acc[dt][4 * i + e] * f + (empty ? 0.f : y[e] * g);
      }
  }
  const int t = r / p.G, h = kvh * p.G + r % p.G;
  const bool none = l == 0.f;
  const int64_t o = pa_out_at(p, note.x, sq, t, h);
  if (r_first + r32 >= nrow) return;
  pa_rows_out<E, D>(p, o, acc, none ? 0.f : 1.f / l, hf);
  if (p.lse && hf == 0) p.lse[pa_lse_at(p, note.x, sq, t, h)] = none ? pa_ninf() : (m + __log2f(l)) * PA_LN2;
}

// Joins the tile that began last in a workgroup's stretch, if others have parts of it.  Bound by the reads
// of the parts (chunks of four prompts, 96 MB, 19 us), or a launch's latency (4 us).
template <class E, int D>
__global__ __launch_bounds__(256) void paged_join_kernel(PaKP p) {
  const int wg = blockIdx.x;
  const int4 note = p.ws_join[wg];
  if (note.z == 0) return;
  const int kvh = wg % p.Hkv, own = note.w ? note.w - 1 : wg / p.Hkv;
  if constexpr (sizeof(E) == 4) {
    pa_join_rows<D, 64>(p, note, own, kvh);
  } else {
    if (note.w) pa_join_rows<D, PA_FEW>(p, note, own, kvh);
    else if (blockIdx.y == 0) pa_join_many<E, D>(p, note, own, kvh);
  }
}

// ------------------------------------------------------------------ host ----
struct PaPlan {
  int64_t W = 1, rows = 128, least = 0, least_few = 0, few_parts = 0;
  int join = 1;  // workgroups of the join for each of the first launch's
  size_t ml = 0, notes = 0, bytes = 0;
};

static PaPlan pa_plan(const la_paged_attn_args *a) {
  PaPlan pl;
  const bool f32 = a->dtype == LA_F32;
  const int64_t G = a->Hq / a->Hkv, R = f32 ? 64 : 128;
  // workgroups that are there at once, shared among the KV heads (one at least for either line); no
  // stretch is shorter than four blocks of keys and a tile's beginning and end.  Of few rows four blocks
  // are enough: four tokens behind 1000 keys each 17.2 us (two blocks 17.0, eight 19.1), eight behind
  // 4000 25.1 (27.4, 23.9), one behind 16384 24.9 (24.6, 23.0), sixteen fp8 ones 19.5 (19.6, 20.3); in
  // fp32, whose blocks take four times as long, two: three tokens behind 1000 keys 17.7 (four 21.4).
  pl.least = G * (4 * DA_BS + PA_AHEAD);
  pl.least_few = G * 4 * DA_BS;
  if (f32) pl.least = pl.least_few = G * 2 * DA_BS;
  const int64_t rows = a->Tq * G, keys = a->pt_pages * a->page;  // (rows: of a sequence, at most)
  const int64_t tiles = a->cu_q ? std::min(rows, rows / R + a->B) : a->B * ceil_div(rows, R);  // at most
  const double most = (double)tiles * ((double)G * (keys + PA_AHEAD) + (a->causal ? R + 0.0 : 0.0));
  pl.W = std::max<int64_t>(f32 ? 1 : 2, (f32 ? 2 : 3) * num_cus() / a->Hkv);
  if (most / pl.least_few + 2 < (double)pl.W) pl.W = (int64_t)(most / pl.least_few) + 2;
  if (most <= 2.0 * G * (4 * DA_BS + PA_AHEAD)) {  // a stretch for each line, nothing to join: a launch less (4 us)
    pl.least = pl.least_few = (int64_t)1 << 60;
    pl.W = 2;
    pl.join = 0;
  }
  if (pl.join && (f32 || tiles < pl.W / 4)) pl.join = 4;  // (fp32's rows, or a row's many parts: 2 us of 26 of one token behind 16384 keys)
  pl.rows = std::min(R, ceil_div(rows, 32) * 32);  // (whole waves)
  pl.few_parts = pl.W * a->Hkv * 2 * pl.rows;
  const int64_t parts = pl.join ? pl.few_parts + (f32 ? 0 : pl.W * a->Hkv * 2 * PA_FEW) : 0;
  pl.ml = ((size_t)parts * 2 * sizeof(float) + 255) / 256 * 256;
  pl.notes = pl.ml + ((size_t)parts * a->D * sizeof(float) + 255) / 256 * 256;
  pl.bytes = pl.notes + (size_t)(pl.W * a->Hkv) * sizeof(int4);
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
  // the line of all tiles is counted in 64 bits and shared out by quotients that are exact below 2^53 (a
  // call of that size would take hours)
  const double G = (double)(a->Hq / a->Hkv), span = (double)std::max(a->pt_pages * a->page, a->Tq) + PA_AHEAD;
  LA_REQUIRE(((a->cu_q ? 1. : (double)a->B) * (double)a->Tq * G / 64 + (double)a->B) * (G * span + 128) < 4e15,
             "la_paged_attention: more products than one call takes");
  return LA_OK;
}

template <class K>
static int pa_launch(K kernel, int64_t wgs, const PaKP &p, hipStream_t st, int y = 1) {
  kernel<<<dim3((uint32_t)wgs, y), dim3(256), 0, st>>>(p);
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
  const Cover::Dim each{a->s_stride * 4, a->n_phys * a->Hkv * a->page};
  const Cover written[] = {Cover(a->out, a->D * osz, {a->o_sb * osz, nb}, {a->o_sh * osz, a->Hq}, {a->o_st * osz, a->Tq}),
                           Cover(a->lse, a->Tq * 4, {a->l_sb * 4, nb}, {a->l_sh * 4, a->Hq}),
                           Cover(a->workspace, a->ws_bytes)};
  const Cover read[] = {Cover(a->q, a->D * esz, {a->q_sb * esz, nb}, {a->q_sh * esz, a->Hq}, {a->q_st * esz, a->Tq}),
                        Cover(a->k_pool, pool),
                        Cover(a->v_pool, pool),
                        Cover(kv8 ? a->k_scale : nullptr, 4, each),
                        Cover(kv8 ? a->v_scale : nullptr, 4, each),
                        Cover(a->page_table, a->pt_pages * 4, {a->pt_sb * 4, a->B}),
                        Cover(a->lengths, a->B * 4),
                        Cover(a->cu_q, (a->B + 1) * 4),
                        Cover(a->q_len, a->B * 4)};
  LA_REQUIRE(!overlap_any(written, read), "la_paged_attention: out, lse or the workspace shares memory with another argument");
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
  p.ws_join = (int4 *)((char *)a->workspace + pl.notes);
  p.Tq = a->Tq;
  p.q_sb = a->q_sb; p.q_sh = a->q_sh; p.q_st = a->q_st;
  p.o_sb = a->o_sb; p.o_sh = a->o_sh; p.o_st = a->o_st;
  p.l_sb = a->l_sb; p.l_sh = a->l_sh;
  p.pt_sb = a->pt_sb; p.s_stride = a->s_stride; p.n_phys = a->n_phys;
  p.least = pl.least; p.least_few = pl.least_few; p.few_parts = pl.few_parts;
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
  if (rc != LA_OK || !pl.join) return rc;
  if (a->dtype == LA_F32) return d128 ? pa_launch(paged_join_kernel<float, 128>, wgs, p, st, pl.join) : pa_launch(paged_join_kernel<float, 64>, wgs, p, st, pl.join);
  if (a->dtype == LA_BF16) return d128 ? pa_launch(paged_join_kernel<__bf16, 128>, wgs, p, st, pl.join) : pa_launch(paged_join_kernel<__bf16, 64>, wgs, p, st, pl.join);
  return d128 ? pa_launch(paged_join_kernel<_Float16, 128>, wgs, p, st, pl.join) : pa_launch(paged_join_kernel<_Float16, 64>, wgs, p, st, pl.join);
}

