// One decode step over an evicted cache (la_evict_decode): the slot of the new token, the
// attention over the cache with it, and the weights its entries gather.
//
// The K/V rows of a (sequence, KV head) are read once and bound the step; the heads of a
// group are the rows of FewRows (few_rows.h), each wave of a workgroup on rounds of its
// own, joined through LDS.  The slot's row is read from k_new / v_new, never from the
// cache, so writing it there races with nothing.  Weights need the row's final sum: the
// scores (a float per head and entry, 1/32 of the K/V bytes at four heads) are kept in
// the workspace.  Where there are enough (sequence, head) pairs, one workgroup does all
// of a pair; else its entries are split over workgroups, each of which looks for the slot
// on its own (all weights and positions of the pair: 8 bytes an entry, from L2 but for
// the first), and evict_join_kernel joins the parts.
// 64 caches of 2049 entries of 8 heads, bf16, D = 128: 109 us, 5.0 TB/s; four of 16385, 58
// (53 and a join of 6; their bytes alone 46); one of 257 entries in fp32, 12 us, dependent
// loads and barriers.
#include <algorithm>

#include "evict.h"
#include "few_rows.h"

namespace la {

struct EdKP {
  const void *q, *k_new, *v_new;
  void *k, *v, *out;
  float *weights;
  int32_t *positions;
  const int32_t *lengths, *pos;
  int32_t *slots;   // [pair] (split form, for evict_join_kernel)
  float *ml;        // [pair][split][G] (max in log2 units, sum)
  float *vals;      // [pair][split][G][D]
  float *scores;    // [pair][G][cs]
  int64_t q_sb, q_sh, kn_sb, kn_sh, vn_sb, vn_sh, o_sb, o_sh, recent, sink, cs;
  int32_t B, Hq, Hkv, G, C, splits, out_dt, chunks;
  float qscale;
};

typedef float ed_f4 __attribute__((ext_vector_type(4), aligned(4)));
typedef int32_t ed_i4 __attribute__((ext_vector_type(4), aligned(4)));

// The entry that makes room (of a full cache), by a workgroup of NT threads: the lowest
// key, of equal ones the highest slot.
template <int NT>
__device__ __forceinline__ int32_t ed_victim(const EdKP &p, int64_t pair, int64_t pos) {
  __shared__ uint64_t best[NT / 64];
  const float *w = p.weights + pair * p.C;
  const int32_t *ps = p.positions + pair * p.C;
  uint64_t mine = ~0ull;
  auto look = [&](int32_t i, float x, int32_t at) {
    const uint64_t k = ev_safe(at, pos, p.recent, p.sink) ? EV_SAFE : ev_key(x);
    mine = min(mine, (k << 32) | (uint32_t)~i);
  };
  const int32_t whole = p.C & ~3;
  constexpr int NB = 8;  // loads of each in flight
  for (int32_t i0 = 4 * (int32_t)threadIdx.x; i0 < whole; i0 += 4 * NB * NT) {
    ed_f4 x[NB];
    ed_i4 y[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int32_t i = min(i0 + 4 * NT * j, whole - 4);
      x[j] = *(const ed_f4 *)(w + i);
      y[j] = *(const ed_i4 *)(ps + i);
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int32_t i = min(i0 + 4 * NT * j, whole - 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) look(i + e, x[j][e], y[j][e]);
    }
  }
  if (whole + (int32_t)threadIdx.x < p.C) look(whole + threadIdx.x, w[whole + threadIdx.x], ps[whole + threadIdx.x]);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) mine = min(mine, (uint64_t)__shfl_xor((unsigned long long)mine, o, 64));
  if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = mine;
  __syncthreads();
  mine = best[0];
#pragma unroll
  for (int x = 1; x < NT / 64; ++x) mine = min(mine, best[x]);
  return (int32_t)~(uint32_t)mine;
}

__device__ __forceinline__ int32_t ed_held(const EdKP &p, int b) { return min(max(p.lengths[b], 0), p.C); }

// Rows' weights over entries first .. end - 1 (first a multiple of 4) added to what they
// gathered; in LDS their references (log2 units) and the reciprocals of their sums.
template <int NT>
__device__ __forceinline__ void ed_weights(const EdKP &p, int64_t pair, int32_t slot, int32_t first, int32_t end,
                                           const float *ref, const float *inv) {
  const float *s = p.scores + pair * p.G * p.cs;
  float *w = p.weights + pair * p.C;
  for (int32_t i = first + 4 * (int32_t)threadIdx.x; i < end; i += 4 * NT) {
    const bool whole = i + 4 <= end;
    float sum[4], old[4];
    if (whole) {
      const ed_f4 o = *(const ed_f4 *)(w + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) old[e] = o[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) old[e] = i + e < end ? w[i + e] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] = 0.f;
#pragma unroll 4
    for (int g = 0; g < p.G; ++g) {
      const float4 x = *(const float4 *)(s + g * p.cs + i);  // (scores are there for whole rounds)
      const float m = ref[g], f = inv[g];
      sum[0] += fast_exp2(__builtin_fmaf(x.x, p.qscale, -m)) * f;
      sum[1] += fast_exp2(__builtin_fmaf(x.y, p.qscale, -m)) * f;
      sum[2] += fast_exp2(__builtin_fmaf(x.z, p.qscale, -m)) * f;
      sum[3] += fast_exp2(__builtin_fmaf(x.w, p.qscale, -m)) * f;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] = (i + e == slot ? 0.f : old[e]) + sum[e];
    if (whole) {
      *(ed_f4 *)(w + i) = ed_f4{sum[0], sum[1], sum[2], sum[3]};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < end) w[i + e] = sum[e];
    }
    if (slot >= i && slot < min(i + 4, end)) p.positions[pair * p.C + slot] = p.pos[pair / p.Hkv];
  }
}

template <class T, int D>
__global__ __launch_bounds__(256, 2) void evict_decode_kernel(EdKP p) {
  typedef FewRows<T, D, true> FR;
  typedef typename FR::elem elem;
  constexpr int NW = 4;
  constexpr int LDS_MERGE = NW * (FR::VALS + 32) * 4;
  constexpr int LDS = NW * FR::LDS_BYTES > LDS_MERGE ? NW * FR::LDS_BYTES : LDS_MERGE;
  __shared__ __align__(16) char smem[LDS];
  __shared__ float ref[16], inv[16];
  __shared__ uint32_t s_bad;  // rows whose sums are not finite
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t pair = blockIdx.x / (uint32_t)p.splits;
  const int split = (int)(blockIdx.x % (uint32_t)p.splits);
  const int b = (int)(pair / p.Hkv), kvh = (int)(pair % p.Hkv);
  const int32_t held = ed_held(p, b), n = min(held + 1, p.C);
  const int32_t slot = __builtin_amdgcn_readfirstlane(held < p.C ? held : ed_victim<256>(p, pair, p.pos[b]));
  if (p.splits > 1 && split == 0 && threadIdx.x == 0) p.slots[pair] = slot;

  const elem *kn = (const elem *)p.k_new + b * p.kn_sb + kvh * p.kn_sh;
  const elem *vn = (const elem *)p.v_new + b * p.vn_sb + kvh * p.vn_sh;
  elem *kc = (elem *)p.k + pair * p.C * D, *vc = (elem *)p.v + pair * p.C * D;
  const int row = min(lane & 15, p.G - 1);
  FR fr;
  fr.begin((const elem *)p.q + b * p.q_sb + (kvh * p.G + row) * p.q_sh);
  const int rounds = (n + FR::RK - 1) / FR::RK;
  const int r0 = (int)((int64_t)rounds * split / p.splits), r1 = (int)((int64_t)rounds * (split + 1) / p.splits);
  float *sc = p.scores + (pair * p.G + row) * p.cs;
  const bool put = (lane & 15) < p.G;
  if (threadIdx.x == 0) s_bad = 0u;
  auto krow = [&](int key) -> const elem * { return key == slot ? kn : kc + (int64_t)key * D; };
  auto vrow = [&](int key) -> const elem * { return key == slot ? vn : vc + (int64_t)key * D; };
  fr.walk(r0 + w, NW, r1, n, n - 1, p.qscale, (elem *)(smem + w * FR::LDS_BYTES), krow, vrow,
          [&](int key, f32x4 s) { if (put) *(f32x4 *)(sc + key) = s; });
  // the new token's rows, by the part that holds its slot
  if (slot / FR::RK >= r0 && slot / FR::RK < r1 && w == 0) {
    constexpr int CHE = FR::CHE;
    if (lane < D / CHE) {
      *(uint4 *)(kc + (int64_t)slot * D + CHE * lane) = *(const uint4 *)(kn + CHE * lane);
      *(uint4 *)(vc + (int64_t)slot * D + CHE * lane) = *(const uint4 *)(vn + CHE * lane);
    }
  }
  __syncthreads();  // the waves' staged rows are read (and their scores written)
  float *ml = (float *)smem, *vals = ml + NW * 32;
  fr.put(ml + w * 32, vals + w * FR::VALS);
  __syncthreads();
  const float ninf = __int_as_float(0xff800000);
  for (int e = threadIdx.x; e < p.G * D; e += 256) {
    const int g = e / D, d = e % D;
    float m = ninf;
#pragma unroll
    for (int x = 0; x < NW; ++x) m = fmaxf(m, ml[x * 32 + 2 * g]);
    float l = 0.f, a = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const float f = fast_exp2(ml[x * 32 + 2 * g] - (m == ninf ? 0.f : m));
      l = __builtin_fmaf(ml[x * 32 + 2 * g + 1], f, l);
      a = __builtin_fmaf(vals[x * FR::VALS + g * (D + 4) + d], f, a);
    }
    // (with scores that are not numbers, l is not, and the row stands)
    if (!(fabsf(a) < __int_as_float(0x7f800000)) && l > 0.f && l < __int_as_float(0x7f800000)) atomicOr(&s_bad, 1u << g);
    if (l == 0.f) a = 0.f;  // (every score -inf)
    if (p.splits > 1) {
      const int64_t at = (pair * p.splits + split) * p.G + g;
      p.vals[at * D + d] = a;
      if (d == 0) {
        p.ml[2 * at] = m;
        p.ml[2 * at + 1] = l;
      }
    } else {
      store_from_f32(p.out, b * p.o_sb + (kvh * p.G + g) * p.o_sh + d, p.out_dt, a / l);
      if (d == 0) {
        ref[g] = m;
        inv[g] = 1.f / l;
      }
    }
  }
  __syncthreads();
  if (s_bad != 0u) {
    uint32_t *marks = (uint32_t *)smem;  // (of which all is read)
    if (threadIdx.x < D) marks[threadIdx.x] = 0u;
    wait_vmcnt<0>();
    __syncthreads();  // (every wave's stores are done, which those below replace)
    few_marks<elem, D, NW>(marks, vrow, r0 * FR::RK, min(n, r1 * FR::RK));
    __syncthreads();
    for (int e = threadIdx.x; e < p.G * D; e += 256) {
      const int g = e / D, d = e % D;
      if (!((s_bad >> g) & 1u) || marks[d] == 0u) continue;
      const float a = few_mark(marks[d]);
      if (p.splits > 1) p.vals[((pair * p.splits + split) * p.G + g) * D + d] = a;
      else store_from_f32(p.out, b * p.o_sb + (kvh * p.G + g) * p.o_sh + d, p.out_dt, a);
    }
  }
  if (p.splits > 1) return;
  ed_weights<256>(p, pair, slot, 0, n, ref, inv);
}

// Parts joined: a pair's output and the weights of 1024 entries a workgroup.
constexpr int ED_CHUNK = 1024;
template <int D>
__global__ __launch_bounds__(256) void evict_join_kernel(EdKP p) {
  __shared__ float ref[16], inv[16], part[16][64];  // part: what each part's values count for
  const int64_t pair = blockIdx.x / (uint32_t)p.chunks;
  const int chunk = (int)(blockIdx.x % (uint32_t)p.chunks), lane = threadIdx.x & 63;
  const int b = (int)(pair / p.Hkv), kvh = (int)(pair % p.Hkv);
  const int32_t n = min(ed_held(p, b) + 1, p.C), slot = p.slots[pair];
  const float ninf = __int_as_float(0xff800000);
  const float2 *ml = (const float2 *)p.ml + pair * p.splits * p.G;
  for (int g = threadIdx.x >> 6; g < p.G; g += 4) {  // a lane a part
    const float2 x = lane < p.splits ? ml[lane * p.G + g] : float2{ninf, 0.f};
    float m = x.x;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    const float f = fast_exp2(x.x - (m == ninf ? 0.f : m)), f_l = 1.f / group_sum<64>(x.y * f);
    part[g][lane] = f * f_l;
    if (lane == 0) {
      ref[g] = m;
      inv[g] = f_l;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x + 256 * chunk; e < p.G * D; e += 256 * p.chunks) {
    const int g = e / D, d = e % D;
    const float *v = p.vals + (pair * p.splits * p.G + g) * D + d;
    float a = 0.f;
#pragma unroll 8
    for (int x = 0; x < p.splits; ++x) a = __builtin_fmaf(v[(int64_t)x * p.G * D], part[g][x], a);
    store_from_f32(p.out, b * p.o_sb + (kvh * p.G + g) * p.o_sh + d, p.out_dt, a);
  }
  ed_weights<256>(p, pair, slot, chunk * ED_CHUNK, min(n, (chunk + 1) * ED_CHUNK), ref, inv);
}

// ------------------------------------------------------------------ host ----
struct EdPlan {
  int64_t splits = 1, cs = 0;
  size_t slots = 0, ml = 0, vals = 0, scores = 0, bytes = 0;
};

static EdPlan ed_plan(const la_evict_decode_args *a) {
  EdPlan pl;
  const int64_t pairs = a->B * a->Hkv, G = a->Hq / a->Hkv;
  // two workgroups a CU, parts of at least 256 entries
  pl.splits = std::max<int64_t>(1, std::min<int64_t>({(int64_t)2 * num_cus() / pairs, a->C / 256, 64}));
  pl.cs = ceil_div(a->C, 32) * 32;
  size_t at = 0;
  auto take = [&](size_t n) { const size_t o = at; at += (n + 255) / 256 * 256; return o; };
  pl.scores = take((size_t)(pairs * G * pl.cs) * sizeof(float));
  if (pl.splits > 1) {
    pl.slots = take((size_t)pairs * sizeof(int32_t));
    pl.ml = take((size_t)(pairs * pl.splits * G * 2) * sizeof(float));
    pl.vals = take((size_t)(pairs * pl.splits * G * a->D) * sizeof(float));
  }
  pl.bytes = at;
  return pl;
}

static int ed_check(const la_evict_decode_args *a) {
  LA_REQUIRE(a != nullptr, "la_evict_decode: null args");
  LA_REQUIRE(a->B > 0 && a->Hq > 0 && a->Hkv > 0 && a->C > 0, "la_evict_decode: sizes must be positive");
  LA_REQUIRE(a->Hq % a->Hkv == 0 && a->Hq / a->Hkv <= 16, "la_evict_decode: Hq must be 1 to 16 times Hkv");
  LA_REQUIRE(a->D == 64 || a->D == 128, "la_evict_decode: head_dim %lld (64 or 128)", (long long)a->D);
  LA_REQUIRE(a->dtype == LA_F32 || a->dtype == LA_BF16 || a->dtype == LA_F16, "la_evict_decode: dtype");
  LA_REQUIRE(a->out_dtype == a->dtype || a->out_dtype == LA_F32, "la_evict_decode: out_dtype is dtype or fp32");
  LA_REQUIRE(a->scale > 0.f && a->scale < 1e30f, "la_evict_decode: scale must be positive");
  LA_REQUIRE(a->recent >= 0 && a->sink >= 0 && a->recent + a->sink < a->C,
             "la_evict_decode: sink + recent must leave an entry of the cache to evict");
  LA_REQUIRE(a->C < ((int64_t)1 << 24) && a->B * a->Hkv < ((int64_t)1 << 24), "la_evict_decode: too many entries");
  return LA_OK;
}

template <class T, int D>
static void ed_launch(const EdKP &p, int64_t pairs, hipStream_t st) {
  evict_decode_kernel<T, D><<<(uint32_t)(pairs * p.splits), 256, 0, st>>>(p);
}

}  // namespace la

extern "C" size_t la_evict_decode_workspace(const la_evict_decode_args *a) {
  if (la::ed_check(a) != LA_OK) return 0;
  return la::ed_plan(a).bytes;
}

extern "C" int la_evict_decode(const la_evict_decode_args *a, void *stream) {
  using namespace la;
  if (int rc = ed_check(a)) return rc;
  LA_REQUIRE(a->q && a->k_new && a->v_new && a->k && a->v && a->weights && a->positions && a->lengths && a->pos && a->out,
             "la_evict_decode: null pointer");
  const int64_t n16 = a->dtype == LA_F32 ? 4 : 8;
  auto ok = [&](const void *x, int64_t sb, int64_t sh, int64_t heads) {
    return (uintptr_t)x % 16 == 0 && (a->B == 1 || sb % n16 == 0) && (heads == 1 || sh % n16 == 0);
  };
  LA_REQUIRE(ok(a->q, a->q_sb, a->q_sh, a->Hq) && ok(a->k_new, a->kn_sb, a->kn_sh, a->Hkv) &&
                 ok(a->v_new, a->vn_sb, a->vn_sh, a->Hkv) && (uintptr_t)a->k % 16 == 0 && (uintptr_t)a->v % 16 == 0,
             "la_evict_decode: rows must be 16-byte aligned");
  const int64_t es = a->dtype == LA_F32 ? 4 : 2, os = a->out_dtype == LA_F32 ? 4 : 2, slots = a->B * a->Hkv * a->C;
  auto rows = [&](const void *x, int64_t e, int64_t sb, int64_t sh, int64_t heads) {
    return Cover(x, a->D * e, {sb * e, a->B}, {sh * e, heads});
  };
  const Cover cov[] = {Cover(a->k, slots * a->D * es), Cover(a->v, slots * a->D * es), Cover(a->weights, slots * 4),
                       Cover(a->positions, slots * 4), rows(a->out, os, a->o_sb, a->o_sh, a->Hq),  // written
                       rows(a->q, es, a->q_sb, a->q_sh, a->Hq), rows(a->k_new, es, a->kn_sb, a->kn_sh, a->Hkv),
                       rows(a->v_new, es, a->vn_sb, a->vn_sh, a->Hkv), Cover(a->lengths, a->B * 4), Cover(a->pos, a->B * 4)};
  for (int i = 0; i < 5; ++i)
    for (int j = i + 1; j < 10; ++j)
      LA_REQUIRE(!overlap(cov[i], cov[j]), "la_evict_decode: caches, weights, positions, out or inputs share memory");
  const EdPlan pl = ed_plan(a);
  if (!a->workspace || a->ws_bytes < (int64_t)pl.bytes)
    return fail(LA_ERR_WORKSPACE, "la_evict_decode: workspace %lld < %lld bytes", (long long)a->ws_bytes,
                (long long)pl.bytes);
  LA_REQUIRE((uintptr_t)a->workspace % 256 == 0, "la_evict_decode: workspace alignment");
  const int64_t pairs = a->B * a->Hkv;
  EdKP p{};
  p.q = a->q; p.k_new = a->k_new; p.v_new = a->v_new; p.k = a->k; p.v = a->v; p.out = a->out;
  p.weights = a->weights; p.positions = a->positions; p.lengths = a->lengths; p.pos = a->pos;
  char *ws = (char *)a->workspace;
  p.scores = (float *)(ws + pl.scores);
  p.slots = (int32_t *)(ws + pl.slots);
  p.ml = (float *)(ws + pl.ml);
  p.vals = (float *)(ws + pl.vals);
  p.q_sb = a->q_sb; p.q_sh = a->q_sh; p.kn_sb = a->kn_sb; p.kn_sh = a->kn_sh;
  p.vn_sb = a->vn_sb; p.vn_sh = a->vn_sh; p.o_sb = a->o_sb; p.o_sh = a->o_sh;
  p.recent = a->recent; p.sink = a->sink; p.cs = pl.cs;
  p.B = (int32_t)a->B; p.Hq = (int32_t)a->Hq; p.Hkv = (int32_t)a->Hkv; p.G = (int32_t)(a->Hq / a->Hkv);
  p.C = (int32_t)a->C; p.splits = (int32_t)pl.splits; p.out_dt = a->out_dtype;
  p.chunks = (int32_t)ceil_div(a->C, ED_CHUNK);
  p.qscale = a->scale * 1.44269504088896340736f;
  hipStream_t st = (hipStream_t)stream;
  const bool d128 = a->D == 128;
  if (a->dtype == LA_F32) d128 ? ed_launch<DaF32, 128>(p, pairs, st) : ed_launch<DaF32, 64>(p, pairs, st);
  else if (a->dtype == LA_BF16) d128 ? ed_launch<DaBf16, 128>(p, pairs, st) : ed_launch<DaBf16, 64>(p, pairs, st);
  else d128 ? ed_launch<DaF16, 128>(p, pairs, st) : ed_launch<DaF16, 64>(p, pairs, st);
  LA_LAUNCHED();
  if (pl.splits > 1) {
    const uint32_t grid = (uint32_t)(pairs * p.chunks);
    if (d128) evict_join_kernel<128><<<grid, 256, 0, st>>>(p);
    else evict_join_kernel<64><<<grid, 256, 0, st>>>(p);
    LA_LAUNCHED();
  }
  return LA_OK;
}
