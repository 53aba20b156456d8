// Eviction from a cache by the weights its entries gathered (la_evict_kv): the entries a
// sequence keeps, and their rows copied to a cache of their own.
//
// evict_select_kernel, one workgroup per (sequence, KV head): the budget-th largest key by
// a radix select over the unprotected entries (digits of 11, 11 and 10 bits, a histogram
// in LDS each), then the kept entries in ascending order: every wave owns a stretch of
// the entries, counts its kept ones, and after one exchange writes them from its own
// offset by ballots.  evict_gather_kernel copies the rows, 16 bytes a lane.
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
  int32_t *list;  // [b][h][budget]
  int64_t T, k_sb, k_sh, k_st, v_sb, v_sh, v_st;  // (k, v: bytes)
  int64_t w_sb, w_sh, ps_sb, ps_sh, budget, capacity, recent, sink;
  int32_t B, Hkv, row16;  // row16: 16-byte chunks of a row
};

// Entries of sequence b and its first row.
__device__ __forceinline__ void ev_seq(const EvKP &p, int b, int64_t &first, int32_t &n) {
  if (p.cu) {
    const int64_t a = min(max((int64_t)p.cu[b], (int64_t)0), p.T), e = min(max((int64_t)p.cu[b + 1], (int64_t)0), p.T);
    first = a;
    n = (int32_t)max(e - a, (int64_t)0);
  } else {
    first = 0;
    n = (int32_t)(p.lengths ? min(max((int64_t)p.lengths[b], (int64_t)0), p.T) : p.T);
  }
}

constexpr int EV_NT = 1024, EV_NW = EV_NT / 64, EV_BINS = 2048;

__global__ __launch_bounds__(EV_NT) void evict_select_kernel(EvKP p) {
  __shared__ uint32_t hist[EV_BINS];
  __shared__ uint32_t part[EV_NW][2];
  __shared__ uint32_t found[2];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int b = blockIdx.x / p.Hkv, h = blockIdx.x % p.Hkv;
  int64_t first;
  int32_t n;
  ev_seq(p, b, first, n);
  const float *wr = p.weights + (p.cu ? first : b * p.w_sb) + h * p.w_sh;
  const int32_t *pr = p.positions ? p.positions + (p.cu ? first : b * p.ps_sb) + h * p.ps_sh : nullptr;
  const int64_t pos = p.positions ? p.pos[b] : n;
  const int32_t kept = (int32_t)min((int64_t)n, p.budget);
  int32_t *list = p.list + (int64_t)blockIdx.x * p.budget;
  float *wo = p.w_out + (int64_t)blockIdx.x * p.capacity;
  int32_t *po = p.pos_out + (int64_t)blockIdx.x * p.capacity;
  if (h == 0 && tid == 0) p.len_out[b] = kept;
  for (int64_t i = kept + tid; i < p.capacity; i += EV_NT) {
    wo[i] = 0.f;
    po[i] = -1;
  }
  auto key = [&](int32_t i) -> uint32_t {
    return ev_safe(pr ? pr[i] : i, pos, p.recent, p.sink) ? EV_SAFE : ev_key(wr[i]);
  };
  uint32_t thr = 0, want = 0;  // kept: keys above thr, and the first `want` of those equal
  if (n <= kept) {
    want = (uint32_t)n;
    thr = 0;
    for (int32_t i = tid; i < n; i += EV_NT) {
      list[i] = i;
      wo[i] = wr[i];
      po[i] = pr ? pr[i] : i;
    }
    return;
  }
  // the wave's stretch
  const int32_t seg = ((n + EV_NT - 1) / EV_NT) * 64;
  const int32_t i0 = min(w * seg, n), i1 = min(i0 + seg, n);
  want = (uint32_t)kept;
  int shift = 32;
  constexpr int BITS[3] = {11, 11, 10};
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int bits = pass == 2 ? BITS[2] : BITS[0];
    shift -= bits;
    for (int i = tid; i < EV_BINS; i += EV_NT) hist[i] = 0u;
    __syncthreads();
    for (int32_t i = i0 + lane; i < i1; i += 64) {
      const uint32_t k = key(i);
      if (pass == 0 || (k >> (shift + bits)) == (thr >> (shift + bits)))
        atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1u)], 1u);
    }
    __syncthreads();
    // the highest bin at which the count from above reaches `want`: wave 0, 32 bins a lane
    if (w == 0) {
      const int per = EV_BINS / 64;
      uint32_t sum = 0;
      for (int j = 0; j < per; ++j) sum += hist[(63 - lane) * per + j];
      uint32_t incl = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = (uint32_t)__shfl_up((int)incl, o, 64);
        if (lane >= o) incl += y;
      }
      const uint64_t reach = __ballot(incl >= want);  // (never empty: n > kept entries)
      if (lane == __ffsll((unsigned long long)reach) - 1) {
        uint32_t above = incl - sum;
        int bin = (63 - lane) * per + per - 1;
        while (above + hist[bin] < want) above += hist[bin--];
        found[0] = (uint32_t)bin;
        found[1] = above;
      }
    }
    __syncthreads();
    thr |= found[0] << shift;
    want -= found[1];
    __syncthreads();
  }
  uint32_t gt = 0, eq = 0;
  for (int32_t i = i0; i < i1; i += 64) {
    const bool in = i + lane < i1;
    const uint32_t k = in ? key(i + lane) : 0u;
    gt += __popcll(__ballot(in && k > thr));
    eq += __popcll(__ballot(in && k == thr));
  }
  if (lane == 0) {
    part[w][0] = gt;
    part[w][1] = eq;
  }
  __syncthreads();
  uint32_t gt0 = 0, eq0 = 0;
  for (int x = 0; x < w; ++x) {
    gt0 += part[x][0];
    eq0 += part[x][1];
  }
  for (int32_t i = i0; i < i1; i += 64) {
    const bool in = i + lane < i1;
    const uint32_t k = in ? key(i + lane) : 0u;
    const uint64_t mg = __ballot(in && k > thr), me = __ballot(in && k == thr);
    const uint64_t below = (1ull << lane) - 1ull;
    const uint32_t e = eq0 + __popcll(me & below);
    const bool keep = in && (k > thr || (k == thr && e < want));
    if (keep) {
      const uint32_t at = gt0 + __popcll(mg & below) + min(e, want);
      list[at] = i + lane;
      wo[at] = wr[i + lane];
      po[at] = pr ? pr[i + lane] : i + lane;
    }
    gt0 += __popcll(mg);
    eq0 += __popcll(me);
  }
}

// 64 slots of one (sequence, KV head) a workgroup; K and V.
__global__ __launch_bounds__(256) void evict_gather_kernel(EvKP p, int32_t blocks) {
  const int bh = blockIdx.x / blocks, blk = blockIdx.x % blocks;
  const int b = bh / p.Hkv, h = bh % p.Hkv;
  int64_t first;
  int32_t n;
  ev_seq(p, b, first, n);
  const int32_t kept = (int32_t)min((int64_t)n, p.budget);
  const char *kb = p.k + (p.cu ? first * p.k_st : b * p.k_sb) + h * p.k_sh;
  const char *vb = p.v + (p.cu ? first * p.v_st : b * p.v_sb) + h * p.v_sh;
  const int32_t *list = p.list + (int64_t)bh * p.budget;
  const int64_t out0 = ((int64_t)bh * p.capacity) * p.row16;
  const int64_t s0 = (int64_t)blk * 64, s1 = min(s0 + 64, p.capacity);
  for (int64_t x = s0 * p.row16 + threadIdx.x; x < s1 * p.row16; x += 256) {
    const int64_t slot = x / p.row16;
    const int64_t ch = x % p.row16;
    uint4 kk{0, 0, 0, 0}, vv{0, 0, 0, 0};
    if (slot < kept) {
      const int64_t i = list[slot];
      kk = *(const uint4 *)(kb + i * p.k_st + 16 * ch);
      vv = *(const uint4 *)(vb + i * p.v_st + 16 * ch);
    }
    *(uint4 *)(p.k_out + 16 * (out0 + x)) = kk;
    *(uint4 *)(p.v_out + 16 * (out0 + x)) = vv;
  }
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
                 a->B * a->Hkv * ceil_div(a->capacity, 64) < ((int64_t)1 << 31),
             "la_evict_kv: too many entries");
  LA_REQUIRE(!(a->cu && a->lengths), "la_evict_kv: lengths are for batched calls");
  LA_REQUIRE(!a->positions || a->pos, "la_evict_kv: positions need pos");
  return LA_OK;
}

}  // namespace la

extern "C" size_t la_evict_kv_workspace(const la_evict_args *a) {
  if (la::ev_check(a) != LA_OK) return 0;
  return (size_t)(a->B * a->Hkv * a->budget) * sizeof(int32_t);
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
  const size_t need = la_evict_kv_workspace(a);
  if (!a->workspace || a->ws_bytes < (int64_t)need)
    return fail(LA_ERR_WORKSPACE, "la_evict_kv: workspace %lld < %lld bytes", (long long)a->ws_bytes, (long long)need);
  EvKP p{};
  p.k = (const char *)a->k; p.v = (const char *)a->v; p.weights = a->weights;
  p.positions = a->positions; p.pos = a->pos; p.lengths = a->lengths; p.cu = a->cu;
  p.k_out = (char *)a->k_out; p.v_out = (char *)a->v_out;
  p.w_out = a->w_out; p.pos_out = a->pos_out; p.len_out = a->len_out; p.list = (int32_t *)a->workspace;
  p.T = a->T;
  p.k_sb = a->k_sb * es; p.k_sh = a->k_sh * es; p.k_st = a->k_st * es;
  p.v_sb = a->v_sb * es; p.v_sh = a->v_sh * es; p.v_st = a->v_st * es;
  p.w_sb = a->w_sb; p.w_sh = a->w_sh; p.ps_sb = a->ps_sb; p.ps_sh = a->ps_sh;
  p.budget = a->budget; p.capacity = a->capacity; p.recent = a->recent; p.sink = a->sink;
  p.B = (int32_t)a->B; p.Hkv = (int32_t)a->Hkv; p.row16 = (int32_t)(a->D * es / 16);
  hipStream_t st = (hipStream_t)stream;
  const uint32_t rows = (uint32_t)(a->B * a->Hkv);
  const int32_t blocks = (int32_t)ceil_div(a->capacity, 64);
  evict_select_kernel<<<rows, EV_NT, 0, st>>>(p);
  LA_LAUNCHED();
  evict_gather_kernel<<<rows * (uint32_t)blocks, 256, 0, st>>>(p, blocks);
  LA_LAUNCHED();
  return LA_OK;
}
