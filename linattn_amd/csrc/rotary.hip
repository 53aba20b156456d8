// Rows of q and k turned by their positions (la_rotary).
//
// A workgroup takes `ts` tokens: their angles once, into LDS (a position times every
// frequency, shared by all heads), then their heads' rows, `hs` heads at a time, each row by
// as many lanes as it has units.  Bound by the rows' reads and writes: 12345
// tokens of 32 heads of 80 fp16 values 27 to 31 us (4.7 to 4.1 TB/s; a large copy has 4.9), 32768 of
// 40 heads of 128 bf16 values 129 us (5.2 TB/s); one token 4.3 us, the chain from its position to its rows.
#include <algorithm>

#include "rotary.h"

namespace la {

struct RoKP {
  RoAngles an;
  const void *q, *k;
  void *q_out, *k_out;
  int64_t tokens, T;
  int64_t q_sb, q_sh, q_st, k_sb, k_sh, k_st, qo_sb, qo_sh, qo_st, ko_sb, ko_sh, ko_st;
  int32_t Hq, Hkv, D, units, ts, hs;
};

template <class E, int V>
__global__ __launch_bounds__(RO_NT) void rotary_kernel(RoKP p) {
  typedef RoUnit<E, V> U;
  extern __shared__ float2 cs[];
  const int tid = threadIdx.x, n = p.an.n;
  const int64_t tok0 = (int64_t)blockIdx.x * p.ts;
  const int slot = tid / p.units, u = tid - slot * p.units;
  const int ti = slot / p.hs, h0 = slot % p.hs, H = p.Hq + p.Hkv;
  const int64_t tok = tok0 + ti, b = tok / p.T, t = tok - b * p.T;
  const bool live = ti < p.ts && tok < p.tokens;
  const U unit(u, p.D, n, p.an.interleaved);
  constexpr int AHEAD = 4;  // rows on their way at a time
  typename U::vec xa[AHEAD], xb[AHEAD];
  auto load = [&](int h, typename U::vec &a, typename U::vec &c) {
    unit.load(h < p.Hq ? (const E *)p.q + b * p.q_sb + t * p.q_st + h * p.q_sh
                       : (const E *)p.k + b * p.k_sb + t * p.k_st + (h - p.Hq) * p.k_sh, a, c);
  };
  if (live)
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (h0 + i * p.hs < H) load(h0 + i * p.hs, xa[i], xb[i]);
  for (int e = tid; e < p.ts * n; e += RO_NT) {
    const int64_t x = tok0 + e / n;
    const int f = e % n;
    if (x < p.tokens) {
      const int64_t xb_ = x / p.T;
      cs[e] = p.an.turn((double)p.an.pos[p.an.axis(f) * p.an.p_sa + xb_ * p.an.p_sb + (x - xb_ * p.T) * p.an.p_st], f);
    }
  }
  __syncthreads();
  if (!live) return;
  RoTurns<V> turns;
  turns.load(cs + ti * n, unit.f0);
  for (int h = h0; h < H; h += AHEAD * p.hs) {
    if (h != h0)
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (h + i * p.hs < H) load(h + i * p.hs, xa[i], xb[i]);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int hi = h + i * p.hs;
      if (hi >= H) break;
      float x[2 * V];
      U::widen(xa[i], xb[i], x);
      if (unit.f0 >= 0) turns.apply(x, p.an.interleaved);
      unit.store(hi < p.Hq ? (E *)p.q_out + b * p.qo_sb + t * p.qo_st + hi * p.qo_sh
                           : (E *)p.k_out + b * p.ko_sb + t * p.ko_st + (hi - p.Hq) * p.ko_sh, x);
    }
  }
}

static int ro_rows_ok(const char *what, const void *x, int64_t esz) {
  LA_REQUIRE(x != nullptr && (uintptr_t)x % esz == 0, "la_rotary: null or unaligned %s", what);
  return LA_OK;
}

template <class E, int V>
static int ro_launch(RoKP p, hipStream_t st) {
  p.units = RoUnit<E, V>::count(p.D, p.an.n);
  const int slots = RO_NT / p.units, H = p.Hq + p.Hkv;
  LA_REQUIRE(slots > 0, "la_rotary: head_dim %d needs rows whose chunks are aligned", p.D);
  // tokens of a workgroup: about four rows a lane, where there are tokens for every CU (with two 27.6 us
  // and 143, with eight 27.8 and 130, in place of 26.8 and 128.6)
  p.ts = (int)std::min<int64_t>(std::max(1, 4 * slots / H), std::max<int64_t>(1, p.tokens / (2 * num_cus())));
  p.ts = std::min(p.ts, slots);
  p.hs = std::min(H, slots / p.ts);
  const int64_t wgs = ceil_div(p.tokens, p.ts);
  LA_REQUIRE(grid_fits(wgs, RO_NT), "la_rotary: too many tokens");
  const size_t lds = (size_t)p.ts * p.an.n * sizeof(float2);
  rotary_kernel<E, V><<<dim3((uint32_t)wgs), RO_NT, lds, st>>>(p);
  LA_LAUNCHED();
  return LA_OK;
}

}  // namespace la

extern "C" int la_rotary(const la_rotary_args *args, void *stream) {
  using namespace la;
  LA_REQUIRE(args != nullptr, "la_rotary: null args");
  la_rotary_args x = *args;
  la_rotary_args *a = &x;
  LA_REQUIRE(a->B >= 0 && a->T >= 0 && a->Hq > 0 && a->Hkv >= 0 && a->D > 0 && a->n > 0 && a->A > 0,
             "la_rotary: sizes must be positive");
  LA_REQUIRE(a->D <= 512 && 2 * a->n <= a->D, "la_rotary: head_dim up to 512, at most half as many frequencies");
  LA_REQUIRE(a->Hq + a->Hkv < 65536 && a->A < 65536, "la_rotary: too many heads");
  LA_REQUIRE(a->dtype == LA_F32 || a->dtype == LA_BF16 || a->dtype == LA_F16, "la_rotary: dtype");
  if (a->B == 0 || a->T == 0) return LA_OK;
  LA_REQUIRE(a->B < ((int64_t)1 << 31) / a->T, "la_rotary: too many tokens");
  const int64_t esz = a->dtype == LA_F32 ? 4 : 2;
  if (int rc = ro_rows_ok("q", a->q, esz)) return rc;
  if (int rc = ro_rows_ok("q_out", a->q_out, esz)) return rc;
  if (a->Hkv > 0) {
    if (int rc = ro_rows_ok("k", a->k, esz)) return rc;
    if (int rc = ro_rows_ok("k_out", a->k_out, esz)) return rc;
  }
  LA_REQUIRE(a->positions && a->inv_freq && (a->axes || a->A == 1), "la_rotary: null positions, frequencies or axes");
  auto flat = [&](int64_t &b, int64_t &h, int64_t &t, int64_t heads) {  // strides that nothing takes a step by
    if (a->B == 1) b = 0;
    if (heads <= 1) h = 0;
    if (a->T == 1) t = 0;
  };
  flat(a->q_sb, a->q_sh, a->q_st, a->Hq);
  flat(a->qo_sb, a->qo_sh, a->qo_st, a->Hq);
  flat(a->k_sb, a->k_sh, a->k_st, a->Hkv);
  flat(a->ko_sb, a->ko_sh, a->ko_st, a->Hkv);
  auto cover = [&](const void *x, int64_t b, int64_t h, int64_t t, int64_t heads) {
    return Cover(x, a->D * esz, {b * esz, a->B}, {h * esz, heads}, {t * esz, a->T});
  };
  // in place: the same rows, each of which one lane reads before it writes
  const bool q_in = a->q_out == a->q && a->qo_sb == a->q_sb && a->qo_sh == a->q_sh && a->qo_st == a->q_st;
  const bool k_in = a->k_out == a->k && a->ko_sb == a->k_sb && a->ko_sh == a->k_sh && a->ko_st == a->k_st;
  const void *k = a->Hkv > 0 ? a->k : nullptr, *k_out = a->Hkv > 0 ? a->k_out : nullptr;
  const Cover written[] = {cover(a->q_out, a->qo_sb, a->qo_sh, a->qo_st, a->Hq), cover(k_out, a->ko_sb, a->ko_sh, a->ko_st, a->Hkv)};
  const Cover read[] = {cover(q_in ? nullptr : a->q, a->q_sb, a->q_sh, a->q_st, a->Hq),
                        cover(k_in ? nullptr : k, a->k_sb, a->k_sh, a->k_st, a->Hkv),
                        Cover(a->positions, 4, {a->p_sa * 4, a->A}, {a->p_sb * 4, a->B}, {a->p_st * 4, a->T}),
                        Cover(a->inv_freq, a->n * 4),
                        Cover(a->axes, a->n * 4)};
  LA_REQUIRE(!overlap_any(written, read), "la_rotary: an output shares memory with another argument");
  RoKP p{};
  p.an = RoAngles{a->positions, a->axes, a->inv_freq, a->p_sa, a->p_sb, a->p_st, (int32_t)a->n, (int32_t)a->A,
                  a->interleaved != 0, a->inverse != 0};
  p.q = a->q; p.k = a->k; p.q_out = a->q_out; p.k_out = a->k_out;
  p.tokens = a->B * a->T; p.T = a->T;
  p.q_sb = a->q_sb; p.q_sh = a->q_sh; p.q_st = a->q_st;
  p.k_sb = a->k_sb; p.k_sh = a->k_sh; p.k_st = a->k_st;
  p.qo_sb = a->qo_sb; p.qo_sh = a->qo_sh; p.qo_st = a->qo_st;
  p.ko_sb = a->ko_sb; p.ko_sh = a->ko_sh; p.ko_st = a->ko_st;
  p.Hq = (int32_t)a->Hq; p.Hkv = (int32_t)a->Hkv; p.D = (int32_t)a->D;
  uint64_t at = (uint64_t)(uintptr_t)a->q | (uint64_t)(uintptr_t)a->q_out;
  uint64_t by = (uint64_t)(a->q_sb | a->q_sh | a->q_st | a->qo_sb | a->qo_sh | a->qo_st);
  if (a->Hkv > 0) {
    at |= (uint64_t)(uintptr_t)a->k | (uint64_t)(uintptr_t)a->k_out;
    by |= (uint64_t)(a->k_sb | a->k_sh | a->k_st | a->ko_sb | a->ko_sh | a->ko_st);
  }
  hipStream_t st = (hipStream_t)stream;
  const int v = ro_vector((int)esz, a->D, a->n, at, by);
  if (a->dtype == LA_F32) return v == 4 ? ro_launch<float, 4>(p, st) : ro_launch<float, 1>(p, st);
  if (a->dtype == LA_BF16)
    return v == 8 ? ro_launch<__bf16, 8>(p, st) : v == 4 ? ro_launch<__bf16, 4>(p, st) : ro_launch<__bf16, 1>(p, st);
  return v == 8 ? ro_launch<_Float16, 8>(p, st) : v == 4 ? ro_launch<_Float16, 4>(p, st) : ro_launch<_Float16, 1>(p, st);
}
