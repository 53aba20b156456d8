"""Rotary positions, their append to a paged cache and attention over it as a server runs them: prompts
in chunks beside the tokens of other sequences, step after step, bf16 and fp8 caches; Quest over the
bounds that the appends kept; a decode step in a graph.  Every step's keys are held against their
64-bit turns, and its outputs against 64-bit attention over what the pages hold."""

from __future__ import annotations

import pytest
import torch

from dense_reference import HALF_STEP, attention
from dense_reference import close as close_to
from linattn_amd.kernels.block_sparse import fp8_scale_pairs, sparse_attention
from linattn_amd.kernels.dense import paged_attention
from linattn_amd.kernels.kv_cache import rotary_kv_append
from linattn_amd.kernels.quest_pages import alloc_page_meta, page_update_hip, quest_select_hip
from rotary_reference import close, rounded, turn

pytestmark = pytest.mark.gpu

HQ, HKV, D, PAGE = 8, 2, 128, 16


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


class Server:
    """Pages given out as sequences grow."""

    def __init__(self, dev, B, pages, fp8, seed):
        self.dev, self.B, self.fp8 = dev, B, fp8
        self.g = torch.Generator().manual_seed(seed)
        self.order = torch.randperm(B * pages, generator=self.g).tolist()
        shape = (B * pages, HKV, PAGE, D)
        kind = torch.float8_e4m3fn if fp8 else torch.bfloat16
        self.k, self.v = (torch.full(shape, float("nan"), device=dev).to(kind) for _ in "kv")
        self.ks, self.vs = fp8_scale_pairs(*shape[:3], dev) if fp8 else (None, None)
        self.table = torch.full((B, pages), -1, dtype=torch.int32, device=dev)
        self.held = [0] * B
        self.freq = (10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))).float()
        self.mn = self.mx = None
        if not fp8:
            self.mn, self.mx = alloc_page_meta(B, HKV, pages, D, torch.bfloat16, dev)
        self.keys = [[torch.zeros(0, HKV, D)] for _ in range(B)]  # turned, 64 bits

    def scales(self):
        return dict(k_scale=self.ks, v_scale=self.vs) if self.fp8 else {}

    def cached(self, b):
        """K and V of sequence b (Hkv, n, D) as the pages hold them, 64 bits, on the CPU."""
        n = self.held[b]
        pages = self.table[b, :-(-n // PAGE)].long()
        r = []
        for pool, s in ((self.k, self.ks), (self.v, self.vs)):
            x = pool.view(torch.uint8)[pages].view(pool.dtype).double() if self.fp8 else pool[pages].double()
            if self.fp8:
                x = x * s[pages][..., None].double()
            r.append(x.transpose(0, 1).flatten(1, 2)[:, :n].cpu())
        return r

    def step(self, lq):
        N, B, dev = sum(lq), self.B, self.dev
        for b in range(B):
            for i in range(-(-self.held[b] // PAGE), -(-(self.held[b] + lq[b]) // PAGE)):
                self.table[b, i] = self.order.pop()
        q, k, v = (torch.randn(N, h, D, generator=self.g).bfloat16() for h in (HQ, HKV, HKV))
        cu = _i32([sum(lq[:b]) for b in range(B + 1)], dev)
        more = self.scales() if self.fp8 else dict(page_min=self.mn, page_max=self.mx, page_size=PAGE)
        gq = rotary_kv_append(q.to(dev), k.to(dev), v.to(dev), self.k, self.v, self.table, _i32(self.held, dev),
                              self.freq.to(dev), cu_seqlens=cu, **more)
        before = list(self.held)
        self.held = [x + y for x, y in zip(self.held, lq)]
        out, lse = paged_attention(gq, self.k, self.v, self.table, _i32(self.held, dev), cu, return_lse=True, **self.scales())
        a = 0
        for b, n in enumerate(lq):
            at = torch.arange(before[b], before[b] + n)
            wq, tq = turn(q[a:a + n], at, self.freq)
            close(gq[a:a + n], wq, rounded(wq, tq, torch.bfloat16), f"q of {b}")
            ck, cv = self.cached(b)
            wk, tk = turn(k[a:a + n], at, self.freq)
            if not self.fp8:
                close(ck[:, before[b]:].transpose(0, 1), wk, rounded(wk, tk, torch.bfloat16), f"keys of {b}")
                assert torch.equal(cv[:, before[b]:].transpose(0, 1), v[a:a + n].double())
            else:  # (half a step of e4m3 of what was scaled, 2^-10 of the scale below its normal range)
                top = wk.abs().amax(-1, keepdim=True)
                close(ck[:, before[b]:].transpose(0, 1), wk, tk + wk.abs() * (2.0 ** -4 + 1e-6) + top / 448 * 2.0 ** -9, f"keys of {b}")
            for h in range(HQ):
                o, ls, tol, tol_l = attention(gq[a:a + n, h].cpu(), ck[h // (HQ // HKV)], cv[h // (HQ // HKV)], True, None,
                                              HALF_STEP[torch.bfloat16])
                close_to(out[a:a + n, h].cpu(), o, tol, f"out of {b}")
                close_to(lse[h, a:a + n].cpu(), ls, tol_l, f"lse of {b}")
            a += n
        return gq, out


@pytest.mark.parametrize("fp8", [False, True])
def test_prompts_in_chunks_beside_tokens(dev, fp8):
    s = Server(dev, 4, 20, fp8, 1)
    s.step([37, 0, 1, 90])
    s.step([1, 70, 15, 1])
    s.step([1, 64, 1, 1])
    for _ in range(3):
        s.step([1, 1, 1, 1])
    if fp8:
        return
    # the bounds that the appends kept are those of the pages
    for b in range(4):
        n = s.held[b]
        ck, _ = s.cached(b)
        mn, mx = page_update_hip(ck.bfloat16()[None].to(dev), PAGE)
        assert torch.equal(s.mn[b, :, :-(-n // PAGE)], mn[0]) and torch.equal(s.mx[b, :, :-(-n // PAGE)], mx[0])
    # Quest over all pages reads what dense attention does
    q = torch.randn(4, HQ, 1, D, generator=s.g).bfloat16().to(dev)
    n = _i32(s.held, dev)
    ids, counts = quest_select_hip(q, s.mn, s.mx, page_size=PAGE, topk=20, offset=max(s.held) - 1, positions=n - 1)
    sparse = sparse_attention(q, s.k, s.v, ids, unit=PAGE, counts=counts, page_table=s.table, page_size=PAGE, kv_len=n,
                              out_dtype=torch.float32)
    dense = paged_attention(q, s.k, s.v, s.table, n, out_dtype=torch.float32)
    assert (sparse - dense).abs().max() < 2e-3  # (the bound both are held to against 64 bits)


@pytest.mark.parametrize("fp8", [False, True])
def test_a_captured_decode_step(dev, fp8):
    """Append and attention in one graph, replayed as the sequences grow, between eager work."""
    s = Server(dev, 3, 12, fp8, 2)
    s.step([40, 9, 1])
    for b in range(3):
        for i in range(-(-s.held[b] // PAGE), 12):
            s.table[b, i] = s.order.pop()
    pools = [s.k, s.v]
    twins = [x.clone() for x in pools]
    scales = s.scales()
    scales2 = {}
    if fp8:
        a, b = fp8_scale_pairs(*s.ks.shape, dev)
        a.copy_(s.ks)
        b.copy_(s.vs)
        scales2 = dict(k_scale=a, v_scale=b)
    q, k, v = (torch.randn(3, h, 1, D, generator=s.g).bfloat16().to(dev) for h in (HQ, HKV, HKV))
    pos, freq = _i32(s.held, dev), s.freq.to(dev)
    n = pos + 1
    out = torch.empty_like(q)

    def decode(kp, vp, sc, out):
        gq = rotary_kv_append(q, k, v, kp, vp, s.table, pos, freq, **sc)
        return paged_attention(gq, kp, vp, s.table, n, out=out, **sc)

    decode(*[x.clone() for x in twins], scales2, torch.empty_like(q))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decode(*twins, scales2, out)
    raw = lambda x: x.view(torch.uint8) if fp8 else x.view(torch.int16)
    for i in range(5):
        want = decode(*pools, scales, torch.empty_like(q))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        for a, b in zip(pools, twins):
            assert torch.equal(raw(a), raw(b)), i
        q.copy_(torch.randn(q.shape, generator=s.g))
        k.copy_(torch.randn(k.shape, generator=s.g))
        pos.add_(1)
        n.add_(1)


@pytest.mark.parametrize("kind,D,page", [("bf16", 128, 64), ("bf16", 128, 24), ("fp32", 64, 64), ("fp8", 128, 64)])
def test_pools_past_4_gib(dev, kind, D, page):
    """Pages more than 2^32 bytes into their pools: the bits are those of small pools."""
    Hq, Hkv, lq, before = 16, 8, [40, 1, 7], [100, 900, 0]
    dtype = torch.float32 if kind == "fp32" else torch.bfloat16
    held = torch.float8_e4m3fn if kind == "fp8" else dtype
    size = Hkv * page * D * torch.empty((), dtype=held).element_size()
    P = 1000 // page + 1
    table = torch.arange(3 * P, dtype=torch.int32).view(3, P)
    g = torch.Generator().manual_seed(9)
    q, k, v = (torch.randn(sum(lq), h, D, generator=g).to(dtype).to(dev) for h in (Hq, Hkv, Hkv))
    old = [torch.randn(3 * P, Hkv, page, D, generator=g).to(held).to(dev) for _ in "kv"]
    olds = torch.rand(2, 3 * P, Hkv, page, generator=g).to(dev)
    cu, pos, freq = _i32([0, 40, 41, 48], dev), _i32(before, dev), torch.rand(D // 2, generator=g).to(dev)
    lengths = _i32([a + b for a, b in zip(before, lq)], dev)
    got = []
    for first in (0, (1 << 32) // size + 1):
        n = first + 3 * P
        pools = [torch.empty(n, Hkv, page, D, dtype=held, device=dev) for _ in "kv"]
        scales = list(fp8_scale_pairs(n, Hkv, page, dev)) if kind == "fp8" else []
        for x, y in zip(pools + scales, old + list(olds)):
            x[first:] = y
        named = dict(zip(("k_scale", "v_scale"), scales))
        t = (table + first).to(dev)
        gq = rotary_kv_append(q, k, v, *pools, t, pos, freq, cu_seqlens=cu, **named)
        out = paged_attention(gq, *pools, t, lengths, cu, **named)
        one = paged_attention(gq[:3, :, None].contiguous(), *pools, t, lengths, **named)  # (single tokens, batched)
        got.append([gq, out, one, *(x[first:].contiguous().view(torch.uint8) for x in pools), *(x[first:].clone() for x in scales)])
    for a, b in zip(*got):
        assert torch.equal(a, b)
