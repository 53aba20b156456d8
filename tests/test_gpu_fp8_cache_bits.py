"""``paged_attention`` of fp16 queries over fp8 caches keeps fp16's bits, in chunks as for single tokens:
weights times the values' scales are rounded by half a step of fp16 at most.  A value whose
scale is infinite gives the infinity, or the NaN, of the definition to the queries that see it.
Bounds: see ``dense_reference.attention``."""

from __future__ import annotations

import math

import pytest
import torch

from dense_reference import HALF_STEP, attention, close
from linattn_amd.kernels.dense import paged_attention

pytestmark = pytest.mark.gpu


def _cache(seed, lk, Hkv, D, page, far):
    """Codes and scales in pages of any order (other slots: NaN), and what they stand for."""
    g = torch.Generator().manual_seed(seed)
    pages = [-(-n // page) for n in lk]
    n_phys = sum(pages) + 2
    order = torch.randperm(n_phys, generator=g)
    table = torch.full((len(lk), max(pages) + 1), -5, dtype=torch.int32)
    codes = [torch.full((n_phys, Hkv, page, D), 0x7F, dtype=torch.uint8) for _ in "kv"]
    scales = [torch.full((n_phys, Hkv, page), math.nan) for _ in "kv"]
    held, at = [[], []], 0
    for b, n in enumerate(lk):
        table[b, :pages[b]] = order[at:at + pages[b]]
        at += pages[b]
        for i in range(2):
            x = torch.randn(Hkv, n, D, generator=g)
            if far and i:  # values of very different size
                x *= 10.0 ** (6 * torch.rand(Hkv, n, 1, generator=g) - 4)
            s = x.abs().amax(-1).clamp(min=1e-8) / 448
            c = (x / s[..., None]).to(torch.float8_e4m3fn)
            held[i].append(c.double() * s.double()[..., None])
            for key in range(n):
                codes[i][table[b, key // page], :, key % page] = c.view(torch.uint8)[:, key]
                scales[i][table[b, key // page], :, key % page] = s[:, key]
    return codes, scales, table, held


def _run(dev, q, codes, scales, table, lk, lq):
    pools = [x.to(dev).view(torch.float8_e4m3fn) for x in codes]
    cu = torch.tensor([sum(lq[:b]) for b in range(len(lq) + 1)], dtype=torch.int32, device=dev)
    out, lse = paged_attention(q.to(dev), *pools, table.to(dev), torch.tensor(lk, dtype=torch.int32, device=dev), cu,
                               k_scale=scales[0].to(dev), v_scale=scales[1].to(dev), return_lse=True)
    return out.cpu(), lse.cpu()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("lq,lk,Hq,Hkv", [
    ([40], [40], 1, 1),                              # rows of few keys: each rounding shows
    ([130, 1, 17, 0, 300], [130, 40, 30, 9, 300], 4, 2),
    ([150, 1], [2500, 300], 8, 1),                   # tiles that end in another stretch
    ([1, 1], [1, 700], 4, 2),
])
def test_fp16_over_fp8(dev, D, page, far, lq, lk, Hq, Hkv):
    q = torch.randn(sum(lq), Hq, D, generator=torch.Generator().manual_seed(60)).half()
    codes, scales, table, (k, v) = _cache(61, lk, Hkv, D, page, far)
    out, lse = _run(dev, q, codes, scales, table, lk, lq)
    a = 0
    for b, n in enumerate(lq):
        for h in range(Hq):
            o, ls, tol, tol_l = attention(q[a:a + n, h], k[b][h // (Hq // Hkv)], v[b][h // (Hq // Hkv)], True, None, HALF_STEP[torch.float16])
            close(out[a:a + n, h], o, tol + 2.0 ** -25, f"out b{b} h{h}")  # (half a step of fp16's smallest values)
            close(lse[h, a:a + n], ls, tol_l, f"lse b{b} h{h}")
        a += n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lq,lk", [([100], [100]), ([1], [100]), ([40], [1500])])
def test_an_infinite_scale(dev, dtype, lq, lk):
    D, page, G, at = 128, 16, 2, lk[0] - 20
    q = torch.randn(sum(lq), G, D, generator=torch.Generator().manual_seed(62)).to(dtype)
    codes, scales, table, (k, v) = _cache(63, lk, 1, D, page, False)
    scales[1][table[0, at // page], 0, at % page] = math.inf
    codes[1][table[0, at // page], 0, at % page, 5] = 0  # (0 times infinity)
    want = v[0][0, at].sign() * math.inf
    want[v[0][0, at] == 0], want[5] = math.nan, math.nan
    out, lse = _run(dev, q, codes, scales, table, lk, lq)
    sees = max(0, at - (lk[0] - lq[0]))  # the first query that sees it
    for h in range(G):
        o, ls, tol, tol_l = attention(q[:, h], k[0][0], v[0][0], True, None, HALF_STEP[dtype])
        close(out[:sees, h], o[:sees], tol[:sees] + 2.0 ** -25)
        close(lse[h], ls, tol_l)
        assert torch.equal(out[sees:, h].double().nan_to_num(7.0), want.expand(lq[0] - sees, D).nan_to_num(7.0))
