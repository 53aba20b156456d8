"""An infinity of V that a query sees, wherever its key lies: the output is infinite there, as
the definition has it, and every other value is within the bounds of ``dense_reference``."""

from __future__ import annotations

import math

import pytest
import torch

from dense_reference import HALF_STEP, attention, close
from linattn_amd.kernels.dense import dense_attention, packed_attention
from linattn_amd.kernels.eviction import evict_decode_step
from test_gpu_eviction import _Plain

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _rand(seed, *shape, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype)


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Tk,G,Tq", [(1, 1, 1), (64, 4, 1), (77, 16, 1), (96, 3, 4), (2560, 4, 1), (1501, 2, 8)])
def test_few_rows(dev, dtype, D, Tk, G, Tq):
    """At most 16 rows: one key (its weight is 1), whole rounds of keys and not, split and not."""
    q, k, v = (_rand(i, 1, h, t, D, dtype=dtype) for i, h, t in ((0, G, Tq), (1, 1, Tk), (2, 1, Tk)))
    for at in {0, Tk // 2, Tk - 1}:
        x = v.clone()
        x[0, 0, at, 5], x[0, 0, at, 40] = math.inf, -math.inf
        x[0, 0, Tk // 3, 41] = math.nan
        out, lse = (y.cpu() for y in dense_attention(q.to(dev), k.to(dev), x.to(dev), return_lse=True))
        for h in range(G):
            o, ls, tol, tol_l = attention(q[0, h], k[0, 0], x[0, 0], True, None, HALF_STEP[dtype])
            assert torch.equal(out[0, h].isnan(), o.isnan()), (at, h)
            close(out[0, h].nan_to_num(0, math.inf, -math.inf), o.nan_to_num(0, math.inf, -math.inf),
                  tol.nan_to_num(0, math.inf), f"inf at {at}, head {h}")
            close(lse[0, h], ls, tol_l)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Hkv,G,C,lens", [
    (1, 1, 1, 1, [0]), (2, 2, 4, 64, [64, 20]), (1, 1, 16, 65, [65]), (1, 2, 3, 1030, [1030]), (2, 1, 5, 2048, [2048, 700])])
def test_decode_step(dev, dtype, D, B, Hkv, G, C, lens):
    """In an entry of the cache (an inner one, the last) and in the new token's row."""
    recent, sink = (C - 1) // 2, min(4, (C - 1) // 2)
    for where in ("inner", "last", "new"):
        k, v = _rand(0, B, Hkv, C, D, dtype=dtype), _rand(1, B, Hkv, C, D, dtype=dtype)
        w, g = _rand(2, B, Hkv, C).exp(), torch.Generator().manual_seed(3)
        w[:, :, 0] += 100.0  # (not given up)
        positions = torch.rand(B, Hkv, C, generator=g).argsort(-1).to(torch.int32)
        q, kn, vn = (_rand(i, B, h, 1, D, dtype=dtype) for i, h in ((4, Hkv * G), (5, Hkv), (6, Hkv)))
        pos = [C + 7 * b for b in range(B)]
        for b in range(B):
            k[b, :, lens[b]:], v[b, :, lens[b]:], w[b, :, lens[b]:], positions[b, :, lens[b]:] = math.nan, math.nan, math.nan, -1
            if where == "new":
                vn[b, :, 0, 7] = math.inf
            elif lens[b] > 0:
                at = 0 if where == "inner" else lens[b] - 1
                w[b, :, at] = 100.0
                v[b, :, at, 7], v[b, :, at, 8] = math.inf, -math.inf
        plain = _Plain(k, v, w, positions, lens)
        kd, vd, wd, pd = k.to(dev), v.to(dev), w.to(dev), positions.to(dev)
        out = evict_decode_step(q.to(dev), kn.to(dev), vn.to(dev), kd, vd, wd, pd, _i32(lens, dev), _i32(pos, dev),
                                recent=recent, sink=sink)
        ref, tol = plain.step(q, kn, vn, pos, recent, sink, None, w)
        close(out, ref, tol, where)
        for b in range(B):
            m = plain.n[b]
            assert torch.equal(vd[b, :, :m].cpu(), plain.v[b, :, :m])
            close(wd[b, :, :m], plain.w[b, :, :m], plain.tol[b, :, :m], where)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("G,T", [(1, 300), (4, 150)])
def test_prompt_with_weights_of_every_size(dev, dtype, G, T):
    """Whole prompts, the infinities at keys whose weights lie up to 70 powers of two below the
    row's largest."""
    D = 64
    q, k, v = (_rand(i, 1, h, T, D, dtype=dtype) for i, h in ((0, G), (1, 1), (2, 1)))
    q[..., 0], k[..., 0] = 1.0, torch.linspace(0.0, -48.0, T).to(dtype)
    v[0, 0, 3, 1], v[0, 0, T // 2, 2], v[0, 0, T - 9, 3], v[0, 0, T - 9, 4] = math.inf, -math.inf, math.inf, math.nan
    v[0, 0, 20, 3], v[0, 0, 21, 5], v[0, 0, T - 30, 5] = math.inf, math.inf, -math.inf
    out, lse = (y.cpu() for y in dense_attention(q.to(dev), k.to(dev), v.to(dev), scale=1.0, return_lse=True))
    for h in range(G):
        o, ls, tol, tol_l = attention(q[0, h], k[0, 0], v[0, 0], True, 1.0, HALF_STEP[dtype])
        assert torch.equal(out[0, h].isnan(), o.isnan())
        close(out[0, h].nan_to_num(0, math.inf, -math.inf), o.nan_to_num(0, math.inf, -math.inf), tol.nan_to_num(0, math.inf))
        close(lse[0, h], ls, tol_l)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,Tq,Tk,packed", [(64, 40, 3000, False), (128, 17, 2100, False), (64, 200, 260, True), (64, 3, 2500, False)])
def test_chunks_with_weights_of_every_size(dev, dtype, D, Tq, Tk, packed):
    """Keys split over workgroups, sequences packed at an offset, few rows: infinities and NaN
    before and behind the rows' last keys, at weights up to 70 powers of two below the largest."""
    q, k, v = (_rand(i, 1, 1, t, D, dtype=dtype) for i, t in ((0, Tq), (1, Tk), (2, Tk)))
    q[..., 0], k[..., 0] = 1.0, torch.linspace(-48.0, 0.0, Tk).to(dtype)
    v[0, 0, 3, 1], v[0, 0, Tk // 2, 2], v[0, 0, 5, 3], v[0, 0, Tk // 3, 3] = math.inf, -math.inf, math.inf, -math.inf
    v[0, 0, Tk - 2, 4], v[0, 0, Tk - 1, 5], v[0, 0, Tk // 2, 6] = math.nan, math.inf, math.nan
    if packed:
        lead = 5
        qd, kd, vd = (torch.cat([torch.full_like(x[0, 0, :lead], math.nan), x[0, 0]])[:, None].to(dev) for x in (q, k, v))
        cu = [_i32([lead, lead + n], dev) for n in (Tq, Tk)]
        out, lse = packed_attention(qd, kd, vd, *cu, scale=1.0, return_lse=True)
        out, lse = out[lead:, 0].cpu(), lse[0, lead:].cpu()
    else:
        out, lse = dense_attention(q.to(dev), k.to(dev), v.to(dev), scale=1.0, return_lse=True)
        out, lse = out[0, 0].cpu(), lse[0, 0].cpu()
    o, ls, tol, tol_l = attention(q[0, 0], k[0, 0], v[0, 0], True, 1.0, HALF_STEP[dtype])
    assert torch.equal(out.isnan(), o.isnan())
    close(out.nan_to_num(0, math.inf, -math.inf), o.nan_to_num(0, math.inf, -math.inf), tol.nan_to_num(0, math.inf))
    close(lse, ls, tol_l)
