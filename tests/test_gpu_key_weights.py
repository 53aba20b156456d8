"""``key_weights`` and ``packed_key_weights`` against a 64-bit reference on the CPU, with the row
sums that the attention kernels returned.  Bounds: see ``dense_reference.key_weights``."""

from __future__ import annotations

import math

import pytest
import torch

from dense_reference import attention, close, key_weights as reference
from linattn_amd.kernels.dense import dense_attention, packed_attention
from linattn_amd.kernels.eviction import key_weights, packed_key_weights

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _rand(seed, *shape, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype)


def _lse(q, k, lq, lk, causal=True, scale=None):
    """Row sums in 64 bits, rounded to fp32, -inf on padding."""
    B, Hq, Tq, D = q.shape
    G = Hq // k.shape[1]
    out = torch.full((B, Hq, Tq), -math.inf)
    for b in range(B):
        for h in range(Hq):
            kk = k[b, h // G, :lk[b]]
            out[b, h, :lq[b]] = attention(q[b, h, :lq[b]], kk, kk, causal, scale)[1].float()
    return out


def _check(w, q, k, lse, lq, lk, causal=True, scale=None, last=None, base=None):
    B, Hkv, Tk, D = k.shape
    G = q.shape[1] // Hkv
    for b in range(B):
        for h in range(Hkv):
            g = slice(h * G, (h + 1) * G)
            ref, tol = reference(q[b, g, :lq[b]], k[b, h, :lk[b]], lse[b, g, :lq[b]], causal, scale, last)
            if base is not None:
                ref = ref + base[b, h, :lk[b]].double()
                tol = tol + ref.abs() * 2.0 ** -24
            close(w[b, h, :lk[b]], ref, tol, f"b{b} h{h}")
            rest = w[b, h, lk[b]:].cpu()
            assert torch.equal(rest, torch.zeros_like(rest) if base is None else base[b, h, lk[b]:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Hkv,G,Tq,Tk,last", [
    (1, 1, 1, 1, 1, None),
    (2, 2, 4, 65, 65, None),
    (1, 2, 3, 130, 130, 50),
    (1, 1, 8, 33, 300, None),    # a chunk behind a cache
    (1, 1, 5, 70, 31, None),     # the first queries see nothing
    (2, 1, 2, 257, 257, 1),
    (1, 1, 2, 300, 515, 1000),
    (1, 1, 4, 700, 700, None),   # rows split over workgroups
])
def test_batched(dev, dtype, D, B, Hkv, G, Tq, Tk, last):
    q, k = (_rand(i, B, h, t, D, dtype=dtype) for i, h, t in ((0, Hkv * G, Tq), (1, Hkv, Tk)))
    lse = _lse(q, k, [Tq] * B, [Tk] * B)
    w = key_weights(q.to(dev), k.to(dev), lse.to(dev), last=last)
    assert w.shape == (B, Hkv, Tk) and w.dtype == torch.float32
    _check(w, q, k, lse, [Tq] * B, [Tk] * B, last=last)
    if Tq < 100:
        lse = _lse(q, k, [Tq] * B, [Tk] * B, False, 0.2)
        base = _rand(9, B, Hkv, Tk).abs()
        out = base.to(dev)
        r = key_weights(q.to(dev), k.to(dev), lse.to(dev), last=last, causal=False, scale=0.2, out=out)
        assert r is out
        _check(out, q, k, lse, [Tq] * B, [Tk] * B, False, 0.2, last, base)


@pytest.mark.parametrize("dtype", TYPES)
def test_ragged_padding_and_empty_rows(dev, dtype):
    B, Hkv, G, T, D = 5, 2, 2, 300, 64
    q, k = (_rand(i, B, h, T, D, dtype=dtype) for i, h in ((0, Hkv * G), (1, Hkv)))
    lk, lq = [300, 64, 1, 0, 97], [300, 64, 1, 20, 120]
    lse = _lse(q, k, lq, lk)
    for b in range(B):
        q[b, :, lq[b]:], k[b, :, lk[b]:], lse[b, :, lq[b]:] = math.nan, math.nan, math.nan
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    for last in (None, 30):
        w = key_weights(q.to(dev), k.to(dev), lse.to(dev), lengths=i32(lk), q_lengths=i32(lq), last=last)
        _check(w, q, k, lse, lq, lk, last=last)
        assert torch.equal(w, key_weights(q.to(dev), k.to(dev), lse.to(dev), lengths=i32(lk), q_lengths=i32(lq),
                                          last=last))


@pytest.mark.parametrize("dtype", TYPES)
def test_what_a_key_is_not_seen_by(dev, dtype):
    """A query that is not finite reaches the keys it sees; a key that is not finite, itself."""
    T, D = 150, 64
    q, k = _rand(0, 1, 2, T, D, dtype=dtype), _rand(1, 1, 1, T, D, dtype=dtype)
    lse = _lse(q, k, [T], [T])
    q[0, 0, 40, 3] = math.nan
    k[0, 0, 100, 5] = math.inf
    w = key_weights(q.to(dev), k.to(dev), lse.to(dev))[0, 0].cpu()
    assert torch.isnan(w[:41]).all() and torch.isfinite(w[41:100]).all() and torch.isfinite(w[101:]).all()
    q[0, 0, 40, 3] = 0.5
    ref, tol = reference(q[0], k[0, 0].nan_to_num(0, 0, 0), lse[0])
    for part in (slice(41, 100), slice(101, T)):
        close(w[part], ref[part], tol[part])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,Hkv,G,last", [
    ([1], 1, 1, None),
    ([37, 0, 300, 1, 200, 65], 2, 4, None),
    ([37, 0, 300, 1, 200, 65], 2, 3, 20),
    ([3] * 70 + [150] + [1] * 69, 1, 2, None),
])
def test_packed(dev, dtype, D, lens, Hkv, G, last):
    n, lead, rest = sum(lens), 4, 9
    total = lead + n + rest
    q, k, v = (_rand(i, total, h, D, dtype=dtype) for i, h in ((0, Hkv * G), (1, Hkv), (2, Hkv)))
    cu = torch.tensor([lead] + [lead + sum(lens[:i + 1]) for i in range(len(lens))], dtype=torch.int32)
    qd, kd, cud = q.to(dev), k.to(dev), cu.to(dev)
    _, lse = packed_attention(qd, kd, v.to(dev), cud, return_lse=True)
    w = packed_key_weights(qd, kd, lse, cud, last=last)
    assert w.shape == (Hkv, total)
    lse = lse.cpu()
    for b, m in enumerate(lens):
        a = int(cu[b])
        if len(lens) > 10 and b > 3 and m < 100:
            continue
        for h in range(Hkv):
            ref, tol = reference(q[a:a + m, h * G:(h + 1) * G].transpose(0, 1), k[a:a + m, h],
                                 lse[h * G:(h + 1) * G, a:a + m], last=last)
            close(w[h, a:a + m], ref, tol, f"sequence {b}")
    assert (w[:, :lead] == 0).all() and (w[:, lead + n:] == 0).all()
    out = torch.full_like(w, 2.0)
    packed_key_weights(qd, kd, lse.to(dev), cud, last=last, out=out)
    assert torch.equal(out[:, lead:lead + n], w[:, lead:lead + n] + 2.0)
    assert (out[:, :lead] == 2).all() and (out[:, lead + n:] == 2).all()


def test_weights_of_chunks_add_up(dev):
    """Chunk after chunk into one buffer: the whole prompt's weights; layouts and graphs too."""
    Hkv, G, T, D = 2, 4, 500, 128
    q, k, v = (_rand(i, 1, T, h, D, dtype=torch.bfloat16).to(dev).transpose(1, 2) for i, h in ((0, Hkv * G), (1, Hkv), (2, Hkv)))
    _, lse = dense_attention(q, k, v, return_lse=True)
    whole = key_weights(q, k, lse)
    qc, kc, lc = q.contiguous(), k.contiguous(), lse.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(whole, key_weights(qc, kc, lc))
    parts = torch.zeros(1, Hkv, T, device=dev)
    for a in range(0, T, 128):
        e = min(T, a + 128)
        key_weights(q[:, :, a:e], k[:, :, :e], lse[:, :, a:e], out=parts[:, :, :e])
    # each sum of up to 2000 weights off by at most that many roundings
    assert ((parts - whole).abs() <= 2 * 2000 * 2.0 ** -24 * whole).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w = key_weights(q, k, lse)
    for _ in range(3):
        w.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(w, key_weights(q, k, lse))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w2 = key_weights(q, k, lse)
    side.synchronize()
    assert torch.equal(w2, whole)
    # every query's weights sum to one
    assert abs(float(whole.sum()) - Hkv * G * T) < 1e-3 * Hkv * G


@pytest.mark.parametrize("G,Tq,last,far", [(4, 40, None, 6_000_000), (4, 129, None, 18_000_000), (2, 300, 17, 18_000_000),
                                           (5, 20, 3, 18_000_000)])
def test_heads_far_apart(dev, G, Tq, last, far):
    """Head strides that with three and with one of them pass 32 bits: a staged tile holds
    fewer heads."""
    D, far = 64, 64 * far
    q, k = _rand(0, 1, G, Tq, D, dtype=torch.bfloat16), _rand(1, 1, 1, Tq, D, dtype=torch.bfloat16)
    lse = _lse(q, k, [Tq], [Tq])
    big = torch.empty(far * (G - 1) + Tq * D, dtype=torch.bfloat16, device=dev)
    wide = big.as_strided((1, G, Tq, D), (0, far, D, 1))
    wide.copy_(q.to(dev))
    w = key_weights(wide, k.to(dev), lse.to(dev), last=last)
    _check(w, q, k, lse, [Tq], [Tq], last=last)
    near = key_weights(q.to(dev), k.to(dev), lse.to(dev), last=last)
    _check(near, q, k, lse, [Tq], [Tq], last=last)
    del big, wide
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lse", [0.3, 0.7, 1.3])
def test_many_equal_weights(dev, dtype, lse):
    """Keys that gather equal weights from up to 131072 rows: a running sum that took all of a
    lane's rows one by one would drift by up to half a step of the sum for each."""
    Hkv, G, T, D = 8, 4, 32768, 64
    q = torch.zeros(T, Hkv * G, D, dtype=dtype, device=dev)
    k = torch.zeros(T, Hkv, D, dtype=dtype, device=dev)
    row = torch.full((Hkv * G, T), lse, dtype=torch.float32, device=dev)
    w = packed_key_weights(q, k, row, torch.tensor([0, T], dtype=torch.int32, device=dev)).double().cpu()
    want = G * torch.arange(T, 0, -1).double() * math.exp(-float(torch.tensor(lse, dtype=torch.float32)))
    # runs of 32 staged tiles, 64 additions a lane (2 of each tile), 5 between lanes, and the
    # runs' sums: 64 of 64 rows' tiles, 128 of 32 rows'; a few steps of exp2 and its argument
    tol = (64 + 5 + (64 if dtype != torch.float32 else 128) + 8 + 2 * lse) * 2.0 ** -24
    assert ((w - want).abs() <= tol * want).all()
