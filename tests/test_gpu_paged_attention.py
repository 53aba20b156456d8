"""``paged_attention`` against a 64-bit reference on the CPU: every type and head size, pages of any
size, chunks beside single tokens, empty sequences, more queries than keys, stretches that end
inside tiles, fp8 caches, slots and keys that are not finite, strides, streams and graphs.
Bounds: see ``dense_reference.attention``."""

from __future__ import annotations

import math

import pytest
import torch

from dense_reference import HALF_STEP, attention, close
from linattn_amd.kernels.block_sparse import fp8_scale_pairs
from linattn_amd.kernels.dense import dense_attention, packed_attention, paged_attention

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _rand(g, *shape):
    return torch.randn(*shape, generator=g)


def _i32(x, dev=None):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _paged(seed, k, v, page, spare=2, fill=math.nan):
    """Pools and a table that hold k, v (lists of (Hkv, Lk, D)); every other slot is `fill`, and what
    the table has behind a sequence's pages points nowhere."""
    g = torch.Generator().manual_seed(seed)
    Hkv, _, D = k[0].shape
    pages = [-(-x.shape[1] // page) for x in k]
    n_phys = sum(pages) + spare
    order = torch.randperm(n_phys, generator=g)
    table = torch.full((len(k), max(pages) + 2), -7, dtype=torch.int32)
    table[:, -1] = 10 ** 6
    pools = [torch.full((n_phys, Hkv, page, D), fill, dtype=k[0].dtype) for _ in "kv"]
    at = 0
    for b in range(len(k)):
        table[b, :pages[b]] = order[at:at + pages[b]]
        at += pages[b]
        for i in range(pages[b]):
            n = min(page, k[b].shape[1] - i * page)
            for pool, x in zip(pools, (k, v)):
                pool[table[b, i], :, :n] = x[b][:, i * page:i * page + n]
    return (*pools, table)


def _case(seed, lq, lk, Hq, Hkv, D, dtype):
    g = torch.Generator().manual_seed(seed)
    q = _rand(g, sum(lq), Hq, D).to(dtype)
    k, v = ([_rand(g, Hkv, n, D).to(dtype) for n in lk] for _ in "kv")
    return q, k, v


def _cu(lq, dev, front=0):
    return _i32([front + sum(lq[:b]) for b in range(len(lq) + 1)], dev)


def _check(out, lse, q, k, v, lq, lk, causal=True, scale=None, half=None, what=""):
    """Packed outputs on the CPU."""
    a, G = 0, q.shape[1] // k[0].shape[0]
    half = HALF_STEP[q.dtype] if half is None else half
    for b, (n, m) in enumerate(zip(lq, lk)):
        for h in range(q.shape[1]):
            o, ls, tol, tol_l = attention(q[a:a + n, h], k[b][h // G], v[b][h // G], causal, scale, half, HALF_STEP[out.dtype])
            close(out[a:a + n, h], o, tol, f"{what} out b{b} h{h}")
            close(lse[h, a:a + n], ls, tol_l, f"{what} lse b{b} h{h}")
        a += n


SHAPES = [
    # lq, lk, Hq, Hkv
    ([1], [1], 1, 1),
    ([1, 1, 1], [64, 65, 200], 8, 2),
    ([5, 0, 70, 1, 33], [5, 12, 200, 0, 31], 4, 2),   # no queries, no keys, more queries than keys
    ([130], [130], 6, 2),                              # a group that divides no tile
    ([1, 257, 2], [90, 300, 2], 5, 1),
    ([40], [1000], 16, 1),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 64, 24, 1, 128])
@pytest.mark.parametrize("lq,lk,Hq,Hkv", SHAPES)
def test_packed(dev, dtype, D, page, lq, lk, Hq, Hkv):
    q, k, v = _case(1, lq, lk, Hq, Hkv, D, dtype)
    kp, vp, table = _paged(2, k, v, page)
    args = (kp.to(dev), vp.to(dev), table.to(dev), _i32(lk, dev), _cu(lq, dev))
    out, lse = paged_attention(q.to(dev), *args, return_lse=True)
    assert out.dtype == dtype and lse.dtype == torch.float32
    _check(out.cpu(), lse.cpu(), q, k, v, lq, lk)
    out32, lse = paged_attention(q.to(dev), *args, causal=False, scale=0.3, out_dtype=torch.float32, return_lse=True)
    _check(out32.cpu(), lse.cpu(), q, k, v, lq, lk, False, 0.3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 20])
@pytest.mark.parametrize("D,lq,lk,Hq,Hkv", [
    (128, [1, 1], [9000, 300], 4, 1),               # few rows over many keys: many parts
    (64, [3, 200, 1, 1], [5000, 2500, 4001, 17], 4, 2),   # tiles that end in another stretch
    (128, [150], [3000], 8, 1),
])
def test_shared_tiles(dev, dtype, page, D, lq, lk, Hq, Hkv):
    q, k, v = _case(3, lq, lk, Hq, Hkv, D, dtype)
    kp, vp, table = _paged(4, k, v, page)
    args = (q.to(dev), kp.to(dev), vp.to(dev), table.to(dev), _i32(lk, dev), _cu(lq, dev))
    out, lse = paged_attention(*args, return_lse=True)
    _check(out.cpu(), lse.cpu(), q, k, v, lq, lk)
    again, lse2 = paged_attention(*args, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)  # the same bits


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_sequences(dev, dtype):
    """More than a wave has lanes, most with a token or none."""
    r = torch.Generator().manual_seed(5)
    lq = torch.randint(0, 3, (150,), generator=r).tolist()
    lk = [x + int(y) for x, y in zip(lq, torch.randint(0, 120, (150,), generator=r))]
    lq[70:75], lk[149] = [0] * 5, 700
    q, k, v = _case(6, lq, lk, 4, 2, 64, dtype)
    kp, vp, table = _paged(7, k, v, 16)
    out, lse = paged_attention(q.to(dev), kp.to(dev), vp.to(dev), table.to(dev), _i32(lk, dev), _cu(lq, dev), return_lse=True)
    _check(out.cpu(), lse.cpu(), q, k, v, lq, lk)


@pytest.mark.parametrize("dtype", TYPES)
def test_as_the_contiguous_forms(dev, dtype):
    """Large chunks, against ``packed_attention`` over the same keys: within both bounds."""
    lq, lk, Hq, Hkv, D = [700, 300, 1], [900, 300, 5000], 8, 2, 128
    q, k, v = _case(8, lq, lk, Hq, Hkv, D, dtype)
    kp, vp, table = _paged(9, k, v, 64)
    got, lse = paged_attention(q.to(dev), kp.to(dev), vp.to(dev), table.to(dev), _i32(lk, dev), _cu(lq, dev), return_lse=True)
    flat = lambda x: torch.cat([y.transpose(0, 1) for y in x]).to(dev)
    want, lse_w = packed_attention(q.to(dev), flat(k), flat(v), _cu(lq, dev), _cu(lk, dev), return_lse=True)
    u = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -16}[dtype]
    assert ((got.double() - want.double()).abs() <= 4 * u * (want.double().abs() + 3.0)).all()
    assert ((lse - lse_w).abs() <= 1e-4).all()


# ------------------------------------------------------------------- fp8 ----
def _fp8(x):
    """Codes, scales and values of (Hkv, L, D)."""
    s = x.abs().amax(-1).clamp(min=1e-8) / 448
    c = (x / s[..., None]).to(torch.float8_e4m3fn)
    return c, s, c.double() * s.double()[..., None]


def _paged_fp8(seed, k, v, page, dev, pairs):
    """As _paged, of codes and scales (slots that hold nothing: NaN in both)."""
    kc, vc = ([_fp8(x) for x in y] for y in (k, v))
    kp, vp, table = _paged(seed, [c[0].view(torch.uint8).clone() for c in kc], [c[0].view(torch.uint8).clone() for c in vc], page, fill=0x7F)
    one = lambda x: [c[1][..., None].contiguous() for c in x]
    ks, vs, _ = _paged(seed, one(kc), one(vc), page)
    if pairs:
        gks, gvs = fp8_scale_pairs(*ks.shape[:3], dev)
        gks.copy_(ks[..., 0])
        gvs.copy_(vs[..., 0])
    else:
        gks, gvs = ks[..., 0].contiguous().to(dev), vs[..., 0].contiguous().to(dev)
    f8 = torch.float8_e4m3fn
    return kp.to(dev).view(f8), vp.to(dev).view(f8), table.to(dev), gks, gvs, [c[2] for c in kc], [c[2] for c in vc]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page,pairs", [(16, True), (64, False), (24, True), (1, False)])
@pytest.mark.parametrize("lq,lk,Hq,Hkv", SHAPES + [([2, 150], [6000, 700], 4, 1)])
def test_fp8(dev, dtype, D, page, pairs, lq, lk, Hq, Hkv):
    q, k, v = _case(10, lq, lk, Hq, Hkv, D, torch.float32)
    q = q.to(dtype)
    for x in v:
        x *= 10.0  # scales of their own
    kp, vp, table, ks, vs, kv_, vv = _paged_fp8(11, k, v, page, dev, pairs)
    out, lse = paged_attention(q.to(dev), kp, vp, table, _i32(lk, dev), _cu(lq, dev), k_scale=ks, v_scale=vs, return_lse=True)
    # weights are rounded to bf16 for their product with codes
    _check(out.cpu(), lse.cpu(), q, kv_, vv, lq, lk, half=HALF_STEP[torch.bfloat16])


# --------------------------------------------------------- batched, strides ----
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_batched(dev, dtype, causal):
    B, Hq, Hkv, Tq, D, page = 4, 4, 2, 40, 64, 16
    lq, lk = [40, 0, 7, 33], [100, 50, 7, 20]
    g = torch.Generator().manual_seed(12)
    q = _rand(g, B, Tq, Hq, D).to(dtype)
    for b in range(B):
        q[b, lq[b]:] = math.nan
    k, v = ([_rand(g, Hkv, n, D).to(dtype) for n in lk] for _ in "kv")
    kp, vp, table = _paged(13, k, v, page)
    there = q.to(dev).transpose(1, 2)  # (heads of a token side by side)
    more = dict(causal=causal, q_lengths=_i32(lq, dev), return_lse=True)
    out, lse = paged_attention(there, kp.to(dev), vp.to(dev), table.to(dev), _i32(lk, dev), **more)
    assert out.shape == there.shape and lse.shape == (B, Hq, Tq)
    for b in range(B):
        _check(out[b, :, :lq[b]].transpose(0, 1).cpu(), lse[b, :, :lq[b]].cpu(), q[b, :lq[b]], [k[b]], [v[b]], [lq[b]], [lk[b]], causal)
        assert (out[b, :, lq[b]:] == 0).all() and (lse[b, :, lq[b]:] == -math.inf).all()
    # lengths past the table are the table's, negative ones none; an out of other strides
    big = torch.full((B, Tq, Hq, 2 * D), 3.0, dtype=dtype, device=dev)
    o2 = big[..., :D].transpose(1, 2)
    full = torch.arange(B * 3, dtype=torch.int32, device=dev).view(B, 3)
    pool = _rand(g, B * 3, Hkv, page, D).to(dtype).to(dev)
    qf = there.nan_to_num()
    got = paged_attention(qf, pool, pool, full, _i32([48, 999, -5, 0], dev), causal=causal, out=o2)
    assert got is o2 and (big[..., D:] == 3).all() and (o2[2:] == 0).all()
    flat = pool.view(B, 3, Hkv, page, D).transpose(1, 2).reshape(B, Hkv, 48, D)
    _check(o2[0].transpose(0, 1).cpu(), paged_attention(qf[:1], pool, pool, full[:1], _i32([48], dev), causal=causal, return_lse=True)[1][0].cpu(),
           qf[0].transpose(0, 1).cpu(), [flat[0].cpu()], [flat[0].cpu()], [Tq], [48], causal)
    same = paged_attention(qf[1:2], pool, pool, full[1:2], _i32([48], dev), causal=causal)
    assert ((o2[1] - same[0]).abs() <= 1e-5).all()


def test_rows_that_no_sequence_holds(dev):
    lq, lk, front, rest = [3, 1], [20, 50], 2, 3
    q, k, v = _case(14, lq, lk, 4, 2, 64, torch.bfloat16)
    kp, vp, table = (x.to(dev) for x in _paged(15, k, v, 16))
    pad = lambda n: torch.full((n, 4, 64), math.nan).bfloat16()
    qp = torch.cat([pad(front), q, pad(rest)]).to(dev)
    out, lse = paged_attention(qp, kp, vp, table, _i32(lk, dev), _cu(lq, dev, front), return_lse=True)
    _check(out[front:-rest].cpu(), lse[:, front:-rest].cpu().contiguous(), q, k, v, lq, lk)
    for x in (out[:front], out[-rest:]):
        assert (x == 0).all()
    assert (lse[:, :front] == -math.inf).all() and (lse[:, -rest:] == -math.inf).all()
    mine = torch.full_like(qp, 5.0)
    got, lse2 = paged_attention(qp, kp, vp, table, _i32(lk, dev), _cu(lq, dev, front), out=mine, return_lse=True)
    assert got is mine and (mine[:front] == 5).all() and (mine[-rest:] == 5).all()
    assert torch.equal(mine[front:-rest], out[front:-rest]) and torch.equal(lse, lse2)
    none = paged_attention(qp[:0], kp, vp, table, _i32(lk, dev), _i32([0, 0, 0], dev), return_lse=True)
    assert none[0].shape == (0, 4, 64) and none[1].shape == (4, 0)


# ------------------------------------------------------------- not finite ----
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,G,page,before", [(64, 1, 16, 0), (128, 4, 24, 0), (128, 2, 64, 3000)])
def test_keys_that_are_not_finite(dev, dtype, D, G, page, before):
    """An infinity or a NaN of a key or value reaches the queries that see it and no other."""
    T = 140
    lq, lk = [T], [before + T]
    q, k, v = _case(16, lq, lk, G, 1, D, dtype)
    vb, kb = [v[0].clone()], [k[0].clone()]
    x = before
    vb[0][0, x + 100, 3], vb[0][0, x + 120, 60], vb[0][0, x + 139] = math.inf, -math.inf, math.nan
    kb[0][0, x + 130, 5] = math.nan
    kp, vp, table = (y.to(dev) for y in _paged(17, kb, vb, page))
    out, lse = (y.cpu() for y in paged_attention(q.to(dev), kp, vp, table, _i32(lk, dev), _cu(lq, dev), return_lse=True))
    for h in range(G):
        o, ls, tol, tol_l = attention(q[:, h], k[0][0], v[0][0], True, None, HALF_STEP[dtype])
        close(out[:100, h], o[:100], tol[:100])
        close(lse[h, :130], ls[:130], tol_l[:130])
        d3 = torch.arange(D) != 3
        close(out[100:120, h][:, d3], o[100:120][:, d3], tol[100:120][:, d3])
        assert torch.isinf(out[100:130, h, 3]).all()
        assert torch.isinf(out[120:130, h, 60]).all() and (out[120:130, h, 60] < 0).all()
        assert torch.isnan(out[130:, h]).all() and torch.isnan(lse[h, 130:]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_fp8_keys_that_are_not_finite(dev, dtype):
    """A code that is no number, and a scale that is not finite, at keys that early rows do not see."""
    T, D, page = 100, 128, 16
    q, k, v = _case(18, [T], [T], 2, 1, D, torch.float32)
    q = q.to(dtype)
    kp, vp, table, ks, vs, kv_, vv = _paged_fp8(19, k, v, page, dev, True)
    at = lambda key: (int(table[0, key // page]), 0, key % page)
    vp.view(torch.uint8)[at(60)][7] = 0x7F
    vs[at(80)] = math.inf
    ks[at(90)] = math.nan
    out, lse = (y.cpu() for y in paged_attention(q.to(dev), kp, vp, table, _i32([T], dev), _i32([0, T], dev), k_scale=ks, v_scale=vs, return_lse=True))
    for h in range(2):
        o, ls, tol, tol_l = attention(q[:, h], kv_[0][0], vv[0][0], True, None, HALF_STEP[torch.bfloat16], HALF_STEP[dtype])
        close(out[:60, h], o[:60], tol[:60])
        close(lse[h, :90], ls[:90], tol_l[:90])
        d7 = torch.arange(D) != 7
        close(out[60:80, h][:, d7], o[60:80][:, d7], tol[60:80][:, d7])
        assert torch.isnan(out[60:, h, 7]).all() and not torch.isfinite(out[80:, h]).any() and torch.isnan(out[90:, h]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_large_scores(dev, dtype):
    """Scores of thousands, keys alike, the lowest values of the type: the maximum is taken off first."""
    lq, lk = [50], [300]
    q, k, v = _case(20, lq, lk, 2, 1, 64, dtype)
    k[0][0, 10:20] = (k[0][0, 10:20].float() * 60).to(dtype)
    k[0][0, 40:] = k[0][0, 40]
    kp, vp, table = (y.to(dev) for y in _paged(21, k, v, 16))
    out, lse = paged_attention(q.to(dev), kp, vp, table, _i32(lk, dev), _cu(lq, dev), scale=2.0, return_lse=True)
    _check(out.cpu(), lse.cpu(), q, k, v, lq, lk, True, 2.0)


# ---------------------------------------------------------- streams, graphs ----
def test_streams_and_graphs(dev):
    """Two calls at once; captured calls that share nothing but inputs, replayed with other lengths."""
    lq, lk, Hq, Hkv, D = [1, 30, 1], [4000, 500, 90], 8, 2, 128
    q, k, v = _case(22, lq, lk, Hq, Hkv, D, torch.bfloat16)
    kp, vp, table = (x.to(dev) for x in _paged(23, k, v, 64, fill=0.0))
    q, cu, n = q.to(dev), _cu(lq, dev), _i32(lk, dev)
    want = paged_attention(q, kp, vp, table, n, cu)
    one = paged_attention(q[:1], kp, vp, table[:1], n[:1], cu[:2])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(dev))
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(paged_attention(q, kp, vp, table, n, cu) if i % 3 else paged_attention(q[:1], kp, vp, table[:1], n[:1], cu[:2]))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, want if i % 3 else one)
    outs = [torch.zeros_like(q) for _ in range(2)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for g, o, c in zip(graphs, outs, (True, False)):
        with torch.cuda.graph(g):
            paged_attention(q, kp, vp, table, n, cu, causal=c, out=o)
    for lens in (lk, [2000, 500, 90], [70, 31, 2], [4000, 100, 1]):
        n.copy_(_i32(lens))
        eager = [paged_attention(q, kp, vp, table, n, cu, causal=c) for c in (True, False)]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for e, o in zip(eager, outs):
            assert torch.equal(e, o), lens


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,G", [(64, 2), (128, 4)])
def test_one_token_of_many_parts(dev, dtype, D, G):
    """A row of more parts than are joined one behind the other, finite and not."""
    lq, lk = [1, 1, 1], [13000, 700, 9001]
    q, k, v = _case(24, lq, lk, G, 1, D, dtype)
    vb = [x.clone() for x in v]
    vb[2][0, 8000, 7], vb[2][0, 3, 9] = math.inf, math.nan
    for values, clean in ((v, [0, 1, 2]), (vb, [0, 1])):
        kp, vp, table = (x.to(dev) for x in _paged(25, k, values, 16))
        out, lse = (x.cpu() for x in paged_attention(q.to(dev), kp, vp, table, _i32(lk, dev), _cu(lq, dev), return_lse=True))
        for b in range(3):
            for h in range(G):
                o, ls, tol, tol_l = attention(q[b:b + 1, h], k[b][0], v[b][0], True, None, HALF_STEP[dtype])
                close(lse[h, b:b + 1], ls, tol_l)
                keep = torch.ones(D, dtype=torch.bool)
                if b not in clean:
                    keep[[7, 9]] = False
                    assert out[b, h, 7] == math.inf and torch.isnan(out[b, h, 9])
                close(out[b:b + 1, h][:, keep], o[:, keep], tol[:, keep])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B", [700, 9000])
def test_batches_of_mostly_empty_sequences(dev, dtype, B):
    """Slots of a server of which few are in use: what lies between two of them is passed over."""
    used = {0: (1, 300), 1: (40, 40), 130: (1, 17), 131: (0, 50), 400: (70, 900), 401: (1, 1), 640: (2, 64), 690: (1, 70),
            B - 1: (33, 2000)}
    lq, lk = ([used.get(b, (0, 0))[i] for b in range(B)] for i in (0, 1))
    q, k, v = _case(26, lq, lk, 4, 2, 64, dtype)
    kp, vp, table = _paged(27, k, v, 16)
    args = (q.to(dev), kp.to(dev), vp.to(dev), table.to(dev), _i32(lk, dev), _cu(lq, dev))
    out, lse = paged_attention(*args, return_lse=True)
    _check(out.cpu(), lse.cpu(), q, k, v, lq, lk)
