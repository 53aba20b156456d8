"""``dense_attention`` and ``packed_attention`` against a 64-bit reference on the CPU: every type
and head size, lengths from none to long, groups that do not divide a tile, strides, padding
and later keys that are not finite, keys shared by several workgroups, streams and graphs.
Bounds: see ``dense_reference.attention``."""

from __future__ import annotations

import math

import pytest
import torch

from dense_reference import HALF_STEP, attention, close
from linattn_amd.kernels.dense import dense_attention, packed_attention

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _rand(seed, *shape, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype)


def _check(out, lse, q, k, v, lq, lk, causal=True, scale=None, what=""):
    """Batched outputs on the CPU against the reference, padding zeros and -inf."""
    B, Hq, Tq, D = q.shape
    G = Hq // k.shape[1]
    u = HALF_STEP[q.dtype]
    for b in range(B):
        for h in range(Hq):
            o, ls, tol, tol_l = attention(q[b, h, :lq[b]], k[b, h // G, :lk[b]], v[b, h // G, :lk[b]],
                                          causal, scale, u, HALF_STEP[out.dtype])
            close(out[b, h, :lq[b]], o, tol, f"{what} out b{b} h{h}")
            close(lse[b, h, :lq[b]], ls, tol_l, f"{what} lse b{b} h{h}")
            assert (out[b, h, lq[b]:] == 0).all() and (lse[b, h, lq[b]:] == -math.inf).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Hkv,G,Tq,Tk", [
    (1, 1, 1, 1, 1),
    (2, 2, 4, 65, 65),
    (1, 2, 3, 130, 130),     # a group that divides no tile
    (1, 1, 8, 33, 200),      # a chunk behind a cache
    (2, 1, 1, 257, 257),
    (1, 1, 5, 70, 31),       # more queries than keys: the first see none
    (1, 1, 2, 300, 333),
])
def test_batched(dev, dtype, D, B, Hkv, G, Tq, Tk):
    q, k, v = (_rand(i, B, h, t, D, dtype=dtype) for i, h, t in ((0, Hkv * G, Tq), (1, Hkv, Tk), (2, Hkv, Tk)))
    out, lse = dense_attention(q.to(dev), k.to(dev), v.to(dev), return_lse=True)
    assert out.dtype == dtype and lse.dtype == torch.float32
    _check(out.cpu(), lse.cpu(), q, k, v, [Tq] * B, [Tk] * B)
    out32, lse = dense_attention(q.to(dev), k.to(dev), v.to(dev), causal=False, scale=0.3,
                                 out_dtype=torch.float32, return_lse=True)
    assert out32.dtype == torch.float32
    _check(out32.cpu(), lse.cpu(), q, k, v, [Tq] * B, [Tk] * B, causal=False, scale=0.3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_ragged_padding_is_never_read(dev, dtype, causal):
    B, Hkv, G, T, D = 5, 2, 2, 150, 64
    q, k, v = (_rand(i, B, h, T, D, dtype=dtype) for i, h in ((0, Hkv * G), (1, Hkv), (2, Hkv)))
    lk, lq = [150, 64, 1, 0, 97], [150, 64, 1, 20, 30]
    for b in range(B):
        q[b, :, lq[b]:] = math.nan
        k[b, :, lk[b]:] = math.nan
        v[b, :, lk[b]:] = math.inf
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    out, lse = dense_attention(q.to(dev), k.to(dev), v.to(dev), causal=causal, lengths=i32(lk),
                               q_lengths=i32(lq), return_lse=True)
    _check(out.cpu(), lse.cpu(), q, k, v, lq, lk, causal)
    # lengths past the tensors are the tensors', negative ones none
    out2 = dense_attention(q[:2].nan_to_num().to(dev), k[:2].nan_to_num().to(dev),
                           v[:2].nan_to_num(0, 0, 0).to(dev), causal=causal, lengths=i32([999, -3]),
                           q_lengths=i32([150, 999]))
    want = dense_attention(q[:2].nan_to_num().to(dev), k[:2].nan_to_num().to(dev),
                           v[:2].nan_to_num(0, 0, 0).to(dev), causal=causal, lengths=i32([150, 0]),
                           q_lengths=i32([150, 150]))
    assert torch.equal(out2, want) and (out2[1] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,G", [(64, 1), (128, 4)])
def test_later_keys_that_are_not_finite(dev, dtype, D, G):
    """An infinity or a NaN of k or v reaches the queries that see it and no other."""
    Hkv, T = 1, 140
    q, k, v = (_rand(i, 1, h, T, D, dtype=dtype) for i, h in ((3, Hkv * G), (4, Hkv), (5, Hkv)))
    vb, kb = v.clone(), k.clone()
    vb[0, 0, 100, 3], vb[0, 0, 120, 60], vb[0, 0, 139] = math.inf, -math.inf, math.nan
    kb[0, 0, 130, 5] = math.nan
    out, lse = (x.cpu() for x in dense_attention(q.to(dev), kb.to(dev), vb.to(dev), return_lse=True))
    clean, clean_lse = (x.cpu() for x in dense_attention(q.to(dev), k.to(dev), v.to(dev), return_lse=True))
    # rows before the first: as without it (done again key by key: to the bounds)
    for h in range(G):
        o, ls, tol, tol_l = attention(q[0, h], k[0, 0], v[0, 0], True, None, HALF_STEP[dtype])
        close(out[0, h, :100], o[:100], tol[:100])
        close(lse[0, h, :130], ls[:130], tol_l[:130])
        close(clean[0, h], o, tol)
        d3 = torch.arange(D) != 3
        close(out[0, h, 100:120][:, d3], o[100:120][:, d3], tol[100:120][:, d3])
        assert torch.isinf(out[0, h, 100:130, 3]).all()
        assert torch.isinf(out[0, h, 120:130, 60]).all() and (out[0, h, 120:130, 60] < 0).all()
        assert torch.isnan(out[0, h, 130:]).all() and torch.isnan(lse[0, h, 130:]).all()
    assert torch.isfinite(clean).all() and torch.isfinite(clean_lse).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Hkv,G,Tq,Tk", [(1, 1, 4, 1, 5003), (2, 2, 1, 3, 1700), (1, 1, 7, 20, 3001)])
def test_few_rows_over_many_keys(dev, dtype, D, B, Hkv, G, Tq, Tk):
    """Keys split over workgroups, some of whose parts no row sees; ragged and not finite."""
    q, k, v = (_rand(i, B, h, t, D, dtype=dtype) for i, h, t in ((6, Hkv * G, Tq), (7, Hkv, Tk), (8, Hkv, Tk)))
    lk = [Tk, 40][:B]
    for b in range(B):
        k[b, :, lk[b]:], v[b, :, lk[b]:] = math.nan, math.nan
    if Tq > 1:
        v[0, 0, Tk - 1, 0] = math.inf  # seen by the last query only
    out, lse = dense_attention(q.to(dev), k.to(dev), v.to(dev), return_lse=True,
                               lengths=torch.tensor(lk, dtype=torch.int32, device=dev))
    if Tq > 1:
        assert torch.isinf(out[0, :G, -1, 0]).all()
        out[0, :G, -1, 0] = 0
        v[0, 0, Tk - 1, 0] = 0
        vv = v.clone()
        ref_last = [attention(q[0, h], k[0, 0], vv[0, 0], True, None, HALF_STEP[dtype])[0][-1, 0] for h in range(G)]
        out[0, :G, -1, 0] = torch.tensor(ref_last, dtype=dtype, device=dev)
    _check(out.cpu(), lse.cpu(), q, k, v, [Tq] * B, lk)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,Hkv,G", [
    ([1], 1, 1),
    ([37, 0, 128, 1, 200, 65], 2, 4),
    ([0, 0, 5], 1, 3),
    ([3] * 70 + [150] + [1] * 69, 1, 2),  # more sequences than a wave has lanes
])
def test_packed_equals_each_alone(dev, dtype, D, lens, Hkv, G):
    N = sum(lens)
    lead, rest = 4, 9  # rows before the first and behind the last sequence
    total = lead + N + rest
    q, k, v = (_rand(i, total, h, D, dtype=dtype) for i, h in ((0, Hkv * G), (1, Hkv), (2, Hkv)))
    for x in (q, k, v):
        x[:lead], x[lead + N:] = math.nan, math.nan
    cu = torch.tensor([lead] + [lead + sum(lens[:i + 1]) for i in range(len(lens))], dtype=torch.int32)
    qd, kd, vd, cud = (x.to(dev) for x in (q, k, v, cu))
    out, lse = packed_attention(qd, kd, vd, cud, return_lse=True)
    for b, n in enumerate(lens):
        a = int(cu[b])
        for h in range(Hkv * G if len(lens) < 10 or n > 100 or b < 3 else 1):
            o, ls, tol, tol_l = attention(q[a:a + n, h], k[a:a + n, h // G], v[a:a + n, h // G], True, None,
                                          HALF_STEP[dtype])
            close(out[a:a + n, h], o, tol, f"sequence {b}")
            close(lse[h, a:a + n], ls, tol_l, f"sequence {b}")
    for x in (out[:lead], out[lead + N:]):
        assert (x == 0).all()
    assert (lse[:, :lead] == -math.inf).all() and (lse[:, lead + N:] == -math.inf).all()
    given = torch.full_like(out, 7.0)
    r, lse2 = packed_attention(qd, kd, vd, cud, out=given, return_lse=True)
    assert r is given and (given[:lead] == 7).all() and (given[lead + N:] == 7).all()
    assert torch.equal(given[lead:lead + N], out[lead:lead + N]) and torch.equal(lse, lse2)


def test_packed_chunks_behind_caches(dev):
    """Queries and keys packed by offsets of their own, without causality too."""
    lq, lk, Hkv, G, D, dt = [5, 1, 0, 40, 7], [100, 300, 20, 40, 3], 2, 2, 128, torch.bfloat16
    q, k, v = (_rand(i, n, h, D, dtype=dt) for i, n, h in ((0, sum(lq), Hkv * G), (1, sum(lk), Hkv), (2, sum(lk), Hkv)))
    cu = [torch.tensor([0] + [sum(x[:i + 1]) for i in range(5)], dtype=torch.int32) for x in (lq, lk)]
    for causal in (True, False):
        out, lse = packed_attention(q.to(dev), k.to(dev), v.to(dev), cu[0].to(dev), cu[1].to(dev), causal=causal,
                                    return_lse=True)
        for b in range(5):
            a, c = int(cu[0][b]), int(cu[1][b])
            for h in range(Hkv * G):
                o, ls, tol, tol_l = attention(q[a:a + lq[b], h], k[c:c + lk[b], h // G], v[c:c + lk[b], h // G], causal,
                                              None, HALF_STEP[dt])
                close(out[a:a + lq[b], h], o, tol)
                close(lse[h, a:a + lq[b]], ls, tol_l)


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(dev, dtype):
    """(B, T, H, D) memory, slices, shared (expanded) heads and rows off 16-byte boundaries give
    what their contiguous copies give; an output slice's neighbours stay."""
    B, Hkv, G, T, D = 2, 2, 2, 77, 64
    q, k, v = (_rand(i, B, T, h, D, dtype=dtype).to(dev) for i, h in ((0, Hkv * G), (1, Hkv), (2, Hkv)))
    want = dense_attention(*(x.transpose(1, 2).contiguous() for x in (q, k, v)))
    assert torch.equal(want, dense_attention(*(x.transpose(1, 2) for x in (q, k, v))))
    wide = [torch.zeros(B, x.shape[2], T + 3, D + 8, dtype=dtype, device=dev) for x in (q, k, v)]
    off = [torch.zeros(x.numel() + 1, dtype=dtype, device=dev)[1:].view(x.transpose(1, 2).shape) for x in (q, k, v)]
    for x, y, z in zip((q, k, v), wide, off):
        y[:, :, 2:-1, 8:] = x.transpose(1, 2)
        z.copy_(x.transpose(1, 2))
    assert torch.equal(want, dense_attention(*(y[:, :, 2:-1, 8:] for y in wide)))
    assert torch.equal(want, dense_attention(*off))
    one = k[:, :, :1].transpose(1, 2)  # one KV head, expanded
    assert torch.equal(dense_attention(q.transpose(1, 2), one.expand(B, Hkv, T, D), one.expand(B, Hkv, T, D)),
                       dense_attention(q.transpose(1, 2), one.repeat(1, Hkv, 1, 1), one.repeat(1, Hkv, 1, 1)))
    out = torch.full((B, Hkv * G, T, D + 16), 5.0, dtype=dtype, device=dev)
    got = dense_attention(*(x.transpose(1, 2) for x in (q, k, v)), out=out[..., 8:D + 8])
    assert torch.equal(got, want) and (out[..., :8] == 5).all() and (out[..., D + 8:] == 5).all()


def test_large_scores_and_equal_keys(dev):
    """Scores far apart (the running maximum is raised many times), and all equal."""
    for dtype in TYPES:
        D, T = 64, 400
        q, k, v = (_rand(i, 1, 1, T, D, dtype=dtype) for i in range(3))
        k = (k * torch.linspace(0.1, 12, T).view(1, 1, T, 1)).to(dtype)
        out, lse = dense_attention(q.to(dev), k.to(dev), v.to(dev), return_lse=True)
        _check(out.cpu(), lse.cpu(), q, k, v, [T], [T])
        z = torch.zeros_like(q)
        out, lse = dense_attention(z.to(dev), k.to(dev), v.to(dev), return_lse=True)
        _check(out.cpu(), lse.cpu(), z, k, v, [T], [T])


def test_offsets_past_32_bits(dev):
    """Keys that start more than 2^31 elements into their tensors."""
    D, lead, n = 128, (1 << 24) + 5, 203
    k, v = (torch.empty(lead + n, 1, D, dtype=torch.bfloat16, device=dev) for _ in range(2))
    assert k.numel() > 1 << 31
    kk, vv, q = (_rand(i, n, h, D, dtype=torch.bfloat16) for i, h in ((1, 1), (2, 1), (0, 2)))
    k[lead:], v[lead:] = kk.to(dev), vv.to(dev)
    cu_k = torch.tensor([lead, lead + n], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    got = packed_attention(q.to(dev), k, v, cu, cu_k)
    for h in range(2):
        o, _, tol, _ = attention(q[:, h], kk[:, 0], vv[:, 0], True, None, HALF_STEP[q.dtype])
        close(got[:, h], o, tol)
    del k, v
    torch.cuda.empty_cache()


def test_streams_and_graph_replays(dev):
    B, Hq, Hkv, T, D = 2, 4, 2, 1500, 128
    q, k, v = (_rand(i, B, h, t, D, dtype=torch.bfloat16).to(dev) for i, h, t in ((0, Hq, 2), (1, Hkv, T), (2, Hkv, T)))
    want, want_lse = dense_attention(q, k, v, return_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = dense_attention(q, k, v)
    side.synchronize()
    assert torch.equal(got, want)
    lengths = torch.full((B,), T, dtype=torch.int32, device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = dense_attention(q, k, v, lengths=lengths, return_lse=True)
    for n in (T, 700, 1, T):
        lengths.fill_(n)
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        eager, eager_lse = dense_attention(q, k, v, lengths=lengths, return_lse=True)
        assert torch.equal(out, eager) and torch.equal(lse, eager_lse)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Tq", [1, 32])
@pytest.mark.parametrize("gap", [0.25, 0.5, 1.1])
def test_log_sum_of_equal_weights(dtype, Tq, gap):
    """The first key's score is `gap` above all others', which are equal: a running sum that
    took the equal weights one by one would drift by up to half a step of the sum for each."""
    dev, n, D = "cuda", 20000, 64
    q, k = torch.zeros(1, 1, Tq, D), torch.zeros(1, 1, n, D)
    q[..., 0] = 1.0
    k[..., 0, 0] = gap
    q, k = q.to(dtype), k.to(dtype)
    out, lse = dense_attention(q.to(dev), k.to(dev), torch.ones_like(k).to(dev), causal=False, scale=1.0,
                               out_dtype=torch.float32, return_lse=True)
    want = math.log(math.exp(float(k[0, 0, 0, 0])) + n - 1.0)
    # a lane's share, n / 2 or fewer, in parts of 8 and more: n / 16 additions, 16 more within
    # the parts and between lanes; a few steps of exp2, log2 and the scores
    tol = (n / 16 + 24 + 2 * want) * 2.0 ** -24
    assert (lse.double().cpu() - want).abs().max() <= tol
    # O sums products of 4 (fp32) or more keys, each weight rounded to the inputs' type
    assert (out.double().cpu() - 1.0).abs().max() <= torch.finfo(dtype).eps / 2 + tol + (n / 4 + 24) * 2.0 ** -24
