"""``rotary`` and ``rotary_kv_append`` against 64-bit references on the CPU: types, head sizes whose
chunks are and are not 16 bytes, one axis and several, far positions, strides, in place, packed
and batched tokens, pages of any size, tokens that no page holds, fp8 codes, Quest's bounds,
streams and graphs.  Bounds: see ``rotary_reference``."""

from __future__ import annotations

import pytest
import torch

from linattn_amd.kernels.kv_cache import paged_kv_append, rotary_kv_append
from linattn_amd.kernels.rotary import rotary, rotary_axes
from rotary_reference import HALF, U, bounds, close, places, rounded, slots, turn

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _rand(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _freq(n):
    return (10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)).float()


def _i32(x, dev=None):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _check(got, x, positions, freq, axes=None, interleaved=False, inverse=False, what=""):
    want, tol = turn(x, positions, freq, axes, interleaved, inverse)
    close(got, want, rounded(want, tol, x.dtype), what)
    n = 2 * freq.shape[0]
    assert torch.equal(got[..., n:].cpu(), x[..., n:])  # what is not turned is copied


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("N,Hq,Hkv,D,n", [
    (1, 32, 8, 128, 64),
    (37, 8, 2, 64, 32),
    (300, 5, 1, 80, 40),     # ten chunks of 16 bytes a row
    (65, 4, 4, 72, 36),      # chunks of 8
    (130, 3, 1, 96, 12),     # an eighth is turned
    (20, 2, 2, 50, 25),      # one value at a time
    (3, 1, 1, 512, 256),
    (700, 12, 4, 40, 4),     # most is copied, an odd number of chunks
    (2, 1, 0, 2, 1),
])
def test_rotary(dev, dtype, interleaved, N, Hq, Hkv, D, n):
    q, k = _rand(1, N, Hq, D, dtype=dtype), _rand(2, N, Hkv, D, dtype=dtype) if Hkv else None
    pos = torch.randint(-50, 5000, (N,), generator=torch.Generator().manual_seed(3)).int()
    freq = _freq(n)
    for inverse in (False, True):
        r = rotary(q.to(dev), None if k is None else k.to(dev), pos.to(dev), freq.to(dev), interleaved=interleaved,
                   inverse=inverse)
        gq, gk = r if k is not None else (r, None)
        assert gq.dtype == dtype and gq.is_contiguous()
        _check(gq, q, pos, freq, None, interleaved, inverse, "q")
        if k is not None:
            _check(gk, k, pos, freq, None, interleaved, inverse, "k")


@pytest.mark.parametrize("dtype", TYPES)
def test_far_positions_keep_their_phase(dev, dtype):
    pos = torch.tensor([0, 1, 2 ** 31 - 1, -2 ** 31, 1 << 20, 123456789, 16777217, -77], dtype=torch.int32)
    q = _rand(4, 8, 3, 64, dtype=dtype)
    for freq in (_freq(32), torch.full((32,), 1.0), _rand(5, 32).abs() * 3):
        _check(rotary(q.to(dev), None, pos.to(dev), freq.to(dev)), q, pos, freq)


@pytest.mark.parametrize("interleaved", [False, True])
def test_axes(dev, interleaved):
    axes = rotary_axes((8, 10, 14), interleaved)
    assert axes.bincount().tolist() == [8, 10, 14]
    if interleaved:
        assert axes[:7].tolist() == [0, 1, 2, 0, 1, 2, 0] and axes[-4:].tolist() == [2, 2, 2, 2]
    pos = torch.randint(0, 3000, (3, 77), generator=torch.Generator().manual_seed(6)).int()
    q, k, freq = _rand(7, 77, 4, 64).bfloat16(), _rand(8, 77, 2, 64).bfloat16(), _freq(32)
    gq, gk = rotary(q.to(dev), k.to(dev), pos.to(dev), freq.to(dev), axes=axes.to(dev))
    _check(gq, q, pos, freq, axes)
    _check(gk, k, pos, freq, axes)
    # batched, positions of each sequence; axes behind the last are the last
    pos4 = torch.randint(0, 300, (2, 3, 11), generator=torch.Generator().manual_seed(9)).int()
    x, far = _rand(10, 3, 2, 11, 64).bfloat16(), torch.where(axes == 2, 7, axes)
    got = rotary(x.to(dev), None, pos4.to(dev), freq.to(dev), axes=far.to(dev))
    for b in range(3):
        _check(got[b].transpose(0, 1), x[b].transpose(0, 1), pos4[:, b], freq, axes.clamp(max=1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_in_place_and_gradient(dev, dtype):
    B, Hq, Hkv, T, D = 2, 6, 2, 45, 64
    freq = _freq(32)
    qkv = _rand(11, B, T, Hq + 2 * Hkv, D, dtype=dtype)  # the heads of a token side by side
    pos = torch.randint(0, 900, (B, T), generator=torch.Generator().manual_seed(12)).int()
    there = qkv.to(dev)
    q, k = there[:, :, :Hq].transpose(1, 2), there[:, :, Hq:Hq + Hkv].transpose(1, 2)
    new_q, new_k = rotary(q, k, pos.to(dev), freq.to(dev))
    rotary(q, k, pos.to(dev), freq.to(dev), q_out=q, k_out=k)  # in place
    assert torch.equal(there[:, :, :Hq].transpose(1, 2), new_q) and torch.equal(there[:, :, Hq:Hq + Hkv].transpose(1, 2), new_k)
    assert torch.equal(there[:, :, Hq + Hkv:].cpu(), qkv[:, :, Hq + Hkv:])
    for b in range(B):
        _check(new_q[b].transpose(0, 1), qkv[b, :, :Hq], pos[b], freq)
        _check(new_k[b].transpose(0, 1), qkv[b, :, Hq:Hq + Hkv], pos[b], freq)
    # one row of positions for every sequence, rows one value apart from 16 bytes
    odd = torch.zeros(B, Hq, T, D + 1, dtype=dtype)
    odd[..., 1:] = qkv[:, :, :Hq].transpose(1, 2)
    got = rotary(odd.to(dev)[..., 1:], None, pos[:1].expand(B, T).to(dev), freq.to(dev))
    for b in range(B):
        _check(got[b].transpose(0, 1), qkv[b, :, :Hq], pos[0], freq)
    if dtype == torch.float32:
        # the gradient of <w, turned x> by x is w turned back: as the formula and as differences have it
        x, w = _rand(13, 5, 2, D), _rand(14, 5, 2, D)
        p = _i32([0, 3, 11, 500, 70000])
        back = rotary(w.to(dev), None, p.to(dev), freq.to(dev), inverse=True).cpu().double()
        xd = x.double().requires_grad_()
        (turn(xd, p, freq)[0] * w.double()).sum().backward()
        close(back, xd.grad, 12 * U * (w.abs().double().amax() * 2) * torch.ones_like(back))
        for i in range(0, D, 7):
            step = torch.zeros_like(x)
            step[..., i] = 0.5  # (linear: differences are exact but for roundings)
            up, down = (rotary((x + z).to(dev), None, p.to(dev), freq.to(dev)).cpu().double() for z in (step, -step))
            diff = ((up - down) * w.double()).sum(-1)
            tol = 16 * U * ((x.abs().double() + 1).amax(-1) * w.abs().double().sum(-1)) + 1e-12
            close(diff, back[..., i], tol)


def test_nothing_and_streams(dev):
    freq = _freq(16).to(dev)
    q = torch.empty(0, 4, 32, device=dev)
    assert rotary(q, None, _i32([], dev), freq).shape == (0, 4, 32)
    x = _rand(15, 9, 0, 32).to(dev), _rand(16, 9, 2, 32).to(dev)
    p = torch.arange(9, dtype=torch.int32, device=dev)
    a, b = rotary(*x, p, freq)
    assert a.shape == (9, 0, 32) and torch.equal(b, rotary(x[1], None, p, freq))
    s = torch.cuda.Stream(dev)
    with torch.cuda.stream(s):
        c = rotary(x[1], None, p, freq)
    s.synchronize()
    assert torch.equal(b, c)


# ---------------------------------------------------------------- the append ----
def _case(seed, lq, before, page, Hq, Hkv, D, dtype, spare=3):
    """Tokens packed, pools of stale values and a table of pages in any order."""
    g = torch.Generator().manual_seed(seed)
    B, N = len(lq), sum(lq)
    pages = [-(-(x + n) // page) for x, n in zip(before, lq)]
    n_phys, width = sum(pages) + spare, max(pages) + 1
    order = torch.randperm(n_phys, generator=g)
    table, at = torch.full((B, width), -1, dtype=torch.int32), 0
    for b in range(B):
        table[b, :pages[b]] = order[at:at + pages[b]]
        at += pages[b]
    q, k, v = (torch.randn(N, h, D, generator=g).to(dtype) for h in (Hq, Hkv, Hkv))
    kp, vp = (torch.randn(n_phys, Hkv, page, D, generator=g) for _ in range(2))
    return q, k, v, kp, vp, table


def _expect(q, k, v, kp, vp, table, positions, lq, freq, rot=None, axes=None, interleaved=False):
    """Pools' new rows and turned queries: values and bounds."""
    b, t = places(positions, lq)
    ok, phys, slot = slots(table, b, t, kp.shape[2], kp.shape[0])
    at = t if rot is None else rot
    return b, t, ok, phys, slot, turn(q, at, freq, axes, interleaved), turn(k, at, freq, axes, interleaved)


SHAPES = [
    # lq, before, page, Hq, Hkv, D, n
    ([1], [0], 16, 8, 2, 128, 64),
    ([1] * 70, list(range(70)), 16, 4, 1, 64, 32),            # more sequences than a wave has lanes
    ([5, 0, 33, 1, 64, 0], [0, 7, 31, 100, 63, 3], 16, 4, 2, 64, 32),
    ([100], [13], 24, 5, 1, 80, 40),
    ([3, 40], [1000, 0], 1, 2, 2, 64, 8),                      # a page a token
    ([50, 7], [0, 5], 128, 12, 4, 72, 36),
    ([9], [2], 5, 2, 1, 30, 15),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lq,before,page,Hq,Hkv,D,n", SHAPES)
def test_append(dev, dtype, lq, before, page, Hq, Hkv, D, n):
    q, k, v, kp, vp, table = _case(20, lq, before, page, Hq, Hkv, D, dtype)
    freq = _freq(n)
    kp, vp = kp.to(dtype), vp.to(dtype)
    cu = torch.tensor([sum(lq[:i]) for i in range(len(lq) + 1)], dtype=torch.int32)
    b, t, ok, phys, slot, (wq, tq), (wk, tk) = _expect(q, k, v, kp, vp, table, before, lq, freq)
    assert ok.all()
    gk, gv = kp.to(dev), vp.to(dev)
    gq = rotary_kv_append(q.to(dev), k.to(dev), v.to(dev), gk, gv, table.to(dev), _i32(before, dev), freq.to(dev),
                          cu_seqlens=cu.to(dev))
    close(gq, wq, rounded(wq, tq, dtype), "q")
    close(gk[phys, :, slot], wk, rounded(wk, tk, dtype), "k")
    assert torch.equal(gv[phys, :, slot].cpu(), v)
    # every other slot as it was
    untouched = torch.ones(kp.shape[0], page, dtype=torch.bool)
    untouched[phys, slot] = False
    for got, was in ((gk, kp), (gv, vp)):
        assert torch.equal(got.cpu().transpose(1, 2)[untouched], was.transpose(1, 2)[untouched])
    # without q, and k alone the same bits
    k2, v2 = kp.to(dev), vp.to(dev)
    assert rotary_kv_append(None, k.to(dev), v.to(dev), k2, v2, table.to(dev), _i32(before, dev), freq.to(dev),
                            cu_seqlens=cu.to(dev)) is None
    assert torch.equal(k2, gk) and torch.equal(v2, gv)
    # the same as rotary on its own
    assert torch.equal(gq, rotary(q.to(dev), None, t.int().to(dev), freq.to(dev)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("lq,before,page,Hq,Hkv,D,n", [SHAPES[i] for i in (0, 1, 2, 3, 5)])
def test_append_fp8(dev, dtype, lq, before, page, Hq, Hkv, D, n):
    q, k, v, kp, vp, table = _case(21, lq, before, page, Hq, Hkv, D, dtype)
    v[0, 0] = 0.0
    freq = _freq(n)
    cu = torch.tensor([sum(lq[:i]) for i in range(len(lq) + 1)], dtype=torch.int32)
    b, t, ok, phys, slot, (wq, tq), (wk, tk) = _expect(q, k, v, kp, vp, table, before, lq, freq, interleaved=True)
    kp, vp = (x.to(torch.float8_e4m3fn) for x in (kp, vp))
    pairs = torch.zeros(*kp.shape[:3], 2, device=dev)
    plain = torch.zeros(2, *kp.shape[:3], device=dev)
    for ks, vs in ((pairs[..., 0], pairs[..., 1]), (plain[0], plain[1])):
        gk, gv = kp.to(dev), vp.to(dev)
        gq = rotary_kv_append(q.to(dev), k.to(dev), v.to(dev), gk, gv, table.to(dev), _i32(before, dev), freq.to(dev),
                              cu_seqlens=cu.to(dev), interleaved=True, k_scale=ks, v_scale=vs)
        close(gq, wq, rounded(wq, tq, dtype), "q")
        for got, sc, want, tol in ((gk, ks, wk, tk), (gv, vs, v.double(), torch.zeros_like(wk))):
            scale = want.abs().amax(-1).clamp(min=1e-8) / 448
            off = tol.amax(-1) / 448 + 2 * U * scale
            s = sc[phys, :, slot].cpu().double()
            close(s, scale, off, "scale")
            codes = got.view(torch.uint8)[phys, :, slot].cpu().view(torch.float8_e4m3fn).double()
            # a code is off by half a step (2^-4 of it, 2^-10 below the smallest normal one) of what
            # was divided, which is off by the turn and by its scale's and the division's roundings
            close(codes * s[..., None], want, tol + want.abs() * (2.0 ** -4 + 4 * U) + (2.0 ** -10 + 1e-6) * scale[..., None], "code")
    assert torch.equal(plain[0], pairs[..., 0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lq,before,page,mp,Hq,Hkv,D,n", [
    ([1, 1, 1], [0, 15, 16], 16, 16, 8, 2, 128, 64),
    ([5, 0, 33, 1, 64, 0], [0, 7, 31, 100, 63, 3], 16, 16, 4, 2, 64, 32),
    ([200, 70], [50, 0], 24, 64, 2, 1, 64, 32),     # pages of bounds and of the pool differ
    ([1] * 67, [3 * i for i in range(67)], 8, 4, 2, 2, 64, 32),
    ([100], [7], 64, 40, 3, 3, 72, 36),             # bounds' pages in more than one step
    ([6], [0], 16, 16, 2, 1, 30, 15),
])
def test_append_bounds(dev, dtype, lq, before, page, mp, Hq, Hkv, D, n):
    q, k, v, kp, vp, table = _case(22, lq, before, page, Hq, Hkv, D, dtype)
    B, freq = len(lq), _freq(n)
    kp, vp = kp.to(dtype), vp.to(dtype)
    cu = torch.tensor([sum(lq[:i]) for i in range(B + 1)], dtype=torch.int32)
    P = max(-(-(x + y) // mp) for x, y in zip(before, lq))
    b, t, ok, phys, slot, (wq, tq), (wk, tk) = _expect(q, k, v, kp, vp, table, before, lq, freq)
    mn, mx = (_rand(s, B, Hkv, P, D, dtype=dtype) for s in (23, 24))
    mn, mx = torch.minimum(mn, mx), torch.maximum(mn, mx)
    for minor in (False, True):  # (pages or dims side by side)
        gk, gv = kp.to(dev), vp.to(dev)
        gmn, gmx = ((x.transpose(2, 3).contiguous().to(dev).transpose(2, 3) if minor else x.to(dev)) for x in (mn, mx))
        gq = rotary_kv_append(q.to(dev), k.to(dev), v.to(dev), gk, gv, table.to(dev), _i32(before, dev), freq.to(dev),
                              cu_seqlens=cu.to(dev), page_min=gmn, page_max=gmx, page_size=mp)
        close(gq, wq, rounded(wq, tq, dtype), "q")
        stored = gk[phys, :, slot].cpu()
        close(stored, wk, rounded(wk, tk, dtype), "k")
        assert torch.equal(gv[phys, :, slot].cpu(), v)
        emn, emx = bounds(mn, mx, stored, b, t, ok, before, mp)
        assert torch.equal(gmn.cpu(), emn) and torch.equal(gmx.cpu(), emx)


@pytest.mark.parametrize("with_bounds", [False, True])
def test_tokens_that_no_page_holds(dev, with_bounds):
    """Places before the first and behind the last page, pages that are none of the pool's: not
    stored, and in no bounds; their queries are turned.  Rows of no sequence: zeros, or left."""
    dtype, page, Hq, Hkv, D = torch.bfloat16, 8, 4, 2, 64
    lq, before = [6, 20, 5, 9], [-3, 10, 100000, 0]
    q, k, v, kp, vp, _ = _case(25, lq, [0, 10, 0, 0], page, Hq, Hkv, D, dtype, spare=9)
    table = torch.tensor([[0, 1, 2, 3], [4, -1, 6, 7], [8, 9, 1, 1], [10 ** 6, 5, 2, 2]], dtype=torch.int32)
    freq = _freq(32)
    kp, vp = kp.to(dtype), vp.to(dtype)
    front, rest = 3, 4  # rows of no sequence before and behind
    pad = lambda x: torch.cat([torch.full((front, *x.shape[1:]), float("nan")).to(dtype), x,
                               torch.full((rest, *x.shape[1:]), float("nan")).to(dtype)])
    cu = _i32([front + sum(lq[:i]) for i in range(5)], dev)
    b, t, ok, phys, slot, (wq, tq), (wk, tk) = _expect(q, k, v, kp, vp, table, before, lq, freq)
    assert 0 < int(ok.sum()) < ok.numel()
    mn, mx = (_rand(s, 4, Hkv, 4, D, dtype=dtype) for s in (26, 27))
    more, gmn, gmx = {}, mn.to(dev), mx.to(dev)
    if with_bounds:
        more = dict(page_min=gmn, page_max=gmx, page_size=page)
    gk, gv = kp.to(dev), vp.to(dev)
    args = (pad(k).to(dev), pad(v).to(dev), gk, gv, table.to(dev), _i32(before, dev), freq.to(dev))
    gq = rotary_kv_append(pad(q).to(dev), *args, cu_seqlens=cu, **more)
    close(gq[front:-rest], wq, rounded(wq, tq, dtype), "q")
    assert (gq[:front] == 0).all() and (gq[-rest:] == 0).all()
    if with_bounds:
        emn, emx = bounds(mn, mx, gk[phys, :, slot].cpu(), b, t, ok, before, page)
        assert torch.equal(gmn.cpu(), emn) and torch.equal(gmx.cpu(), emx)
    close(gk[phys, :, slot].cpu()[ok], wk[ok], rounded(wk, tk, dtype)[ok], "k")
    untouched = torch.ones(kp.shape[0], page, dtype=torch.bool)
    untouched[phys[ok], slot[ok]] = False
    for got, was in ((gk, kp), (gv, vp)):
        assert torch.equal(got.cpu().transpose(1, 2)[untouched], was.transpose(1, 2)[untouched])
    out = torch.full_like(pad(q), 7.0).to(dev)
    rotary_kv_append(pad(q).to(dev), *args, cu_seqlens=cu, q_out=out, **more)
    assert (out[:front] == 7).all() and (out[-rest:] == 7).all() and torch.equal(out[front:-rest], gq[front:-rest])


@pytest.mark.parametrize("with_bounds", [False, True])
def test_batched_axes_and_in_place(dev, with_bounds):
    """(B, H, Tn, D) of a larger tensor, positions of their own on three axes, q in place."""
    dtype, page, B, Hq, Hkv, T, D = torch.float16, 16, 3, 6, 3, 21, 64
    lq, before = [T] * B, [0, 30, 11]
    q, k, v, kp, vp, table = _case(28, lq, before, page, Hq, Hkv, D, dtype)
    kp, vp, freq, axes = kp.to(dtype), vp.to(dtype), _freq(32), rotary_axes((8, 12, 12))
    rot = torch.randint(0, 500, (3, B, T), generator=torch.Generator().manual_seed(29)).int()
    b, t, ok, phys, slot, (wq, tq), (wk, tk) = _expect(q, k, v, kp, vp, table, before, lq, freq, rot.flatten(1), axes)
    whole = torch.cat([q, k, v], 1).view(B, T, Hq + 2 * Hkv, D).to(dev)
    hq, hk, hv = (whole[:, :, a:e].transpose(1, 2) for a, e in ((0, Hq), (Hq, Hq + Hkv), (Hq + Hkv, Hq + 2 * Hkv)))
    more, (mn, mx) = {}, (_rand(s, B, Hkv, 4, D, dtype=dtype) for s in (30, 31))
    gmn, gmx = mn.to(dev), mx.to(dev)
    if with_bounds:
        more = dict(page_min=gmn, page_max=gmx, page_size=16)
    gk, gv = kp.to(dev), vp.to(dev)
    got = rotary_kv_append(hq, hk, hv, gk, gv, table.to(dev), _i32(before, dev), freq.to(dev), rotary_positions=rot.to(dev),
                           axes=axes.to(dev), q_out=hq, **more)
    assert got is hq
    close(whole[:, :, :Hq].flatten(0, 1), wq, rounded(wq, tq, dtype), "q")
    assert torch.equal(whole[:, :, Hq:].cpu(), torch.cat([k, v], 1).view(B, T, 2 * Hkv, D))
    close(gk[phys, :, slot], wk, rounded(wk, tk, dtype), "k")
    assert torch.equal(gv[phys, :, slot].cpu(), v)
    if with_bounds:
        emn, emx = bounds(mn, mx, gk[phys, :, slot].cpu(), b, t, ok, before, 16)
        assert torch.equal(gmn.cpu(), emn) and torch.equal(gmx.cpu(), emx)


def test_without_a_turn_it_is_paged_kv_append(dev):
    """At position 0 nothing turns: pools and bounds are those of ``paged_kv_append``, bit for bit."""
    B, Hkv, T, D, page = 2, 2, 19, 64, 16
    _, k, v, kp, vp, table = _case(32, [T] * B, [5, 16], page, 2, Hkv, D, torch.bfloat16)
    k, v = (x.view(B, T, Hkv, D).transpose(1, 2).contiguous().to(dev) for x in (k, v))
    mn, mx = (_rand(s, B, Hkv, 4, D).bfloat16().to(dev) for s in (33, 34))
    still = torch.zeros(B, T, dtype=torch.int32, device=dev)
    results = []
    for turned in (False, True):
        pools = [kp.bfloat16().to(dev), vp.bfloat16().to(dev)]
        more = dict(page_min=mn.clone(), page_max=mx.clone(), page_size=page)
        args = (k, v, *pools, table.to(dev), _i32([5, 16], dev))
        if turned:
            rotary_kv_append(None, *args, _freq(32).to(dev), rotary_positions=still, **more)
        else:
            paged_kv_append(*args, **more)
        results.append((*pools, more["page_min"], more["page_max"]))
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_captured_and_replayed(dev):
    """A decode step in a graph: positions are read on the device, a replay goes by what they hold then."""
    B, page, Hq, Hkv, D = 4, 16, 8, 2, 128
    lq, before = [1] * B, [3, 15, 16, 40]
    q, k, v, kp, vp, table = _case(35, [6] * B, before, page, Hq, Hkv, D, torch.bfloat16)
    q, k, v = q[:B].to(dev), k[:B].to(dev), v[:B].to(dev)
    freq, cu, table = _freq(64).to(dev), torch.arange(B + 1, dtype=torch.int32, device=dev), table.to(dev)
    pos = _i32(before, dev)
    mn, mx = (_rand(s, B, Hkv, 4, D).bfloat16().to(dev) for s in (36, 37))
    def step(kp, vp, mn, mx, out):
        rotary_kv_append(q, k, v, kp, vp, table, pos, freq, cu_seqlens=cu, q_out=out, page_min=mn, page_max=mx, page_size=page)
    eager = [kp.bfloat16().to(dev), vp.bfloat16().to(dev), mn.clone(), mx.clone(), torch.empty_like(q)]
    held = [x.clone() for x in eager]
    step(*[x.clone() for x in held])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(*held)
    for i in range(4):
        step(*eager)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, held):
            assert torch.equal(a, b), i
        pos.add_(1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_bounds_of_the_widest_heads(dev, dtype):
    """512 values, all of them turned: the angles of 32 tokens are 64 KB."""
    lq, before, page, Hq, Hkv, D, n = [70, 1], [10, 31], 32, 2, 1, 512, 256
    q, k, v, kp, vp, table = _case(38, lq, before, page, Hq, Hkv, D, dtype)
    freq, kp, vp = _freq(n), kp.to(dtype), vp.to(dtype)
    b, t, ok, phys, slot, (wq, tq), (wk, tk) = _expect(q, k, v, kp, vp, table, before, lq, freq)
    mn, mx = (_rand(s, 2, Hkv, 3, D, dtype=dtype) for s in (39, 40))
    gk, gv, gmn, gmx = (x.to(dev) for x in (kp, vp, mn, mx))
    gq = rotary_kv_append(q.to(dev), k.to(dev), v.to(dev), gk, gv, table.to(dev), _i32(before, dev), freq.to(dev),
                          cu_seqlens=_i32([0, 70, 71], dev), page_min=gmn, page_max=gmx, page_size=page)
    close(gq, wq, rounded(wq, tq, dtype), "q")
    stored = gk[phys, :, slot].cpu()
    close(stored, wk, rounded(wk, tk, dtype), "k")
    assert torch.equal(gv[phys, :, slot].cpu(), v)
    emn, emx = bounds(mn, mx, stored, b, t, ok, before, page)
    assert torch.equal(gmn.cpu(), emn) and torch.equal(gmx.cpu(), emx)


@pytest.mark.parametrize("with_bounds", [False, True])
@pytest.mark.parametrize("B", [65, 700, 9000])
def test_batches_of_mostly_empty_sequences(dev, with_bounds, B):
    """Slots of a server of which few are in use, the first and last among them."""
    dtype, page, Hq, Hkv, D = torch.bfloat16, 16, 4, 2, 64
    used = {0: (1, 30), 1: (40, 0), 3: (1, 17), 31: (0, 50), 32: (20, 9), 63: (1, 1), 64: (2, 14), B - 2: (1, 15), B - 1: (33, 20)}
    lq, before = ([used.get(b, (0, 5))[i] for b in range(B)] for i in (0, 1))
    q, k, v, kp, vp, table = _case(41, lq, before, page, Hq, Hkv, D, dtype)
    freq, kp, vp = _freq(32), kp.to(dtype), vp.to(dtype)
    b, t, ok, phys, slot, (wq, tq), (wk, tk) = _expect(q, k, v, kp, vp, table, before, lq, freq)
    mn, mx = (_rand(s, B, Hkv, 4, D, dtype=dtype) for s in (42, 43))
    gk, gv, gmn, gmx = (x.to(dev) for x in (kp, vp, mn, mx))
    more = dict(page_min=gmn, page_max=gmx, page_size=page) if with_bounds else {}
    cu = _i32([sum(lq[:i]) for i in range(B + 1)], dev)
    gq = rotary_kv_append(q.to(dev), k.to(dev), v.to(dev), gk, gv, table.to(dev), _i32(before, dev), freq.to(dev),
                          cu_seqlens=cu, **more)
    close(gq, wq, rounded(wq, tq, dtype), "q")
    stored = gk[phys, :, slot].cpu()
    close(stored, wk, rounded(wk, tk, dtype), "k")
    assert torch.equal(gv[phys, :, slot].cpu(), v)
    if with_bounds:
        emn, emx = bounds(mn, mx, stored, b, t, ok, before, page)
        assert torch.equal(gmn.cpu(), emn) and torch.equal(gmx.cpu(), emx)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float32, 80), (torch.float16, 30)])
@pytest.mark.parametrize("page,mp", [(16, 16), (24, 300), (64, 48)])
@pytest.mark.parametrize("packed", [False, True])
def test_many_tokens_as_few_at_a_time(dev, dtype, D, page, mp, packed):
    """What a call turns and stores is what calls of a few tokens each do, bit for bit, and its bounds are of
    the keys as stored: pages of more tokens than a workgroup has threads, places outside of the table and
    pages outside of the pool among them.  (The bounds of both need not be the same: where a page's first
    tokens are stored nowhere, a later call that brings its others keeps its old bounds.)"""
    Hq, Hkv, T, before = 8, 4, 410, [-9, 37, 700, 0]
    B, P = len(before), 1100 // page
    g = torch.Generator().manual_seed(44)
    table = torch.randperm(B * P, generator=g).int().view(B, P)
    table[1, 100 // page], table[3, 0] = -1, 10 ** 6
    table = table.to(dev)
    q, k, v = (torch.randn(B, T, h, D, generator=g).to(dtype).to(dev) for h in (Hq, Hkv, Hkv))
    old = [torch.randn(B * P, Hkv, page, D, generator=g).to(dtype).to(dev) for _ in "kv"]
    M = P * page // mp + 1
    low = (torch.randn(B, Hkv, M, D, generator=g) - 1).to(dtype).to(dev)
    freq, results = _freq(D // 2).to(dev), []
    for step in (T, 30 if packed else 31):
        pools, mn, mx = [x.clone() for x in old], low.clone(), -low
        out, want = [], (low.cpu(), -low.cpu())
        for t in range(0, T, step):
            n = min(step, T - t)
            part = [x[:, t:t + n] for x in (q, k, v)]
            pos = _i32([b + t for b in before], dev)
            more = dict(page_min=mn, page_max=mx, page_size=mp)
            if packed:
                o = rotary_kv_append(*[x.reshape(B * n, -1, D) for x in part], *pools, table, pos, freq,
                                     cu_seqlens=_i32([n * b for b in range(B + 1)], dev), **more).view(B, n, Hq, D)
            else:
                o = rotary_kv_append(*[x.transpose(1, 2) for x in part], *pools, table, pos, freq, **more).transpose(1, 2)
            out.append(o)
            at = [b + t for b in before]
            seq, place = places(at, [n] * B)
            ok, phys, slot = slots(table.cpu(), seq, place, page, B * P)
            want = bounds(*want, pools[0].cpu()[phys, :, slot], seq, place, ok, at, mp)
            for got, x in zip((mn, mx), want):
                assert torch.equal(got.cpu(), x), (step, t)
        results.append([torch.cat(out, 1), *pools])
    for a, b in zip(*results):
        assert torch.equal(a, b)
