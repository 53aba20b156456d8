"""``evict_kv`` and ``evict_decode_step`` against plain references on the CPU: kept entries are
exact, ties and weights that are not numbers included; the step's output and weights to
the bounds of ``dense_reference``; prompt, weights, eviction and steps as one run."""

from __future__ import annotations

import math

import pytest
import torch

from dense_reference import F32, HALF_STEP, attention, close, keep, key_weights as reference_weights, victim
from linattn_amd.kernels.dense import dense_attention, packed_attention
from linattn_amd.kernels.eviction import (evict_decode_step, evict_kv, key_weights, packed_evict_kv,
                                          packed_key_weights)

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _rand(seed, *shape, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype)


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _check(got, k, v, w, lists, capacity, positions=None):
    """got: what evict_kv returned; lists[b][h]: the kept indices of k, v, w (B, Hkv, T, ..)."""
    ko, vo, wo, po, lo = (x.cpu() for x in got)
    for b, heads in enumerate(lists):
        for h, ids in enumerate(heads):
            m = len(ids)
            at = torch.tensor(ids, dtype=torch.int64)
            assert int(lo[b]) == m
            assert torch.equal(po[b, h, :m], at.int() if positions is None else positions[b, h, at])
            assert torch.equal(ko[b, h, :m], k[b, h, at]) and torch.equal(vo[b, h, :m], v[b, h, at])
            assert torch.equal(wo[b, h, :m].nan_to_num(-1), w[b, h, at].nan_to_num(-1))
            assert (po[b, h, m:] == -1).all() and (wo[b, h, m:] == 0).all()
            assert (ko[b, h, m:] == 0).all() and (vo[b, h, m:] == 0).all()
    assert ko.shape[2] == capacity


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64), (torch.float32, 8)])
@pytest.mark.parametrize("T,budget,recent,sink,extra", [
    (1, 1, 0, 0, 0), (5, 8, 4, 2, 1), (64, 64, 0, 0, 0), (300, 64, 32, 4, 1), (300, 1, 0, 0, 0),
    (300, 64, 64, 0, 3), (1100, 1000, 0, 1000, 0), (2500, 777, 100, 3, 1),
    (2048, 100, 10, 1, 1), (2049, 2000, 7, 0, 0), (16384, 500, 50, 4, 1), (16385, 500, 50, 4, 1),  # each form's ends
    (40000, 39000, 100, 5, 1),
])
def test_evict_keeps_the_heaviest(dev, dtype, D, T, budget, recent, sink, extra):
    B, Hkv = 2, 3
    k, v = _rand(0, B, Hkv, T, D, dtype=dtype), _rand(1, B, Hkv, T, D, dtype=dtype)
    w = _rand(2, B, Hkv, T).exp()
    got = evict_kv(k.to(dev), v.to(dev), w.to(dev), budget=budget, recent=recent, sink=sink, capacity=budget + extra)
    lists = [[keep(w[b, h], T, budget, recent, sink) for h in range(Hkv)] for b in range(B)]
    _check(got, k, v, w, lists, budget + extra)


@pytest.mark.parametrize("kind", ["equal", "few", "odd", "tiny"])
def test_ties_and_odd_weights(dev, kind):
    _ties(dev, kind, 3000, (40, 1024, 2900, 2999))


@pytest.mark.parametrize("kind", ["equal", "few", "odd", "tiny"])
@pytest.mark.parametrize("T", [700, 20000])
def test_ties_in_short_and_long_caches(dev, kind, T):
    _ties(dev, kind, T, (T // 50 + 23, T // 3, T - 1))


def _ties(dev, kind, T, budgets):
    B, Hkv, D = 2, 2, 64
    k, v = _rand(0, B, Hkv, T, D), _rand(1, B, Hkv, T, D)
    w = torch.ones(B, Hkv, T) if kind == "equal" else _rand(2, B, Hkv, T)
    if kind == "few":
        w = w.round().clamp(-1, 1)  # three values, -0 and +0 among them
    if kind == "odd":
        w[:, :, ::7], w[:, :, 1::11], w[:, :, 2::13] = math.nan, math.inf, -math.inf
    if kind == "tiny":
        w = w * 1e-44  # subnormal
    for budget in budgets:
        got = evict_kv(k.to(dev), v.to(dev), w.to(dev), budget=budget, recent=20, sink=3)
        _check(got, k, v, w, [[keep(w[b, h], T, budget, 20, 3) for h in range(Hkv)] for b in range(B)], budget)


def test_evict_lengths_positions_and_layouts(dev):
    B, Hkv, T, D = 5, 2, 700, 64
    k, v = _rand(0, B, T, Hkv, D, dtype=torch.bfloat16).transpose(1, 2), _rand(1, B, T, Hkv, D, dtype=torch.bfloat16).transpose(1, 2)
    w = _rand(2, B, T, Hkv).exp().transpose(1, 2)
    lens = [700, 0, 1, 130, 64]
    got = evict_kv(k.to(dev), v.to(dev), w.to(dev), budget=64, recent=16, sink=2, lengths=_i32(lens, dev))
    _check(got, k, v, w, [[keep(w[b, h], lens[b], 64, 16, 2) for h in range(Hkv)] for b in range(B)], 64)
    _unordered(dev, k, v, w, lens, [2200, 2200, 10, 900, 2100], 100)


@pytest.mark.parametrize("T", [5000, 18000])
def test_long_caches_by_position(dev, T):
    B, Hkv, D = 3, 2, 64
    k, v, w = _rand(0, B, Hkv, T, D), _rand(1, B, Hkv, T, D), _rand(2, B, Hkv, T).exp()
    w[1] = 1.0
    _unordered(dev, k, v, w, [T, T - 7, 2100], [3 * T, 2 * T, 900], 1500)
    _unordered(dev, k, v, w, [T, T - 7, 2100], [3 * T, 2 * T, 900], 40, recent=20)


def _unordered(dev, k, v, w, lens, pos, budget, recent=30):
    # entries in no order, as a cache that decodes and evicts holds them
    B, Hkv, T = w.shape
    g = torch.Generator().manual_seed(5)
    positions = torch.rand(B, Hkv, T, generator=g).argsort(-1).to(torch.int32) * 3
    got = evict_kv(k.to(dev), v.to(dev), w.to(dev), budget=budget, recent=recent, sink=9, lengths=_i32(lens, dev),
                   positions=positions.to(dev), pos=_i32(pos, dev), capacity=budget + 1)
    lists = [[keep(w[b, h], lens[b], budget, recent, 9, positions[b, h], pos[b]) for h in range(Hkv)] for b in range(B)]
    _check(got, k, v, w, lists, budget + 1, positions)


@pytest.mark.parametrize("lens", [[1], [300, 0, 1, 64, 65, 2000], [70000, 3]])
def test_packed_evict(dev, lens):
    Hkv, D, dt = 2, 64, torch.float16
    n, lead = sum(lens), 3
    k, v = _rand(0, lead + n + 5, Hkv, D, dtype=dt), _rand(1, lead + n + 5, Hkv, D, dtype=dt)
    w = _rand(2, Hkv, lead + n + 5).exp()
    cu = [lead + sum(lens[:i]) for i in range(len(lens) + 1)]
    budget = 64 if n < 10000 else 40000
    got = packed_evict_kv(k.to(dev), v.to(dev), w.to(dev), _i32(cu, dev), budget=budget, recent=32, sink=4,
                          capacity=budget + 1)
    ko, vo, wo, po, lo = (x.cpu() for x in got)
    for b, m in enumerate(lens):
        for h in range(Hkv):
            ids = torch.tensor(keep(w[h, cu[b]:cu[b] + m], m, budget, 32, 4), dtype=torch.int64)
            c = len(ids)
            assert int(lo[b]) == c and torch.equal(po[b, h, :c], ids.int())
            assert torch.equal(ko[b, h, :c], k[cu[b] + ids, h]) and torch.equal(vo[b, h, :c], v[cu[b] + ids, h])
            assert torch.equal(wo[b, h, :c], w[h, cu[b] + ids])
            assert (po[b, h, c:] == -1).all() and (ko[b, h, c:] == 0).all() and (wo[b, h, c:] == 0).all()


class _Plain:
    """A cache kept on the CPU by the definition."""

    def __init__(self, k, v, w, positions, lengths):
        self.k, self.v, self.w, self.p, self.n = k.clone(), v.clone(), w.double(), positions.clone(), list(lengths)
        self.tol = torch.zeros_like(self.w)

    def step(self, q, kn, vn, pos, recent, sink, scale=None, seen_weights=None, out_half=None):
        """seen_weights: the weights the step under test saw (fp32), which pick the victim."""
        B, Hkv, C, D = self.k.shape
        G = q.shape[1] // Hkv
        u = HALF_STEP[q.dtype]
        out, tol = torch.zeros(B, Hkv * G, 1, D).double(), torch.zeros(B, Hkv * G, 1, D).double()
        for b in range(B):
            n = min(self.n[b] + 1, C)
            for h in range(Hkv):
                s = self.n[b] if self.n[b] < C else victim(seen_weights[b, h], recent, sink, self.p[b, h], pos[b])
                self.k[b, h, s], self.v[b, h, s] = kn[b, h, 0], vn[b, h, 0]
                self.w[b, h, s], self.tol[b, h, s], self.p[b, h, s] = 0.0, 0.0, pos[b]
                lse = torch.zeros(G, 1)
                for g in range(G):
                    i = h * G + g
                    o, ls, t, tl = attention(q[b, i], self.k[b, h, :n], self.v[b, h, :n], False, scale, u, out_half or u)
                    out[b, i], tol[b, i] = o, t
                    lse[g] = ls.float()
                add, t = reference_weights(q[b, h * G:(h + 1) * G], self.k[b, h, :n], lse, False, scale)
                self.w[b, h, :n] += add
                # (the kernel's own row sums are off by as much as the attention's)
                self.tol[b, h, :n] += 2 * t + add * float(2 * tl.max()) + F32 * self.w[b, h, :n].abs()
            self.n[b] = n
        return out, tol


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Hkv,G,C,lens", [
    (1, 1, 1, 1, [0]),
    (2, 2, 4, 33, [33, 5]),
    (1, 2, 3, 200, [200]),
    (1, 1, 16, 65, [65]),
    (1, 1, 2, 1030, [1030]),   # entries split over workgroups
    (2, 1, 5, 2051, [2051, 700]),
])
def test_steps(dev, dtype, D, B, Hkv, G, C, lens):
    """Steps one after another: caches fill up, then evict; slots behind the entries hold NaN."""
    k, v = _rand(0, B, Hkv, C, D, dtype=dtype), _rand(1, B, Hkv, C, D, dtype=dtype)
    w, g = _rand(2, B, Hkv, C).exp(), torch.Generator().manual_seed(3)
    positions = torch.rand(B, Hkv, C, generator=g).argsort(-1).to(torch.int32)
    for b in range(B):
        k[b, :, lens[b]:], v[b, :, lens[b]:], w[b, :, lens[b]:], positions[b, :, lens[b]:] = math.nan, math.nan, math.nan, -1
    recent, sink = (C - 1) // 2, min(4, (C - 1) // 2)
    plain = _Plain(k, v, w, positions, lens)
    kd, vd, wd, pd = k.to(dev), v.to(dev), w.to(dev), positions.to(dev)
    n = list(lens)
    for step in range(4):
        q, kn, vn = (_rand(10 * step + i, B, h, 1, D, dtype=dtype) for i, h in ((1, Hkv * G), (2, Hkv), (3, Hkv)))
        pos = [C + step + 7 * b for b in range(B)]
        out_dtype, scale = (torch.float32, 0.2) if step == 2 else (None, None)
        before = wd.cpu()
        out = evict_decode_step(q.to(dev), kn.to(dev), vn.to(dev), kd, vd, wd, pd, _i32(n, dev), _i32(pos, dev),
                                recent=recent, sink=sink, scale=scale, out_dtype=out_dtype)
        assert out.dtype == (out_dtype or dtype)
        ref, tol = plain.step(q, kn, vn, pos, recent, sink, scale, before, HALF_STEP[out.dtype])
        n = [min(x + 1, C) for x in n]
        assert n == plain.n
        close(out, ref, tol, f"step {step} out")
        for b in range(B):
            m = n[b]
            assert torch.equal(pd[b].cpu(), plain.p[b])
            assert torch.equal(kd[b, :, :m].cpu(), plain.k[b, :, :m]) and torch.equal(vd[b, :, :m].cpu(), plain.v[b, :, :m])
            assert torch.isnan(kd[b, :, m:]).all() and torch.isnan(wd[b, :, m:]).all()
            close(wd[b, :, :m], plain.w[b, :, :m], plain.tol[b, :, :m], f"step {step} weights")


def test_step_ties_and_protection(dev):
    """Equal weights give up the highest slot, a NaN goes first, and where everything is
    protected the highest slot goes."""
    B, Hkv, C, D = 4, 2, 100, 64
    q, kn, vn = (_rand(i, B, Hkv, 1, D).to(dev) for i in range(3))
    k, v = (_rand(i, B, Hkv, C, D).to(dev) for i in (3, 4))
    w = torch.ones(B, Hkv, C)
    w[1, :, 40], w[1, :, 10], w[2, :, 55] = 0.5, 0.5, math.nan
    w[3, 0, 3], w[3, 1, 95] = -0.0, 0.0
    positions = torch.arange(C, dtype=torch.int32).expand(B, Hkv, C).contiguous()
    pos = [C, C, C, C]
    for recent, sink in ((30, 4), (95, 4), (0, 0)):
        wd, pd = w.to(dev), positions.to(dev)
        evict_decode_step(q, kn, vn, k.clone(), v.clone(), wd, pd, _i32([C] * B, dev), _i32(pos, dev), recent=recent, sink=sink)
        for b in range(B):
            for h in range(Hkv):
                want = positions[b, h].clone()
                want[victim(w[b, h], recent, sink, positions[b, h], pos[b])] = pos[b]
                assert torch.equal(pd[b, h].cpu(), want), (recent, b, h)
    pd = torch.full((B, Hkv, C), 7, dtype=torch.int32, device=dev)  # all below the sink
    evict_decode_step(q, kn, vn, k.clone(), v.clone(), w.to(dev), pd, _i32([C] * B, dev), _i32(pos, dev), recent=1, sink=9)
    assert (pd[:, :, -1] == C).all() and (pd[:, :, :-1] == 7).all()


def test_steps_replayed(dev):
    """A captured step, replayed over lengths and positions advanced in place, equals eager
    steps; so does one on another stream, beside a step on other caches."""
    B, Hkv, G, C, D = 2, 2, 4, 1500, 128
    q, kn, vn = (_rand(i, B, h, 1, D, dtype=torch.bfloat16).to(dev) for i, h in ((1, Hkv * G), (2, Hkv), (3, Hkv)))
    state = [_rand(i, B, Hkv, C, D, dtype=torch.bfloat16).to(dev) for i in (4, 5)]
    state += [_rand(6, B, Hkv, C).exp().to(dev), torch.arange(C, dtype=torch.int32, device=dev).expand(B, Hkv, C).contiguous()]
    lengths, pos = _i32([C, C - 2], dev), _i32([C, C - 2], dev)
    a, b = [x.clone() for x in state], [x.clone() for x in state]
    kw = dict(recent=700, sink=4)
    want = []
    for step in range(4):
        want.append(evict_decode_step(q, kn, vn, *a, (lengths + step).clamp(max=C), pos + step, **kw))
    graph = torch.cuda.CUDAGraph()
    ld, pd = lengths.clone(), pos.clone()
    with torch.cuda.graph(graph):
        out = evict_decode_step(q, kn, vn, *b, ld, pd, **kw)
    for x, y in zip(b, state):
        x.copy_(y)
    for step in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[step])
        ld.add_(1).clamp_(max=C)
        pd.add_(1)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    c, d = [x.clone() for x in state], [x.clone() for x in state]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        o1 = evict_decode_step(q, kn, vn, *c, lengths, pos, **kw)
    with torch.cuda.stream(s2):
        o2 = evict_decode_step(q, kn, vn, *d, lengths, pos, **kw)
    torch.cuda.synchronize()
    assert torch.equal(o1, want[0]) and torch.equal(o2, want[0]) and torch.equal(c[2], d[2])


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_to_decode(dev, dtype):
    """Packed prompts, their weights, eviction, then tokens: against the definition all the way."""
    lens, Hkv, G, D, budget, recent, sink = [150, 40, 90], 2, 2, 64, 64, 20, 4
    N, B = sum(lens), 3
    q, k, v = (_rand(i, N, h, D, dtype=dtype) for i, h in ((0, Hkv * G), (1, Hkv), (2, Hkv)))
    cu = [0, 150, 190, 280]
    qd, kd, vd, cud = q.to(dev), k.to(dev), v.to(dev), _i32(cu, dev)
    _, lse = packed_attention(qd, kd, vd, cud, return_lse=True)
    w = packed_key_weights(qd, kd, lse, cud)
    kc, vc, wc, pc, n = packed_evict_kv(kd, vd, w, cud, budget=budget, recent=recent, sink=sink, capacity=budget + 1)
    wh = w.cpu()
    for b in range(B):
        for h in range(Hkv):
            ids = keep(wh[h, cu[b]:cu[b + 1]], lens[b], budget, recent, sink)
            assert torch.equal(pc[b, h, :len(ids)].cpu(), torch.tensor(ids, dtype=torch.int32))
    plain = _Plain(kc.cpu(), vc.cpu(), wc.cpu(), pc.cpu(), n.tolist())
    pos = torch.tensor(lens, dtype=torch.int32)
    for step in range(6):
        qn, kn, vn = (_rand(100 + 10 * step + i, B, h, 1, D, dtype=dtype) for i, h in ((1, Hkv * G), (2, Hkv), (3, Hkv)))
        before = wc.cpu()
        out = evict_decode_step(qn.to(dev), kn.to(dev), vn.to(dev), kc, vc, wc, pc, n, pos.to(dev), recent=recent, sink=sink)
        ref, tol = plain.step(qn, kn, vn, pos.tolist(), recent, sink, None, before)
        close(out, ref, tol)
        n = (n + 1).clamp(max=budget + 1)
        pos += 1
        assert torch.equal(pc.cpu(), plain.p) and n.tolist() == plain.n
    # a step equals evicting one entry, appending and attending by the other entry points
    k2, v2, w2, p2, n2 = evict_kv(kc, vc, wc, budget=budget, recent=recent, sink=sink, lengths=n, positions=pc,
                                  pos=pos.to(dev), capacity=budget + 1)
    full = (n == budget + 1).tolist()
    assert full == [True, False, True]
    qn, kn, vn = (_rand(500 + i, B, h, 1, D, dtype=dtype).to(dev) for i, h in ((1, Hkv * G), (2, Hkv), (3, Hkv)))
    for b in range(B):
        k2[b, :, int(n2[b])], v2[b, :, int(n2[b])] = kn[b, :, 0], vn[b, :, 0]
    n2 = n2 + 1
    want, lse = dense_attention(qn, k2, v2, lengths=n2, return_lse=True, out_dtype=torch.float32)
    key_weights(qn, k2, lse, lengths=n2, out=w2)
    got = evict_decode_step(qn, kn, vn, kc, vc, wc, pc, n, pos.to(dev), recent=recent, sink=sink, out_dtype=torch.float32)
    assert (got - want).norm() < 2e-3 * want.norm()
    for b in range(B):
        for h in range(Hkv):
            a = sorted(zip(pc[b, h, :int(n2[b])].tolist(), wc[b, h, :int(n2[b])].tolist()))
            c = sorted((p if p >= 0 else int(pos[b]), x) for p, x in zip(p2[b, h, :int(n2[b])].tolist(), w2[b, h, :int(n2[b])].tolist()))
            assert [x for x, _ in a] == [x for x, _ in c]
            assert all(abs(x - y) < 1e-4 * (1 + abs(y)) for (_, x), (_, y) in zip(a, c))


def test_prompts_captured_and_on_two_streams(dev):
    """Attention, weights and eviction of packed prompts as one graph, replayed over other
    sequences; two such chains at once on two streams."""
    N, Hq, Hkv, D, budget = 20000, 4, 2, 64, 600
    q, k, v = (_rand(i, N, h, D, dtype=torch.bfloat16).to(dev) for i, h in ((0, Hq), (1, Hkv), (2, Hkv)))
    cu = torch.tensor([0, 18000, 20000], dtype=torch.int32, device=dev)

    def chain():
        out, lse = packed_attention(q, k, v, cu, return_lse=True)
        w = packed_key_weights(q, k, lse, cu, last=64)
        return (out, lse, w, *packed_evict_kv(k, v, w, cu, budget=budget, recent=200, sink=4, capacity=budget + 1))

    cuts = [[0, 18000, 20000], [0, 700, 20000], [5, 5, 19000], [0, 18000, 20000]]
    want = []
    for c in cuts:
        cu.copy_(torch.tensor(c, dtype=torch.int32))
        want.append([x.clone() for x in chain()])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain()
    for c, ref in zip(cuts, want):
        cu.copy_(torch.tensor(c, dtype=torch.int32))
        for x in got:
            x.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, ref):
            assert torch.equal(x, y)
        assert torch.equal(chain()[3], ref[3])
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    results = [[], []]
    for _ in range(3):
        for s, r in zip(streams, results):
            with torch.cuda.stream(s):
                r.append(chain())
    torch.cuda.synchronize()
    for r in results:
        for once in r:
            for x, y in zip(once, want[-1]):
                assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", TYPES)
def test_nothing_to_read(dev, dtype):
    """No keys, no queries, no entries: zeros, -inf and empty caches, from tensors without rows."""
    z = lambda *s: torch.zeros(*s, dtype=dtype, device=dev)
    cu, none = _i32([0, 3, 5], dev), _i32([0, 0, 0], dev)
    for Tq in (1, 40):
        out, lse = dense_attention(z(2, 4, Tq, 64) + 1, z(2, 2, 0, 64), z(2, 2, 0, 64), return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()
    out, lse = packed_attention(z(5, 4, 64) + 1, z(0, 2, 64), z(0, 2, 64), cu, none, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    out, lse = packed_attention(z(0, 4, 64), z(5, 2, 64), z(5, 2, 64), none, cu, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (4, 0)
    w = key_weights(z(2, 4, 0, 64), z(2, 2, 70, 64), torch.zeros(2, 4, 0, device=dev))
    assert w.shape == (2, 2, 70) and (w == 0).all()
    w = packed_key_weights(z(0, 4, 64), z(5, 2, 64), torch.zeros(4, 0, device=dev), none, cu)
    assert w.shape == (2, 5) and (w == 0).all()
    assert key_weights(z(2, 4, 3, 64), z(2, 2, 0, 64), torch.zeros(2, 4, 3, device=dev)).shape == (2, 2, 0)
    for got in (evict_kv(z(2, 2, 0, 64), z(2, 2, 0, 64), torch.zeros(2, 2, 0, device=dev), budget=4, recent=2, capacity=5),
                packed_evict_kv(z(0, 2, 64), z(0, 2, 64), torch.zeros(2, 0, device=dev), none, budget=4, recent=2, capacity=5)):
        k, v, w, pos, n = got
        assert (k == 0).all() and (v == 0).all() and (w == 0).all() and (pos == -1).all() and (n == 0).all()
        assert k.shape == (2, 2, 5, 64)
    k, v, w, pos, n = evict_kv(z(0, 2, 9, 64), z(0, 2, 9, 64), torch.zeros(0, 2, 9, device=dev), budget=4, recent=2)
    assert k.shape == (0, 2, 4, 64) and n.shape == (0,)
