"""Serving from a paged cache: rotary positions on several axes, the rotation and append of new
keys and values to the pages, and dense attention of the new tokens over the pages: what these
operators cost.

``listed()`` names the calls, ``draw(rng)`` makes another of the same ranges, ``prepare``
builds what a program has in hand, ``run`` is one pass: by plain torch operations, or, where
``own`` is set, through the framework's entry points.  ``work`` counts the bytes and operations
a pass cannot do without, ``exact`` is the result in 64 bits.
"""

import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "fp8": torch.float8_e4m3fn}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "fp8": 1}
_NINF = float("-inf")
_ROOM = 16 << 30  # bytes of scores the plain form holds at a time


# ------------------------------------------------------------------ cases ----
# rotary: N tokens packed, the first R of D dims turned (in halves, or in neighbours), by one
#   position or by three (time, height, width); `start`: the first position; inverse: the
#   gradient's direction
# append, attend: B sequences bring `new` tokens together, `ones` of them a single one, the others
#   unevenly many, behind up to T tokens in pages of `page`; kv: what the pages hold
def listed():
    return [
        # a token of one user, far into its conversation: launches and latency
        dict(name="rotary_token", kind="rotary", N=1, Hq=32, Hkv=8, D=128, R=128, axes=1, start=1000003,
             neighbours=False, inverse=False, dtype="bf16"),
        # the patches of a few images and a video: three axes, an odd number of tokens
        dict(name="rotary_video", kind="rotary", N=12345, Hq=16, Hkv=16, D=80, R=80, axes=3, start=0,
             neighbours=False, inverse=False, dtype="fp16"),
        # the gradient of a long training batch
        dict(name="rotary_gradient", kind="rotary", N=32768, Hq=32, Hkv=8, D=128, R=128, axes=1, start=0,
             neighbours=True, inverse=True, dtype="bf16"),
        # a token of each of 64 sequences into the pages that Quest selects from, bounds kept
        dict(name="append_quest", kind="append", B=64, new=64, ones=64, T=8191, page=64, mix=1, Hq=32, Hkv=8,
             D=128, dtype="bf16", kv="bf16", bounds=True),
        # the chunks of four prompts into an fp8 cache
        dict(name="append_fp8", kind="append", B=4, new=2048, ones=0, T=8192, page=64, mix=2, Hq=32, Hkv=8,
             D=128, dtype="bf16", kv="fp8", bounds=False),
        # twelve whole prompts into small pages
        dict(name="append_prompts", kind="append", B=12, new=14567, ones=0, T=0, page=16, mix=3, Hq=32, Hkv=8,
             D=128, dtype="bf16", kv="bf16", bounds=False),
        # one user's short conversation, fp32 at the harness's head size: the smallest call
        dict(name="attend_short", kind="attend", B=1, new=5, ones=0, T=130, page=16, mix=4, Hq=8, Hkv=8, D=64,
             dtype="fp32", kv="fp32"),
        # a decode step of a full batch, contexts of very different length
        dict(name="attend_tokens", kind="attend", B=48, new=48, ones=48, T=16384, page=64, mix=5, Hq=32, Hkv=8,
             D=128, dtype="bf16", kv="bf16"),
        # a decode step of few users with long contexts in an fp8 cache
        dict(name="attend_tokens_fp8", kind="attend", B=8, new=8, ones=8, T=65537, page=64, mix=6, Hq=32, Hkv=8,
             D=128, dtype="bf16", kv="fp8"),
        # chunked prefill: the next tokens of four prompts
        dict(name="attend_chunks", kind="attend", B=4, new=2048, ones=0, T=8192, page=16, mix=7, Hq=32, Hkv=8,
             D=128, dtype="fp16", kv="fp16"),
        # what a server runs most: the tokens of many sequences and the chunks of two prompts
        dict(name="attend_mixed", kind="attend", B=34, new=1056, ones=32, T=12000, page=64, mix=8, Hq=32, Hkv=8,
             D=128, dtype="bf16", kv="bf16"),
        # a large chunk of one very long prompt: the largest call
        dict(name="attend_long", kind="attend", B=1, new=8192, ones=0, T=24576, page=64, mix=9, Hq=32, Hkv=8,
             D=128, dtype="bf16", kv="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "append", "attend", "attend", "attend"])
    Hq, Hkv = rng.choice([(32, 8), (16, 8), (16, 4), (8, 8), (8, 1), (12, 4), (5, 1)])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "rotary":
        D, R = rng.choice([(128, 128), (64, 64), (80, 80), (128, 64), (96, 24), (72, 72)])
        return dict(kind=kind, N=_log(rng, 1, 16384), Hq=Hq, Hkv=Hkv, D=D, R=R, axes=rng.choice([1, 1, 3]),
                    start=rng.choice([0, rng.randint(0, 2000000)]), neighbours=rng.random() < 0.5,
                    inverse=rng.random() < 0.5, dtype=dtype)
    kv = "fp8" if dtype != "fp32" and rng.random() < 0.3 else dtype
    c = dict(kind=kind, page=rng.choice([16, 16, 64, 64, 128, 24]), mix=rng.randint(0, 999), Hq=Hq, Hkv=Hkv,
             D=rng.choice([64, 128]), dtype=dtype, kv=kv)
    shape = rng.choice(["tokens", "chunks", "mixed"])
    B = _log(rng, 1, 48) if shape == "tokens" else rng.randint(1, 8)
    if shape == "mixed":
        ones = _log(rng, 1, 32)
    else:
        ones = B if shape == "tokens" else 0
    if kind == "append":
        B = ones + (B if shape == "mixed" else 0) if ones else B
        new = ones + (_log(rng, B - ones, 8192) if B > ones else 0)
        return dict(c, B=B, new=new, ones=ones, T=rng.choice([0, _log(rng, 16, 8192)]),
                    bounds=kv != "fp8" and rng.random() < 0.4)
    B = ones + (B if shape == "mixed" else 0) if ones else B
    top = 512 if dtype == "fp32" else 2048
    new = ones + (_log(rng, B - ones, top) if B > ones else 0)
    return dict(c, B=B, new=new, ones=ones, T=_log(rng, 64, 8192 if dtype == "fp32" else 16384))


def _lens(c):
    """(tokens held before, new tokens) of each sequence, from the case alone."""
    r = random.Random(c["mix"])
    B, ones, new = c["B"], c["ones"], c["new"]
    rest, more = B - ones, new - ones
    part = [math.exp(r.uniform(0.0, 1.5)) for _ in range(rest)]
    cuts = [0]
    for b in range(rest):
        cuts.append(min(more - (rest - 1 - b), max(cuts[-1] + 1, round(more * sum(part[:b + 1]) / sum(part)))))
    lq = [cuts[b + 1] - cuts[b] for b in range(rest)] + [1] * ones
    r.shuffle(lq)
    before = [c["T"] if b == 0 else int(c["T"] * r.uniform(0.1, 1.0)) for b in range(B)]
    return before, lq


# ----------------------------------------------------------------- inputs ----
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _frequencies(R, axes):
    """(R / 2) frequencies, and for several axes which of them each goes by: a quarter time, the
    rest height and width in turn."""
    n = R // 2
    f = (10000.0 ** (-torch.arange(n, dtype=torch.float64, device="cuda") / n)).float()
    if axes == 1:
        return f, None
    i = torch.arange(n, device="cuda")
    return f, torch.where(i < n // 4, 0, 1 + (i - n // 4) % 2).to(torch.int32)


def prepare(case, seed):
    c, g, dt = case, _gen(seed), _DT[case["dtype"]]
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    s = {"case": c}
    if c["kind"] == "rotary":
        N = c["N"]
        s["q"], s["k"] = _randn(g, N, Hq, D).to(dt), _randn(g, N, Hkv, D).to(dt)
        s["freq"], s["axes"] = _frequencies(c["R"], c["axes"])
        t = c["start"] + torch.arange(N, device="cuda")
        if c["axes"] == 3:  # frames of 28 rows of 36 patches
            t = torch.stack([c["start"] + t // 1008, t // 36 % 28, t % 36])
        s["positions"] = t.to(torch.int32)
        return s
    B, page = c["B"], c["page"]
    before, lq = _lens(c)
    after = [x + y for x, y in zip(before, lq)]
    s["before"], s["lq"], s["longest"] = before, lq, max(after)
    pages = [-(-n // page) for n in after]
    n_phys, width = sum(pages) + 7, max(pages) + 3
    # pages of the sequences lie in any order; what a table has behind a sequence's own is stale
    order = torch.randperm(n_phys, generator=g, device="cuda")
    table = torch.randint(0, n_phys, (B, width), generator=g, device="cuda")
    at = 0
    for b in range(B):
        table[b, :pages[b]] = order[at:at + pages[b]]
        at += pages[b]
    s["table"] = table.to(torch.int32)
    s["cu"] = _i32([sum(lq[:b]) for b in range(B + 1)])
    s["positions"], s["lengths"] = _i32(before), _i32(after)
    kv = _DT[c["kv"]]
    for name in "kv":
        x = _randn(g, n_phys, Hkv, page, D)
        if c["kv"] == "fp8":  # (both scales of a token side by side, as the framework keeps them)
            if "scales" not in s:
                s["scales"] = torch.empty(n_phys, Hkv, page, 2, device="cuda")
            scale = x.abs().amax(-1) / 448.0
            s["scales"][..., "kv".index(name)] = scale
            x = x / scale[..., None]
        s[name] = x.to(kv)
        del x
    s["q"] = _randn(g, c["new"], Hq, D).to(dt)
    if c["kind"] == "append":
        s["k_new"], s["v_new"] = _randn(g, c["new"], Hkv, D).to(dt), _randn(g, c["new"], Hkv, D).to(dt)
        s["freq"], s["axes"] = _frequencies(D, 1)
        if c["bounds"]:
            s["mins"], s["maxs"] = _bounds(s, s["positions"])
    return s


# ------------------------------------------------------- the plain forms ----
def _rotate(x, angle, neighbours, inverse):
    """x (N, H, D), its first 2 n dims turned by the angles (N, n)."""
    n = angle.shape[-1]
    cos, sin = (f(angle).to(x.dtype)[:, None] for f in (torch.cos, torch.sin))
    if inverse:
        sin = -sin
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if neighbours else (x[..., :n], x[..., n:2 * n])
    y = (a * cos - b * sin, b * cos + a * sin)
    y = torch.stack(y, -1).flatten(-2) if neighbours else torch.cat(y, -1)
    return torch.cat([y, x[..., 2 * n:]], -1)


def _angles(positions, freq, axes):
    """(N, n): 64 bits, since far positions make many turns."""
    if axes is None:
        return positions[:, None].double() * freq.double()
    return positions[axes.long()].t().double() * freq.double()


def _tokens(s):
    """Sequence and position of each new token, packed."""
    cu, n = s["cu"].long(), s["case"]["new"]
    i = torch.arange(n, device="cuda")
    b = torch.searchsorted(cu, i, right=True) - 1
    return b, s["positions"].long()[b] + i - cu[b]


def _bounds(s, lengths):
    """Least and largest key of each page of each sequence of that many tokens, (B, Hkv, pages, D)
    (what is behind a sequence's end: zeros)."""
    page = s["case"]["page"]
    keys = s["k"][s["table"].long()]  # (B, width, Hkv, page, D)
    slot = torch.arange(page, device="cuda") + page * torch.arange(keys.shape[1], device="cuda")[:, None]
    held = (slot < lengths.long()[:, None, None])[:, :, None, :, None]
    some = held.any(3)
    least = torch.where(some, torch.where(held, keys, math.inf).amin(3), 0.0)
    most = torch.where(some, torch.where(held, keys, -math.inf).amax(3), 0.0)
    return least.transpose(1, 2).contiguous(), most.transpose(1, 2).contiguous()


def _raw(x):
    """(indexing as bytes, for fp8)"""
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def _store(s, name, x, b, t):
    page = s["case"]["page"]
    phys = s["table"].long()[b, t // page]
    if s["case"]["kv"] == "fp8":
        scale = x.abs().amax(-1).clamp(min=1e-8) / 448.0
        s["scales"][phys, :, t % page, "kv".index(name)] = scale
        x = x / scale[..., None]
    _raw(s[name])[phys, :, t % page] = _raw(x.to(s[name].dtype))


def _plain_append(s):
    c = s["case"]
    b, t = _tokens(s)
    angle = _angles(t, s["freq"], None)
    q = _rotate(s["q"].float(), angle, False, False).to(s["q"].dtype)
    _store(s, "k", _rotate(s["k_new"].float(), angle, False, False), b, t)
    _store(s, "v", s["v_new"].float(), b, t)
    if c["bounds"]:
        least, most = _bounds(s, s["lengths"])
        s["mins"].copy_(least)
        s["maxs"].copy_(most)
    return q


def _cached(s, name, wide):
    """K or V of every sequence, (B, Hkv, longest, D), what is behind its end zero."""
    c = s["case"]
    used = s["table"].long()[:, :-(-s["longest"] // c["page"])]
    x = _raw(s[name])[used].view(s[name].dtype).to(wide)
    if c["kv"] == "fp8":
        x = x * s["scales"][used][..., "kv".index(name), None].to(wide)
    x = x.transpose(1, 2).flatten(2, 3)[:, :, :s["longest"]]
    held = torch.arange(s["longest"], device="cuda") < s["lengths"].long()[:, None]
    return x.masked_fill_(~held[:, None, :, None], 0.0)


def _plain_attend(s, wide=torch.float32):
    """Sequences side by side, their new tokens padded to the most of any; as many KV heads at a
    time as there is room for scores of."""
    c, cu, most = s["case"], s["cu"].long(), max(s["lq"])
    B, Hkv, D, T = c["B"], c["Hkv"], c["D"], s["longest"]
    G = c["Hq"] // Hkv
    k, v = _cached(s, "k", wide), _cached(s, "v", wide)
    n = cu[1:] - cu[:-1]
    i = torch.arange(most, device="cuda")
    q = s["q"][(cu[:-1, None] + i).clamp(max=c["new"] - 1)].to(wide)  # (B, most, Hq, D)
    q = q.transpose(1, 2).unflatten(1, (Hkv, G))
    end = (s["lengths"].long() - n)[:, None] + i + 1  # keys that a query sees, (B, most)
    hidden = (torch.arange(T, device="cuda") >= end[:, :, None])[:, None, None]
    step = max(1, min(Hkv, _ROOM // (q.element_size() * B * G * most * T)))
    out, lse = [], []
    for h in range(0, Hkv, step):
        x = torch.matmul(q[:, h:h + step].flatten(2, 3), k[:, h:h + step].transpose(-1, -2)).unflatten(2, (G, most))
        x.mul_(D ** -0.5).masked_fill_(hidden, _NINF)
        m = x.amax(-1, keepdim=True)
        x.sub_(m).exp_()
        z = x.sum(-1, keepdim=True)
        y = torch.matmul(x.flatten(2, 3), v[:, h:h + step]).unflatten(2, (G, most))
        out.append((y / z).flatten(1, 2))
        lse.append((z.log() + m).squeeze(-1).flatten(1, 2))
        del x
    live = i < n[:, None]
    out, lse = (torch.cat(x, 1).transpose(1, 2)[live] for x in (out, lse))
    return out, lse.t().contiguous()


# ---------------------------------------------------------------- one pass ----
def _appended(s, q):
    r = {"q": q, "k": s["k"], "v": s["v"]}
    if s["case"]["kv"] == "fp8":
        r["scales"] = s["scales"]
    if s["case"]["bounds"]:
        r["mins"], r["maxs"] = s["mins"], s["maxs"]
    return r


def run(s):
    c = s["case"]
    if own:
        return _own(s)
    dt = _DT[c["dtype"]]
    if c["kind"] == "rotary":
        angle = _angles(s["positions"], s["freq"], s["axes"])
        q, k = (_rotate(s[n].float(), angle, c["neighbours"], c["inverse"]).to(dt) for n in "qk")
        return {"q": q, "k": k}
    if c["kind"] == "append":
        return _appended(s, _plain_append(s))
    out, lse = _plain_attend(s)
    return {"out": out.to(dt), "lse": lse}


def _own(s):
    from linattn_amd.kernels import dense, kv_cache, rotary

    c = s["case"]
    if c["kind"] == "rotary":
        q, k = rotary.rotary(s["q"], s["k"], s["positions"], s["freq"], axes=s["axes"],
                             interleaved=c["neighbours"], inverse=c["inverse"])
        return {"q": q, "k": k}
    more = {}
    if c["kv"] == "fp8":
        more = dict(k_scale=s["scales"][..., 0], v_scale=s["scales"][..., 1])
    if c["kind"] == "append":
        if c["bounds"]:
            more = dict(page_min=s["mins"], page_max=s["maxs"], page_size=c["page"])
        q = kv_cache.rotary_kv_append(s["q"], s["k_new"], s["v_new"], s["k"], s["v"], s["table"], s["positions"],
                                      s["freq"], cu_seqlens=s["cu"], **more)
        return _appended(s, q)
    out, lse = dense.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], s["cu"],
                                     return_lse=True, **more)
    return {"out": out, "lse": lse}


# ------------------------------------------------------------------- work ----
def work(case):
    c, D, Hq, Hkv, e = case, case["D"], case["Hq"], case["Hkv"], _SIZE[case["dtype"]]
    if c["kind"] == "rotary":
        return {"bytes": c["N"] * ((Hq + Hkv) * D * e * 2 + 4 * c["axes"]), "flops": 3 * c["N"] * (Hq + Hkv) * c["R"]}
    before, lq = _lens(c)
    row = D * _SIZE[c["kv"]] + (4 if c["kv"] == "fp8" else 0)
    if c["kind"] == "append":
        bounds = 0
        if c["bounds"]:  # a page's old bounds are read where it had tokens, the new ones written
            old = sum(x % c["page"] > 0 for x in before)
            now = sum(-(-(x + n) // c["page"]) - x // c["page"] for x, n in zip(before, lq))
            bounds = 2 * (old + now) * Hkv * D * e
        return {"bytes": c["new"] * (Hq * D * e * 2 + 2 * Hkv * (D * e + row)) + bounds,
                "flops": 3 * c["new"] * (Hq + Hkv) * D}
    pairs = sum(n * x + n * (n + 1) // 2 for x, n in zip(before, lq))
    keys = sum(before) + sum(lq)
    return {"bytes": c["new"] * Hq * (2 * e * D + 4) + keys * 2 * Hkv * row, "flops": 4 * D * Hq * pairs}


# ------------------------------------------------------------------ exact ----
def _turned(x, positions, freq, axes, neighbours, inverse):
    """(N, H, D) as complex numbers times e^(i angle), in 64 bits."""
    n = freq.shape[0]
    p = positions.double()
    p = p[:, None].expand(-1, n) if axes is None else torch.stack([p[int(a)] for a in axes], 1)
    turn = torch.polar(torch.ones_like(p), p * freq.double() * (-1 if inverse else 1))[:, None]
    x, y = x.double(), x.double().clone()
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if neighbours else (slice(0, n), slice(n, 2 * n))
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_append(c, s):
    before, lq, page = s["before"], s["lq"], c["page"]
    t = torch.cat([torch.arange(x, x + n, device="cuda") for x, n in zip(before, lq)])
    q = _turned(s["q"], t, s["freq"], None, False, False)
    rows = {"k": _turned(s["k_new"], t, s["freq"], None, False, False), "v": s["v_new"].double()}
    r = {"q": q, **{n: s[n].double() for n in "kv"}}
    if c["kv"] == "fp8":
        r["scales"] = s["scales"].double()
    table, a = s["table"].tolist(), 0
    for b, (x, n) in enumerate(zip(before, lq)):
        for first in range(x - x % page, x + n, page):
            lo, hi = max(first, x), min(first + page, x + n)
            at, slots = table[b][first // page], slice(lo - first, hi - first)
            for i, name in enumerate("kv"):
                new = rows[name][a + lo - x:a + hi - x].transpose(0, 1)
                if c["kv"] == "fp8":
                    scale = new.abs().amax(-1).clamp(min=1e-8) / 448.0
                    r["scales"][at, :, slots, i] = scale
                    new = (new / scale[..., None]).to(torch.float8_e4m3fn).double()
                r[name][at, :, slots] = new
            if c["bounds"]:
                if "mins" not in r:
                    r["mins"], r["maxs"] = s["mins"].double(), s["maxs"].double()
                whole = r["k"][at, :, :hi - first]
                r["mins"][b, :, first // page], r["maxs"][b, :, first // page] = whole.amin(1), whole.amax(1)
        a += n
    return r


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "rotary":
        return {n: _turned(s[n], s["positions"], s["freq"], s["axes"], c["neighbours"], c["inverse"]) for n in "qk"}
    if c["kind"] == "append":
        return _exact_append(c, s)
    Hq, Hkv, D, page = c["Hq"], c["Hkv"], c["D"], c["page"]
    G, scale = Hq // Hkv, 1.0 / math.sqrt(D)
    out = torch.zeros(c["new"], Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.zeros(Hq, c["new"], dtype=torch.float64, device="cuda")
    a = 0
    for b, (x, n) in enumerate(zip(s["before"], s["lq"])):
        used = s["table"][b, :-(-(x + n) // page)].long()
        for h in range(Hkv):
            k, v = (_raw(s[name])[used, h].view(s[name].dtype).double() for name in "kv")
            if c["kv"] == "fp8":
                sc = s["scales"][used, h].double()
                k, v = k * sc[..., 0, None], v * sc[..., 1, None]
            k, v = k.flatten(0, 1)[:x + n], v.flatten(0, 1)[:x + n]
            for i in range(0, n, 1024):  # a piece of the queries, up to the keys the last of them sees
                m = min(n, i + 1024)
                q = s["q"][a + i:a + m, h * G:(h + 1) * G].transpose(0, 1).double()
                y = q @ k[:x + m].t() * scale
                see = torch.arange(x + m, device="cuda")[None] <= x + torch.arange(i, m, device="cuda")[:, None]
                y = torch.where(see, y, _NINF)
                z = torch.logsumexp(y, -1)
                lse[h * G:(h + 1) * G, a + i:a + m] = z
                out[a + i:a + m, h * G:(h + 1) * G] = (torch.exp(y - z[..., None]) @ v[:x + m]).transpose(0, 1)
        a += n
    return {"out": out, "lse": lse}
