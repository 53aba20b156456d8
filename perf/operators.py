"""Dense attention of prompts, the attention weight each cached key gathers, eviction of
cached keys by it, and the decode step over the evicted cache: what these operators cost.

``listed()`` names the calls, ``draw(rng)`` makes another of the same ranges, ``prepare``
builds what a program has in hand, ``run`` is one pass: by plain torch operations, or, where
``own`` is set, through the framework's entry points.  ``work`` counts the bytes and operations
a pass cannot do without, ``exact`` is the result in 64 bits.
"""

import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
_NINF = float("-inf")
_ROOM = 16 << 30  # bytes of scores the plain form holds at a time


# ------------------------------------------------------------------ cases ----
def listed():
    return [
        # a few short prompts packed together, fp32 at the harness's head size: the smallest call
        dict(name="attn_short", kind="packed", B=4, total=202, mix=3, Hq=8, Hkv=8, D=64, dtype="fp32"),
        # the prefill batch of a server: twelve prompts of very different lengths, packed
        dict(name="attn_packed", kind="packed", B=12, total=14567, mix=1, Hq=32, Hkv=8, D=128,
             dtype="bf16"),
        # chunked prefill: the next 512 tokens of four sequences against caches of up to 8K
        dict(name="attn_chunk", kind="dense", B=4, Tq=512, T=8192, mix=2, Hq=32, Hkv=8, D=128,
             dtype="fp16"),
        # a dense layer's decode step: one token of each sequence over its whole cache
        dict(name="attn_token", kind="dense", B=16, Tq=1, T=12345, mix=4, Hq=32, Hkv=8, D=128,
             dtype="bf16"),
        # one 32K prompt: the largest call
        dict(name="attn_32k", kind="packed", B=1, total=32768, mix=0, Hq=32, Hkv=8, D=128,
             dtype="bf16"),
        # the weights of a packed prefill batch, every query counted
        dict(name="weights_packed", kind="weights", B=12, total=14567, last=0, mix=1, Hq=32, Hkv=8,
             D=128, dtype="bf16"),
        # the weights by the last 64 queries of two long prompts only
        dict(name="weights_last", kind="weights", B=2, total=50001, last=64, mix=5, Hq=32, Hkv=8,
             D=128, dtype="fp16"),
        # a short prompt's cache cut to 256 entries, fp32
        dict(name="evict_short", kind="evict", B=2, total=1400, budget=256, mix=6, Hkv=8, D=64,
             dtype="fp32"),
        # long prompts' caches cut to 4096 entries each
        dict(name="evict_long", kind="evict", B=4, total=100003, budget=4096, mix=7, Hkv=8, D=128,
             dtype="bf16"),
        # one user's token over a small evicted cache, fp32: launches and latency
        dict(name="step_one", kind="step", B=1, C=257, fill=1.0, Hq=8, Hkv=8, D=64, dtype="fp32"),
        # a token of each sequence of a full batch, caches at their budget
        dict(name="step_batch", kind="step", B=64, C=2049, fill=1.0, Hq=32, Hkv=8, D=128,
             dtype="bf16"),
        # few sequences with large caches, some not yet full
        dict(name="step_large", kind="step", B=4, C=16385, fill=0.5, Hq=32, Hkv=8, D=128,
             dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["packed", "packed", "dense", "dense", "weights", "weights", "evict", "step", "step"])
    Hq, Hkv = rng.choice([(32, 8), (16, 8), (16, 4), (8, 8), (8, 1), (12, 4), (5, 1)])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    D = rng.choice([64, 128])
    mix = rng.randint(0, 999)
    c = dict(kind=kind, mix=mix, Hq=Hq, Hkv=Hkv, D=D, dtype=dtype)
    top = 8192 if dtype == "fp32" else 32768
    if kind == "packed":
        total = _log(rng, 100, top)
        return dict(c, B=rng.randint(1, min(16, total)), total=total)
    if kind == "dense":
        B = _log(rng, 1, 16)
        return dict(c, B=B, Tq=_log(rng, 1, 1024 // B), T=_log(rng, 1024, 16384))
    if kind == "weights":
        total = _log(rng, 100, top)
        return dict(c, B=rng.randint(1, min(16, total)), total=total, last=rng.choice([0, 32, 64, 129]))
    del c["Hq"]
    if kind == "evict":
        total = _log(rng, 200, 131072)
        return dict(c, B=rng.randint(1, 8), total=total, budget=_log(rng, 64, 8192))
    del c["mix"]
    return dict(c, Hq=Hq, B=_log(rng, 1, 64), C=_log(rng, 64, 8192) + 1, fill=rng.choice([0.5, 0.9, 1.0]))


def _lens(c):
    """Lengths of the sequences, one to `total` tokens of it, from the case alone."""
    if c["kind"] == "dense":
        r = random.Random(c["mix"])
        return [max(c["Tq"], int(c["T"] * (1.0 if b == 0 else r.uniform(0.3, 1.0)))) for b in range(c["B"])]
    if c["kind"] == "step":  # entries held before the step; the first cache is the fullest
        r = random.Random(c["C"])
        return [c["C"] if b == 0 or c["fill"] == 1.0 else int(c["C"] * r.uniform(c["fill"], 1.2)) for b in range(c["B"])]
    r = random.Random(c["mix"])
    part = [math.exp(r.uniform(0.0, 4.0)) for _ in range(c["B"])]
    cuts = [0]
    for b in range(c["B"]):
        cuts.append(min(c["total"] - (c["B"] - 1 - b),
                        max(cuts[-1] + 1, round(c["total"] * sum(part[:b + 1]) / sum(part)))))
    return [cuts[b + 1] - cuts[b] for b in range(c["B"])]


def _protected(c):
    """(recent, sink): half of a cache is the newest tokens, four the first."""
    n = c["budget"] if c["kind"] == "evict" else c["C"] - 1
    return n // 2, 4


# ----------------------------------------------------------------- inputs ----
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _tokens(g, N, Hq, Hkv, D, dt):
    """q (N, Hq, D), k, v (N, Hkv, D): stretches of 128 tokens share one of 24 topics, and one
    key in a hundred is an outlier, as attention sinks and rare tokens are."""
    topics = _randn(g, 24, Hkv, D)
    pick = torch.randint(0, 24, (-(-N // 128),), generator=g, device="cuda")
    base = topics[pick].repeat_interleave(128, 0)[:N]
    q = (0.7 * base).repeat_interleave(Hq // Hkv, 1) + 0.7 * _randn(g, N, Hq, D)
    k = 0.7 * base + 0.7 * _randn(g, N, Hkv, D)
    k *= 1.0 + 2.0 * (torch.rand(N, Hkv, 1, generator=g, device="cuda") < 0.01)
    return q.to(dt), k.to(dt), _randn(g, N, Hkv, D).to(dt)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _heavy(g, *shape):
    """Gathered attention weights: most keys little, some very much."""
    return torch.exp(2.0 * _randn(g, *shape) - 2.0)


def prepare(case, seed):
    c, g, dt, D, Hkv, B = case, _gen(seed), _DT[case["dtype"]], case["D"], case["Hkv"], case["B"]
    lens = _lens(c)
    s = {"case": c, "lens": lens, "longest": max(lens)}
    if c["kind"] in ("packed", "weights", "evict"):
        s["cu"] = _i32([sum(lens[:b]) for b in range(B + 1)])
    if c["kind"] in ("packed", "weights"):
        s["q"], s["k"], s["v"] = _tokens(g, c["total"], c["Hq"], Hkv, D, dt)
        if c["kind"] == "weights":  # (the attention's own, which ran before)
            s["lse"] = _plain_packed(s, want="lse")
    elif c["kind"] == "dense":
        s["lengths"] = _i32(lens)
        x = [_tokens(g, c["T"], c["Hq"], Hkv, D, dt) for _ in range(B)]
        s["k"], s["v"] = (torch.stack([y[i].transpose(0, 1) for y in x]) for i in (1, 2))
        s["q"] = torch.stack([y[0][n - c["Tq"]:n].transpose(0, 1) for y, n in zip(x, lens)])
    elif c["kind"] == "evict":
        s["k"], s["v"] = (_randn(g, c["total"], Hkv, D).to(dt) for _ in range(2))
        s["w"] = _heavy(g, Hkv, c["total"])
    else:
        C = c["C"]
        s["q"] = _randn(g, B, c["Hq"], 1, D).to(dt)
        s["k_new"], s["v_new"] = (_randn(g, B, Hkv, 1, D).to(dt) for _ in range(2))
        s["k"], s["v"] = (_randn(g, B, Hkv, C, D).to(dt) for _ in range(2))
        s["lengths"] = _i32([min(n, C) for n in lens])
        held = torch.arange(C, device="cuda") < s["lengths"].view(B, 1, 1)
        s["w"] = torch.where(held, _heavy(g, B, Hkv, C), 0.0)
        # kept entries are old, the rest new; a decoding cache is in no order
        pos = (torch.rand(B, Hkv, C, generator=g, device="cuda") * 3 * C).to(torch.int32)
        s["positions"] = torch.where(held, pos, -1)
        s["pos"] = torch.full((B,), 3 * C, dtype=torch.int32, device="cuda")
    return s


# ------------------------------------------------------- the plain forms ----
def _pad(x, cu, longest):
    """Packed rows (N, ...) as (B, longest, ...), with rows past a sequence's end repeated."""
    at = cu[:-1, None].long() + torch.arange(longest, device=x.device)
    return x[at.clamp(max=x.shape[0] - 1)]


def _unpad(x, cu, longest):
    """The inverse: (B, longest, ...) to (N, ...)."""
    lens = (cu[1:] - cu[:-1]).long()
    return x[torch.arange(longest, device=x.device) < lens[:, None]]


def _scores(q, k, lk, lq, first=0):
    """Scaled scores (B, h, G, Tq, Tk) of q (B, h, G, Tq, D) and k (B, h, Tk, D); what a row may
    not see (past its own position, or past the end of keys) is -inf.  Rows end with the keys:
    the sequence's last query (number lq - 1, rows counted from `first`) sees all lk."""
    x = torch.matmul(q.flatten(2, 3), k.transpose(-1, -2)).unflatten(2, q.shape[2:4])
    x *= q.shape[-1] ** -0.5
    t = first + torch.arange(q.shape[3], device=q.device)
    end = (lk - lq)[:, None] + t + 1  # (B, Tq)
    hidden = torch.arange(k.shape[2], device=q.device) >= end[:, :, None]
    return x.masked_fill_(hidden[:, None, None], _NINF)


def _attend(q, k, v, lk, lq, want="both"):
    """(out, lse) of q (B, Hq, Tq, D) over k, v (B, Hkv, Tk, D), in the inputs' (wide) type;
    as many KV heads at a time as there is room for scores of."""
    B, Hq, Tq, D = q.shape
    Hkv, Tk = k.shape[1:3]
    q = q.unflatten(1, (Hkv, Hq // Hkv))
    step = max(1, min(Hkv, _ROOM // (q.element_size() * B * (Hq // Hkv) * Tq * Tk)))
    out, lse = [], []
    for h in range(0, Hkv, step):
        x = _scores(q[:, h:h + step], k[:, h:h + step], lk, lq)
        m = x.amax(-1, keepdim=True)
        m = torch.where(m == _NINF, 0.0, m)
        x.sub_(m).exp_()
        z = x.sum(-1, keepdim=True)
        lse.append((z.log() + m).squeeze(-1).flatten(1, 2))
        if want == "both":
            y = torch.matmul(x.flatten(2, 3), v[:, h:h + step]).unflatten(2, x.shape[2:4])
            out.append((y / torch.where(z > 0, z, 1.0)).flatten(1, 2))
        del x
    return (torch.cat(out, 1) if out else None), torch.cat(lse, 1)


def _plain_packed(s, want="both", wide=torch.float32):
    q, k, v = (_pad(s[n], s["cu"], s["longest"]).transpose(1, 2).to(wide) for n in "qkv")
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    out, lse = _attend(q, k, v, n, n, want)
    lse = _unpad(lse.transpose(1, 2), s["cu"], s["longest"]).t().contiguous()
    if want == "lse":
        return lse
    return {"out": _unpad(out.transpose(1, 2), s["cu"], s["longest"]), "lse": lse}


def _plain_weights(s, wide=torch.float32):
    c, cu, longest = s["case"], s["cu"], s["longest"]
    n = (cu[1:] - cu[:-1]).long()
    rows = min(longest, c["last"] or longest)  # the last queries, as rows that end with the keys
    t = n[:, None] - rows + torch.arange(rows, device="cuda")
    at = (cu[:-1, None].long() + t).clamp(min=0)
    q = s["q"][at].transpose(1, 2).to(wide).unflatten(1, (c["Hkv"], -1))
    lse = s["lse"].t()[at].transpose(1, 2).to(wide)
    lse = torch.where(t[:, None] >= 0, lse, float("inf")).unflatten(1, (c["Hkv"], -1))
    k = _pad(s["k"], cu, longest).transpose(1, 2).to(wide)
    step = max(1, min(c["Hkv"], _ROOM // (q.element_size() * c["B"] * q.shape[2] * rows * longest)))
    w = []
    for h in range(0, c["Hkv"], step):
        x = _scores(q[:, h:h + step], k[:, h:h + step], n, torch.full_like(n, rows))
        w.append(x.sub_(lse[:, h:h + step, ..., None]).exp_().sum((2, 3)))
        del x
    return {"weights": _unpad(torch.cat(w, 1).transpose(1, 2), cu, longest).t().contiguous()}


def _plain_evict(s):
    c, cu, longest, keep = s["case"], s["cu"], s["longest"], s["case"]["budget"]
    recent, sink = _protected(c)
    n = (cu[1:] - cu[:-1]).long()[:, None, None]
    i = torch.arange(longest, device="cuda")
    w = _pad(s["w"].t(), cu, longest).transpose(1, 2)  # (B, Hkv, longest)
    # the first and the newest tokens above all, what is past the end below all
    key = torch.where((i < sink) | (i >= n - recent), float("inf"), w)
    key = torch.where(i < n, key, _NINF)
    pick = key.sort(dim=-1, descending=True, stable=True).indices[..., :keep]  # ties: lowest first
    pick = torch.where(pick < n, pick, longest).sort(-1).values
    pick = torch.nn.functional.pad(pick, (0, keep + 1 - pick.shape[-1]), value=longest)
    there = pick < longest
    at = (cu[:-1].long()[:, None, None] + pick).clamp(max=c["total"] - 1)
    h = torch.arange(c["Hkv"], device="cuda")[None, :, None]
    return {"k": torch.where(there[..., None], s["k"][at, h], 0.0),
            "v": torch.where(there[..., None], s["v"][at, h], 0.0),
            "weights": torch.where(there, s["w"][h, at], 0.0),
            "positions": torch.where(there, pick, -1).to(torch.int32),
            "lengths": n.flatten().clamp(max=keep).to(torch.int32)}


def _plain_step(s, wide=torch.float32):
    c, C, B = s["case"], s["case"]["C"], s["case"]["B"]
    recent, sink = _protected(c)
    k, v, w, positions = s["k"], s["v"], s["w"], s["positions"]
    n = s["lengths"].long()[:, None, None]
    # the lightest entry that is neither among the newest nor the first; ties: the last slot
    safe = (positions >= s["pos"][:, None, None] - recent) | (positions < sink)
    lightest = (C - 1) - torch.where(safe, float("inf"), w).flip(-1).argmin(-1, keepdim=True)
    slot = torch.where(n < C, n, lightest)  # (B, Hkv, 1)
    k.scatter_(2, slot[..., None].expand(-1, -1, -1, c["D"]), s["k_new"])
    v.scatter_(2, slot[..., None].expand(-1, -1, -1, c["D"]), s["v_new"])
    w.scatter_(2, slot, 0.0)
    positions.scatter_(2, slot, s["pos"][:, None, None].expand_as(slot).contiguous())
    q = s["q"].to(wide).unflatten(1, (c["Hkv"], -1))
    n = (s["lengths"].long() + 1).clamp(max=C)
    x = _scores(q, k.to(wide), n, torch.ones_like(n))
    p = torch.softmax(x, -1)
    out = torch.matmul(p.flatten(2, 3), v.to(wide)).unflatten(2, p.shape[2:4])
    w += p.sum((2, 3))
    return {"out": out.flatten(1, 2), "k": k, "v": v, "weights": w, "positions": positions}


# ---------------------------------------------------------------- one pass ----
def run(s):
    c, kind = s["case"], s["case"]["kind"]
    if own:
        return _own(s)
    dt = _DT[c["dtype"]]
    if kind == "packed":
        r = _plain_packed(s)
        return {"out": r["out"].to(dt), "lse": r["lse"]}
    if kind == "dense":
        n = s["lengths"].long()
        out, lse = _attend(s["q"].float(), s["k"].float(), s["v"].float(), n, torch.full_like(n, c["Tq"]))
        return {"out": out.to(dt), "lse": lse}
    if kind == "weights":
        return _plain_weights(s)
    if kind == "evict":
        return _plain_evict(s)
    r = _plain_step(s)
    return dict(r, out=r["out"].to(dt))


def _own(s):
    from linattn_amd.kernels import dense, eviction

    c, kind = s["case"], s["case"]["kind"]
    if kind == "packed":
        out, lse = dense.packed_attention(s["q"], s["k"], s["v"], s["cu"], return_lse=True)
        return {"out": out, "lse": lse}
    if kind == "dense":
        out, lse = dense.dense_attention(s["q"], s["k"], s["v"], lengths=s["lengths"], return_lse=True)
        return {"out": out, "lse": lse}
    if kind == "weights":
        return {"weights": eviction.packed_key_weights(s["q"], s["k"], s["lse"], s["cu"],
                                                       last=c["last"] or None)}
    recent, sink = _protected(c)
    if kind == "evict":
        k, v, w, positions, lengths = eviction.packed_evict_kv(
            s["k"], s["v"], s["w"], s["cu"], budget=c["budget"], recent=recent, sink=sink,
            capacity=c["budget"] + 1)
        return {"k": k, "v": v, "weights": w, "positions": positions, "lengths": lengths}
    out = eviction.evict_decode_step(s["q"], s["k_new"], s["v_new"], s["k"], s["v"], s["w"],
                                     s["positions"], s["lengths"], s["pos"], recent=recent, sink=sink)
    return {"out": out, "k": s["k"], "v": s["v"], "weights": s["w"], "positions": s["positions"]}


# ------------------------------------------------------------------- work ----
def work(case):
    c, D, Hkv, B, e = case, case["D"], case["Hkv"], case["B"], _SIZE[case["dtype"]]
    Hq, lens = c.get("Hq", 0), _lens(case)
    if c["kind"] == "packed":
        pairs = sum(n * (n + 1) // 2 for n in lens)
        return {"bytes": c["total"] * (2 * e * D * (Hq + Hkv) + 4 * Hq), "flops": 4 * D * Hq * pairs}
    if c["kind"] == "dense":
        Tq = c["Tq"]
        pairs = sum(Tq * (n - Tq) + Tq * (Tq + 1) // 2 for n in lens)
        return {"bytes": 2 * e * D * (Hq * B * Tq + Hkv * sum(lens)) + 4 * Hq * B * Tq,
                "flops": 4 * D * Hq * pairs}
    if c["kind"] == "weights":
        rows = [min(n, c["last"] or n) for n in lens]
        pairs = sum(r * (n - r) + r * (r + 1) // 2 for n, r in zip(lens, rows))
        return {"bytes": c["total"] * Hkv * (e * D + 4) + sum(rows) * Hq * (e * D + 4),
                "flops": 2 * D * Hq * pairs}
    if c["kind"] == "evict":
        kept = sum(min(n, c["budget"]) for n in lens)
        slots = B * (c["budget"] + 1)
        return {"bytes": Hkv * (4 * c["total"] + kept * 2 * e * D + slots * (2 * e * D + 8)),
                "flops": Hkv * c["total"]}
    held = sum(min(n + 1, c["C"]) for n in lens)
    return {"bytes": Hkv * held * (2 * e * D + 12) + B * (2 * Hq + 4 * Hkv) * D * e,
            "flops": 4 * D * Hq * held}


# ------------------------------------------------------------------ exact ----
def _one(q, k, v, first, scale):
    """One KV head of one sequence in 64 bits: out and lse of q (G, Tq, D), whose row t sees keys
    0 .. first + t of k, v (Tk, D); rows in pieces that fit."""
    G, Tq, D = q.shape
    out = torch.zeros(G, Tq, D, dtype=torch.float64, device=q.device)
    lse = torch.full((G, Tq), _NINF, dtype=torch.float64, device=q.device)
    rows = max(1, (1 << 28) // (G * max(1, k.shape[0])))
    for a in range(0, Tq, rows):
        b = min(Tq, a + rows)
        n = min(k.shape[0], first + b)
        if n <= 0:
            continue
        x = q[:, a:b].double() @ k[:n].double().t() * scale
        see = torch.arange(n, device=q.device)[None] <= first + torch.arange(a, b, device=q.device)[:, None]
        x = torch.where(see, x, _NINF)
        lse[:, a:b] = torch.logsumexp(x, -1)
        out[:, a:b] = torch.exp(x - lse[:, a:b, None]).nan_to_num() @ v[:n].double()
    return out, lse


def _exact_evict(c, s):
    B, Hkv, D, keep = c["B"], c["Hkv"], c["D"], c["budget"]
    recent, sink = _protected(c)
    k, v = (torch.zeros(B, Hkv, keep + 1, D, dtype=torch.float64, device="cuda") for _ in range(2))
    w = torch.zeros(B, Hkv, keep + 1, dtype=torch.float64, device="cuda")
    positions = torch.full((B, Hkv, keep + 1), -1, dtype=torch.int32, device="cuda")
    a = 0
    for b, n in enumerate(s["lens"]):
        weights = s["w"][:, a:a + n].double().cpu().tolist()
        for h in range(Hkv):
            safe = set(range(min(sink, n))) | set(range(max(0, n - recent), n))
            others = sorted((i for i in range(n) if i not in safe), key=lambda i: (-weights[h][i], i))
            kept = sorted(sorted(safe) + others[:max(0, keep - len(safe))])
            at, m = torch.tensor(kept, device="cuda"), len(kept)
            k[b, h, :m], v[b, h, :m] = s["k"][a + at, h].double(), s["v"][a + at, h].double()
            w[b, h, :m], positions[b, h, :m] = s["w"][h, a + at].double(), at.to(torch.int32)
        a += n
    return {"k": k, "v": v, "weights": w, "positions": positions,
            "lengths": torch.tensor([min(n, keep) for n in s["lens"]], dtype=torch.int32, device="cuda")}


def exact(case, seed):
    c, s = case, prepare(case, seed)
    Hkv, D = c["Hkv"], c["D"]
    scale = 1.0 / math.sqrt(D)
    if c["kind"] == "evict":
        return _exact_evict(c, s)
    G = c["Hq"] // Hkv
    if c["kind"] in ("packed", "weights"):
        out = torch.zeros(c["total"], c["Hq"], D, dtype=torch.float64, device="cuda")
        lse = torch.zeros(c["Hq"], c["total"], dtype=torch.float64, device="cuda")
        weights = torch.zeros(Hkv, c["total"], dtype=torch.float64, device="cuda")
        a = 0
        for n in s["lens"]:
            for h in range(Hkv):
                q = s["q"][a:a + n, h * G:(h + 1) * G].transpose(0, 1)
                k, v = s["k"][a:a + n, h], s["v"][a:a + n, h]
                if c["kind"] == "packed":
                    out[a:a + n, h * G:(h + 1) * G], lse[h * G:(h + 1) * G, a:a + n] = (
                        x.transpose(0, 1) if x.dim() == 3 else x for x in _one(q, k, v, 0, scale))
                    continue
                t0 = max(0, n - (c["last"] or n))
                for t in range(t0, n, 2048):
                    e = min(n, t + 2048)
                    x = torch.exp(q[:, t:e].double() @ k[:e].double().t() * scale
                                  - s["lse"][h * G:(h + 1) * G, a + t:a + e, None].double())
                    see = torch.arange(e, device="cuda")[None] <= torch.arange(t, e, device="cuda")[:, None]
                    weights[h, a:a + e] += torch.where(see, x, 0.0).sum((0, 1))
            a += n
        return {"out": out, "lse": lse} if c["kind"] == "packed" else {"weights": weights}
    if c["kind"] == "dense":
        B, Tq = c["B"], c["Tq"]
        out = torch.zeros(B, c["Hq"], Tq, D, dtype=torch.float64, device="cuda")
        lse = torch.zeros(B, c["Hq"], Tq, dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["lens"]):
            for h in range(Hkv):
                g = slice(h * G, (h + 1) * G)
                out[b, g], lse[b, g] = _one(s["q"][b, g], s["k"][b, h, :n], s["v"][b, h, :n], n - Tq, scale)
        return {"out": out, "lse": lse}
    recent, sink = _protected(c)
    out = torch.zeros(c["B"], c["Hq"], 1, D, dtype=torch.float64, device="cuda")
    weights, positions = s["w"].double(), s["positions"].clone()
    caches = s["k"].double(), s["v"].double()
    for b in range(c["B"]):
        n, pos = int(s["lengths"][b]), int(s["pos"][b])
        for h in range(Hkv):
            slot = n
            if n == c["C"]:
                p = s["positions"][b, h]
                free = torch.nonzero((p < pos - recent) & (p >= sink)).flatten()
                w = s["w"][b, h, free]
                slot = int(free[torch.nonzero(w == w.min()).flatten()[-1]])
            k, v = (x[b, h] for x in caches)
            k[slot], v[slot] = s["k_new"][b, h, 0].double(), s["v_new"][b, h, 0].double()
            positions[b, h, slot] = pos
            m, g = min(n + 1, c["C"]), slice(h * G, (h + 1) * G)
            p = torch.softmax(s["q"][b, g, 0].double() @ k[:m].t() * scale, -1)
            out[b, g, 0] = p @ v[:m]
            weights[b, h, slot] = 0.0
            weights[b, h, :m] += p.sum(0)
    return {"out": out, "k": caches[0], "v": caches[1], "weights": weights, "positions": positions}
