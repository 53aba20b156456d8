"""Dense attention, the weights of keys and eviction in 64 bits, by plain torch on the CPU,
with how far a kernel that holds scores, weights and sums in fp32 may be off."""

from __future__ import annotations

import math

import torch

F32 = 2.0 ** -24  # half a step of fp32


def attention(q, k, v, causal=True, scale=None, half_step=F32, out_half_step=None):
    """One head of one sequence: q (Lq, D), k, v (Lk, D), the queries at the end of the keys.
    Returns out (Lq, D), lse (Lq,), and bounds on the errors of both.

    A score is a sum of D products in fp32, off by at most E = F32 (D + 4) scale sum |q k|
    (the scaling, the reference maximum's product and their difference round too); a weight
    by twice that and a few steps of exp2, relatively; it is rounded to the inputs' type
    (half_step) for its product with v; sums of n weights add n F32.  The output rounds once
    more (out_half_step, default the same)."""
    q, k, v = q.double(), k.double(), v.double()
    (Lq, D), Lk = q.shape, k.shape[0]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out, lse = torch.zeros(Lq, v.shape[1]).double(), torch.full((Lq,), -math.inf).double()
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    u_out = half_step if out_half_step is None else out_half_step
    for t in range(Lq):
        n = max(0, Lk - Lq + t + 1) if causal else Lk
        if n == 0:
            continue
        x = k[:n] @ q[t] * scale
        lse[t] = torch.logsumexp(x, 0)
        p = torch.exp(x - lse[t])
        out[t] = p @ v[:n]
        E = F32 * (D + 4) * scale * (k[:n].abs() @ q[t].abs()).max()
        w = 2 * E + 8 * F32
        spread = p @ v[:n].abs()
        tol[t] = u_out * out[t].abs() + (half_step + 2 * w + n * F32) * spread + 1e-30
        tol_lse[t] = w + (n + 8) * F32 + 2 * F32 * lse[t].abs()
    return out, lse, tol, tol_lse


def key_weights(q, k, lse, causal=True, scale=None, last=None):
    """One KV head of one sequence: q (G, Lq, D), k (Lk, D), lse (G, Lq): the weights (Lk,) of
    the last `last` queries, and a bound on their error."""
    q, k, lse = q.double(), k.double(), lse.double()
    (G, Lq, D), Lk = q.shape, k.shape[0]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    w, tol = torch.zeros(Lk).double(), torch.zeros(Lk).double()
    rows = Lq if last is None else min(last, Lq)
    for t in range(Lq - rows, Lq):
        n = max(0, Lk - Lq + t + 1) if causal else Lk
        for g in range(G):
            if n == 0 or lse[g, t] == -math.inf:
                continue
            x = k[:n] @ q[g, t] * scale
            p = torch.exp(x - lse[g, t])
            E = F32 * (D + 4) * scale * (k[:n].abs() @ q[g, t].abs())
            w[:n] += p
            tol[:n] += p * (2 * E + (8 + 4 * abs(float(lse[g, t]))) * F32)
    return w, tol + (G * rows + 8) * F32 * w + 1e-30


HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}


def close(got, want, tol, what=""):
    got, want, tol = (x.detach().cpu().double() for x in (got, want, tol))
    bad = ~((got - want).abs() <= tol) & ~(got == want)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{float(((got - want).abs() / tol)[bad].max()):.3g} times the bound, first at "
                           f"{bad.nonzero()[0].tolist()}")


def keep(weights, n, budget, recent, sink, positions=None, pos=None):
    """Indices a cache of n entries keeps, ascending."""
    positions = list(range(n)) if positions is None else [int(x) for x in positions[:n]]
    pos = n if pos is None else int(pos)

    def rank(i):
        if positions[i] < sink or positions[i] >= pos - recent:
            return (0, 0.0, i)
        w = float(weights[i])
        return (2, 0.0, i) if math.isnan(w) else (1, -w, i)

    return sorted(sorted(range(n), key=rank)[:budget])


def victim(weights, recent, sink, positions, pos):
    """The slot a full cache gives up."""
    free = [i for i, p in enumerate(positions) if sink <= int(p) < int(pos) - recent]
    if not free:
        return len(positions) - 1
    return max(free, key=lambda i: (1, 0.0, i) if math.isnan(float(weights[i])) else (0, -float(weights[i]), i))
