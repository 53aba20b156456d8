"""Rotary positions and their append to a paged cache in 64 bits, by plain torch on the CPU, with
how far a kernel that counts turns in fp32 may be off."""

from __future__ import annotations

import torch

U = 2.0 ** -24  # half a step of fp32
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: U}
LEAST = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -149}


def turn(x, positions, freq, axes=None, interleaved=False, inverse=False):
    """x (N, H, D) turned in 64 bits and a bound on the error before the last rounding.

    Angles are products in 64 bits (off by a few 2^-53 of themselves); what is left of a
    quarter turn is rounded to 32 (pi / 4 U), its sine and cosine are series whose last steps
    round (under 3 U together), and a pair's two products and their sum round twice more."""
    x = x.double()
    n = freq.shape[0]
    p = positions.double()
    p = p[:, None].expand(-1, n) if axes is None else p[axes.long()].t()
    angle = p * freq.double()
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None] * (-1 if inverse else 1)
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., first], x[..., second]
    y, tol = x.clone(), torch.zeros_like(x)
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    off = (6 * U + 2.0 ** -50 * angle.abs()[:, None]) * (a.abs() + b.abs())
    tol[..., first], tol[..., second] = off, off
    return y, tol


def rounded(y, tol, dtype):
    """The bound after the rounding to `dtype`."""
    return tol * (1 + HALF[dtype]) + HALF[dtype] * y.abs() + LEAST[dtype]


def close(got, want, tol, what=""):
    got, want, tol = got.double().cpu(), want.double(), tol.double()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: "
                           f"{got[bad][0]} for {want[bad][0]} +- {tol[bad][0]}")


def places(positions, lq):
    """Sequence and place of each new token, packed."""
    b = torch.cat([torch.full((n,), i, dtype=torch.long) for i, n in enumerate(lq)])
    t = torch.cat([torch.arange(int(p), int(p) + n) for p, n in zip(positions, lq)])
    return b, t


def slots(table, b, t, page, n_phys):
    """(stored, page, slot) of each token."""
    inside = (t >= 0) & (t < table.shape[1] * page)
    phys = table[b, (t.clamp(min=0) // page).clamp(max=table.shape[1] - 1)].long()
    ok = inside & (phys >= 0) & (phys < n_phys)
    return ok, torch.where(ok, phys, 0), t % page


def bounds(mn, mx, keys, b, t, ok, positions, mp):
    """Quest's bounds (B, Hkv, P, D) after keys (N, Hkv, D), as stored, at places t of sequences b."""
    mn, mx = mn.clone(), mx.clone()
    for s in range(mn.shape[0]):
        for page in sorted({int(x) // mp for x in t[(b == s) & ok]}):
            if page >= mn.shape[2]:
                continue
            k = keys[(b == s) & ok & (t // mp == page)]
            lo, hi = k.amin(0), k.amax(0)
            if page * mp < int(positions[s]):
                lo, hi = torch.minimum(lo, mn[s, :, page]), torch.maximum(hi, mx[s, :, page])
            mn[s, :, page], mx[s, :, page] = lo, hi
    return mn, mx
