"""fp32 scores of few rows: few roundings in a dot product, and none of a score before the
row's maximum is taken off."""

from __future__ import annotations

import pytest
import torch

from linattn_amd.kernels.dense import dense_attention
from linattn_amd.kernels.eviction import evict_decode_step

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24


@pytest.mark.parametrize("D", [64, 128])
def test_small_products_behind_a_large_one(dev, D):
    """One key's score is 1 and a product just below half a step of 1 for every fourth dim:
    added to the 1 one by one they would all be lost."""
    q, k = torch.ones(1, 1, 1, D), torch.zeros(1, 1, 1, D)
    small = 0.98 * F32
    for s in range(D // 16):
        k[..., 16 * s:16 * s + 4] = small
    k[..., 0] = 1.0
    _, lse = dense_attention(q.to(dev), k.to(dev), k.to(dev), scale=1.0, return_lse=True)
    want = float(k.double().sum())
    # four sums of D / 16 products each round to half a step of 1 (which is F32); joining them,
    # the scale and its way back 4 more
    assert abs(float(lse) - want) <= (D // 16 + 4) * F32


def _far(n, D=64):
    """Scores 1000 + i / 64, exact in fp32, and the weights they give."""
    q, k, v = torch.zeros(1, 1, 1, D), torch.zeros(1, 1, n, D), torch.zeros(1, 1, n, D)
    q[..., 0] = 1.0
    k[0, 0, :, 0] = 1000.0 + torch.arange(n) / 64.0
    v[0, 0, torch.arange(n), torch.arange(n)] = 1.0
    want = torch.softmax(k[0, 0, :, 0].double(), 0)
    # the difference to the reference is below 1.5 and rounds once, exp2 is off by two steps at
    # most, sums of n weights round n times, the quotient and the output once each
    return q, k, v, want, want * (n + 12) * F32


@pytest.mark.parametrize("n", [17, 64])
def test_scores_far_from_zero(dev, n):
    q, k, v, want, tol = _far(n)
    out = dense_attention(q.to(dev), k.to(dev), v.to(dev), scale=1.0)
    assert ((out[0, 0, 0, :n].double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("C", [64, 700])
def test_decode_step_far_from_zero(dev, C):
    n = 64
    q, k, v, want, tol = _far(n)
    cache = lambda x: torch.cat([x, torch.zeros(1, 1, C - n, 64)], 2).to(dev)
    w = torch.zeros(1, 1, C, device=dev)
    i32 = lambda x: torch.tensor([x], dtype=torch.int32, device=dev)
    out = evict_decode_step(q.to(dev), k[:, :, n - 1:].to(dev), v[:, :, n - 1:].to(dev), cache(k), cache(v), w,
                            torch.zeros(1, 1, C, dtype=torch.int32, device=dev), i32(n - 1), i32(n - 1), recent=8, scale=1.0)
    assert ((out[0, 0, 0].double().cpu() - want).abs() <= tol).all()
    assert ((w[0, 0, :n].double().cpu() - want).abs() <= tol).all() and (w[0, 0, n:] == 0).all()


def _rising(n, D=64):
    """Scores from 1000 to 1032, exact in fp32: the reference maximum is raised again and again.
    Output dim i is the weight of the i-th of D stretches of keys."""
    q, k, v = torch.zeros(1, 1, 1, D), torch.zeros(1, 1, n, D), torch.zeros(1, 1, n, D)
    q[..., 0] = 1.0
    x = 1000.0 + 32.0 * torch.arange(n) / n
    k[0, 0, :, 0] = x
    v[0, 0, torch.arange(n), torch.arange(n) // (n // D)] = 1.0
    want = torch.softmax(x.double(), 0).view(D, -1).sum(1)
    # a weight rounds 4 times (its argument, exp2 and the product); the reference is raised at
    # most 8 times, each for 4 roundings of what was before; a lane adds at most 32 parts of 8
    # weights, which 8 more additions join; the quotient
    return q, k, v, want, want * (4 + 8 * 4 + 32 + 8 + 8 + 2) * F32


@pytest.mark.parametrize("Tq", [1, 40])
def test_rising_scores(dev, Tq):
    q, k, v, want, tol = _rising(1024)
    out = dense_attention(q.expand(1, 1, Tq, 64).to(dev), k.to(dev), v.to(dev), causal=False, scale=1.0)
    assert ((out[0, 0].double().cpu() - want).abs() <= tol).all()


def test_decode_step_with_rising_scores(dev):
    q, k, v, want, tol = _rising(1024)
    i32 = lambda x: torch.tensor([x], dtype=torch.int32, device=dev)
    out = evict_decode_step(q.to(dev), k[:, :, 1023:].to(dev), v[:, :, 1023:].to(dev), k.to(dev), v.to(dev),
                            torch.zeros(1, 1, 1024, device=dev), torch.zeros(1, 1, 1024, dtype=torch.int32, device=dev),
                            i32(1023), i32(1023), recent=8, scale=1.0)
    assert ((out[0, 0, 0].double().cpu() - want).abs() <= tol).all()
