"""``key_weights``: a query whose lse is -inf adds nothing, whatever its row of q holds."""

from __future__ import annotations

import math

import pytest
import torch

from dense_reference import attention, close, key_weights as reference
from linattn_amd.kernels.eviction import key_weights, packed_key_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G,T,causal", [(1, 300, True), (4, 300, True), (2, 520, False), (3, 65, True)])
def test_rows_marked_absent(dev, dtype, D, G, T, causal):
    g = torch.Generator().manual_seed(0)
    q, k = (torch.randn(1, h, T, D, generator=g).to(dtype) for h in (G, 1))
    lse = torch.stack([attention(q[0, h], k[0, 0], k[0, 0], causal)[1] for h in range(G)])[None].float()
    for h, t in ((0, T - 1), (0, T // 2), (G - 1, 10), (0, 0)):
        lse[0, h, t] = -math.inf
    want, tol = reference(q[0], k[0, 0], lse[0], causal)
    q[0, 0, T - 1], q[0, 0, T // 2, 3], q[0, G - 1, 10], q[0, 0, 0] = math.nan, math.inf, -math.inf, math.nan
    qd, kd, ld = q.to(dev), k.to(dev), lse.to(dev)
    close(key_weights(qd, kd, ld, causal=causal)[0, 0], want, tol)
    cu = torch.tensor([0, T], dtype=torch.int32, device=dev)
    got = packed_key_weights(qd[0].transpose(0, 1), kd[0].transpose(0, 1), ld[0], cu, causal=causal)
    close(got[0], want, tol)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("G,T", [(1, 300), (4, 130)])
def test_infinite_sums(dev, dtype, G, T):
    """lse +inf: finite scores weigh nothing, an infinite one inf - inf, which is not a number."""
    g = torch.Generator().manual_seed(0)
    q, k = (torch.randn(1, h, T, 64, generator=g).to(dtype) for h in (G, 1))
    lse = torch.stack([attention(q[0, h], k[0, 0], k[0, 0])[1] for h in range(G)])[None].float()
    rows = [T - 1, T // 2 + 3]
    for t in rows:
        lse[0, 0, t] = -math.inf
    want, tol = reference(q[0], k[0, 0], lse[0])
    for t in rows:
        lse[0, 0, t] = math.inf
    close(key_weights(q.to(dev), k.to(dev), lse.to(dev))[0, 0], want, tol)
    for t in rows:
        q[0, 0, t, 3] = 1.0
    k[0, 0, 20, 3] = k[0, 0, T // 2, 3] = math.inf
    w = key_weights(q.to(dev), k.to(dev), lse.to(dev))[0, 0].cpu()
    assert w[20].isnan() and w[T // 2].isnan()
