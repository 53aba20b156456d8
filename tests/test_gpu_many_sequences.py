"""More (sequence, KV head) pairs than a grid's second dimension has room for."""

from __future__ import annotations

import pytest
import torch

from linattn_amd.kernels.dense import dense_attention
from linattn_amd.kernels.eviction import key_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,Hkv,T", [(65536, 1, 2), (9000, 8, 3)])
def test_key_weights(dev, dtype, B, Hkv, T):
    D, G = 64, 2
    g = torch.Generator().manual_seed(0)
    q, k = (torch.randn(B, h, T, D, generator=g).to(dtype).to(dev) for h in (Hkv * G, Hkv))
    _, lse = dense_attention(q, k, k, return_lse=True)
    w = key_weights(q, k, lse)
    x = (q.double().unflatten(1, (Hkv, G)) * k.double()[:, :, None, 0, None]).sum(-1) * D ** -0.5
    rows = lse.double().unflatten(1, (Hkv, G))
    # key 0 is seen by every query, the last one by the last query
    first = torch.exp(x - rows).sum((2, 3))
    last = torch.exp((q.double().unflatten(1, (Hkv, G))[:, :, :, -1] * k.double()[:, :, None, -1]).sum(-1) * D ** -0.5
                     - rows[..., -1]).sum(2)
    # scores are sums of 64 products of up to about 5 x 5 / 8, lse rounds once; up to 6 weights
    tol = 2 * 2.0 ** -24 * (D + 4) * 40 + 16 * 2.0 ** -24
    assert ((w[:, :, 0] - first).abs() <= tol * (first + 1)).all()
    assert ((w[:, :, -1] - last).abs() <= tol * (last + 1)).all()
    assert ((w.sum(2) - G * T).abs() <= 8 * G * T * tol).all()
