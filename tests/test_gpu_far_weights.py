"""Weights far below a row's largest: many of them together are a part of the result that the
largest key, whose value is 0, does not hide."""

from __future__ import annotations

import pytest
import torch

from dense_reference import HALF_STEP, attention, close
from linattn_amd.kernels.dense import dense_attention, packed_attention
from linattn_amd.kernels.eviction import evict_decode_step

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _inputs(dtype, D, Tq, n, gap, first):
    """Scores `gap` (nats, scale 1) for the key `first`, 0 for the others; values 0 and about 1."""
    q, k = torch.zeros(Tq, D), torch.zeros(n, D)
    q[:, 0] = 1.0
    k[first, 0] = gap
    v = 1.0 + torch.rand(n, D, generator=torch.Generator().manual_seed(1))
    v[first] = 0.0
    return q.to(dtype), k.to(dtype), v.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gap", [10.0, 13.0, 16.0, 17.5, 20.0])
@pytest.mark.parametrize("Tq,n,first", [(1, 4096, 0), (1, 300, 299), (40, 4096, 0), (40, 200, 100), (300, 2000, 1), (300, 1000, 650)])
def test_attention(dev, dtype, gap, Tq, n, first):
    q, k, v = _inputs(dtype, 64, Tq, n, gap, first)
    out, lse = dense_attention(*(x[None, None].to(dev) for x in (q, k, v)), scale=1.0, out_dtype=torch.float32, return_lse=True)
    o, ls, tol, tol_l = attention(q, k, v, True, 1.0, HALF_STEP[dtype], HALF_STEP[torch.float32])
    close(out[0, 0], o, tol, "out")
    close(lse[0, 0], ls, tol_l, "lse")


@pytest.mark.parametrize("dtype", TYPES)
def test_packed_attention(dev, dtype):
    """Every row of a prompt, the largest key in the middle."""
    q, k, v = _inputs(dtype, 128, 700, 700, 18.0, 300)
    cu = torch.tensor([0, 700], dtype=torch.int32, device=dev)
    out = packed_attention(*(x[:, None].to(dev) for x in (q, k, v)), cu, scale=1.0, out_dtype=torch.float32)
    o, _, tol, _ = attention(q, k, v, True, 1.0, HALF_STEP[dtype], HALF_STEP[torch.float32])
    close(out[:, 0], o, tol)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gap", [10.0, 16.0, 20.0])
@pytest.mark.parametrize("n", [300, 2049])
def test_decode_step(dev, dtype, gap, n):
    q, k, v = _inputs(dtype, 64, 1, n, gap, 5)
    kd, vd = k[None, None].to(dev), v[None, None].to(dev)
    w = torch.zeros(1, 1, n, device=dev)
    positions = torch.arange(n, dtype=torch.int32, device=dev)[None, None].contiguous()
    i32 = lambda x: torch.tensor([x], dtype=torch.int32, device=dev)
    new = (k[n - 1:], v[n - 1:])
    out = evict_decode_step(q[None, None].to(dev), *(x[None, None].to(dev) for x in new), kd, vd, w, positions, i32(n - 1),
                            i32(n - 1), recent=8, sink=4, scale=1.0, out_dtype=torch.float32)
    o, _, tol, _ = attention(q, k, v, False, 1.0, HALF_STEP[dtype], HALF_STEP[torch.float32])
    close(out[0, 0], o, tol)
