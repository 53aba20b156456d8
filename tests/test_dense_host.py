"""What ``dense_attention`` and ``packed_attention`` refuse, and the 64-bit reference they are
tested against, on the CPU."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from dense_reference import attention, key_weights
from linattn_amd import _native as N
from linattn_amd.kernels import dense
from linattn_amd.kernels.dense import dense_attention, packed_attention


@pytest.fixture
def as_gpu(monkeypatch):
    """Lets CPU tensors past the device check, so that what follows it can be tested here."""
    monkeypatch.setattr(N, "require_gpu", lambda *t, what: torch.device("cpu"))

    def never(*a):
        raise AssertionError("the call was not refused")

    monkeypatch.setattr(dense, "_run", never)


def test_cpu_tensors_are_rejected():
    x = torch.zeros(1, 1, 4, 64)
    with pytest.raises(RuntimeError, match="GPU"):
        dense_attention(x, x, x)
    with pytest.raises(RuntimeError, match="GPU"):
        packed_attention(x[0], x[0], x[0], torch.tensor([0, 1], dtype=torch.int32))


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(2, 4, 8, 96), k=torch.zeros(2, 2, 8, 96), v=torch.zeros(2, 2, 8, 96)),
    dict(q=torch.zeros(2, 3, 8, 64)),
    dict(q=torch.zeros(2, 4, 8, 128)),
    dict(q=torch.zeros(2, 4, 8, 64, dtype=torch.float64)),
    dict(q=torch.zeros(4, 8, 64)),
    dict(k=torch.zeros(1, 2, 8, 64)),
    dict(k=torch.zeros(2, 0, 8, 64), v=torch.zeros(2, 0, 8, 64)),
    dict(k=torch.zeros(2, 2, 8, 64).bfloat16()),
    dict(v=torch.zeros(2, 2, 9, 64)),
    dict(v=torch.zeros(2, 2, 8, 64).half()),
    dict(lengths=torch.zeros(3, dtype=torch.int32)),
    dict(lengths=torch.zeros(2, dtype=torch.int64)),
    dict(q_lengths=torch.zeros(2, 1, dtype=torch.int32)),
    dict(out=torch.zeros(2, 4, 8, 32)),
    dict(out=torch.zeros(2, 4, 8, 64).half()),
    dict(out=torch.zeros(2, 4, 8, 65)[..., 1:]),
    dict(out=torch.zeros(2, 4, 8, 64), out_dtype=torch.bfloat16),
    dict(out_dtype=torch.bfloat16),
])
def test_dense_attention_refuses(as_gpu, change):
    a = dict(q=torch.zeros(2, 4, 8, 64), k=torch.zeros(2, 2, 8, 64), v=torch.zeros(2, 2, 8, 64))
    a.update(change)
    with pytest.raises(ValueError):
        dense_attention(a.pop("q"), a.pop("k"), a.pop("v"), **a)


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(9, 4, 64)),
    dict(q=torch.zeros(1, 8, 4, 64)),
    dict(cu_seqlens=torch.zeros(3)),
    dict(cu_seqlens=torch.zeros(1, dtype=torch.int32)),
    dict(cu_seqlens=torch.zeros(2, 2, dtype=torch.int32)),
    dict(cu_seqlens_k=torch.zeros(4, dtype=torch.int32)),
    dict(v=torch.zeros(8, 2, 128)),
])
def test_packed_attention_refuses(as_gpu, change):
    a = dict(q=torch.zeros(8, 4, 64), k=torch.zeros(8, 2, 64), v=torch.zeros(8, 2, 64),
             cu_seqlens=torch.tensor([0, 3, 8], dtype=torch.int32))
    a.update(change)
    with pytest.raises(ValueError):
        packed_attention(**a)


def test_outputs_that_share_memory_are_refused(as_gpu):
    q, kv = torch.zeros(2, 4, 8, 64), torch.zeros(2, 2, 8, 64)
    for out in (q, q[:, :, :, :], torch.zeros(1, 4, 8, 64).expand(2, 4, 8, 64)):
        with pytest.raises(ValueError, match="shares memory|twice"):
            dense_attention(q, kv, kv.clone(), out=out)
    whole = torch.zeros(3 * 8, 2, 64)  # q and out overlap by eight rows
    cu = torch.tensor([0, 16], dtype=torch.int32)
    k = torch.zeros(16, 2, 64)
    with pytest.raises(ValueError, match="shares memory"):
        packed_attention(whole[:16], k, k.clone(), cu, out=whole[8:])
    both = torch.zeros(16, 4, 64)  # heads of one buffer, interleaved: no row is shared
    with pytest.raises(AssertionError, match="not refused"):
        packed_attention(both[:, :2], k, k.clone(), cu, out=both[:, 2:])


@pytest.mark.parametrize("scale", [0.0, -1.0, math.inf, math.nan])
def test_scale_is_positive(scale):
    with pytest.raises(ValueError):
        dense._scale(scale, 64)
    assert dense._scale(None, 64) == 0.125


def test_c_entry_refuses_without_a_gpu():
    L = N.load()
    a = N.LaDenseAttnArgs()
    assert L.la_dense_attention(ctypes.byref(a), None) == N.LA_ERR_INVALID
    a.B, a.Hq, a.Hkv, a.Tq, a.Tk, a.D, a.scale, a.dtype, a.out_dtype = 1, 4, 2, 8, 8, 64, 0.1, N.LA_F32, N.LA_F32
    assert L.la_dense_attention(ctypes.byref(a), None) == N.LA_ERR_INVALID
    assert b"null q" in L.la_last_error()
    a.q = a.k = a.v = a.out = 4096 + 4
    assert L.la_dense_attention(ctypes.byref(a), None) == N.LA_ERR_INVALID
    assert b"aligned" in L.la_last_error()
    a.D = 80
    assert L.la_dense_attention(ctypes.byref(a), None) == N.LA_ERR_INVALID


def test_reference_is_the_masked_softmax():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(n, 64, generator=g).double() for n in (5, 9, 9))
    x = q @ k.t() / 8.0
    x = x.masked_fill(torch.ones(5, 9, dtype=torch.bool).triu(9 - 5 + 1), -math.inf)
    out, lse, tol, tol_lse = attention(q, k, v)
    assert torch.allclose(out, torch.softmax(x, -1) @ v, rtol=1e-13, atol=1e-13)
    assert torch.allclose(lse, torch.logsumexp(x, -1), rtol=1e-13)
    assert (tol < 1e-3).all() and (tol_lse < 1e-3).all()
    w, tol = key_weights(q[None], k, lse[None])
    assert torch.allclose(w, torch.softmax(x, -1).sum(0), rtol=1e-12)
    w, _ = key_weights(q[None], k, lse[None], last=2)
    assert torch.allclose(w, torch.softmax(x, -1)[-2:].sum(0), rtol=1e-12)
    out, lse, _, _ = attention(k, q, v[:5])  # more queries than keys
    assert (out[:4] == 0).all() and (lse[:4] == -math.inf).all() and torch.equal(out[4], v[0].double())
