"""What the eviction entry points refuse, the layouts of their C structures and the plain
selection they are tested against, on the CPU."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import test_abi
from dense_reference import keep, victim
from linattn_amd import _native as N
from linattn_amd.kernels.eviction import (evict_decode_step, evict_kv, key_weights, packed_evict_kv,
                                          packed_key_weights)


@pytest.fixture
def as_gpu(monkeypatch):
    """Lets CPU tensors past the device check; the library itself must not be reached."""
    monkeypatch.setattr(N, "require_gpu", lambda *t, what: torch.device("cpu"))

    def never():
        raise AssertionError("the call was not refused")

    monkeypatch.setattr(N, "load", never)


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def test_cpu_tensors_are_rejected():
    x, w = torch.zeros(1, 1, 4, 64), torch.zeros(1, 1, 4)
    cu = _i32(0, 1)
    for call in (lambda: key_weights(x, x, w), lambda: packed_key_weights(x[0], x[0], w[0], cu),
                 lambda: evict_kv(x, x, w, budget=2, recent=1), lambda: packed_evict_kv(x[0], x[0], w[0], cu, budget=2, recent=1),
                 lambda: evict_decode_step(x[:, :, :1], x[:, :, :1], x[:, :, :1], x, x, w, w.int(), _i32(1), _i32(1), recent=1)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


@pytest.mark.parametrize("change", [
    dict(last=0), dict(last=-4), dict(scale=0.0), dict(scale=math.nan),
    dict(k=torch.zeros(1, 2, 9, 64)), dict(k=torch.zeros(2, 3, 9, 64)), dict(k=torch.zeros(2, 2, 9, 64).half()),
    dict(lse=torch.zeros(2, 4, 7)), dict(lse=torch.zeros(2, 4, 8).double()),
    dict(out=torch.zeros(2, 2, 8)), dict(out=torch.zeros(2, 2, 9).half()), dict(out=torch.zeros(2, 9, 2).transpose(1, 2)),
    dict(lengths=_i32(1)), dict(q_lengths=torch.zeros(2)),
])
def test_key_weights_refuses(as_gpu, change):
    a = dict(q=torch.zeros(2, 4, 8, 64), k=torch.zeros(2, 2, 9, 64), lse=torch.zeros(2, 4, 8))
    a.update(change)
    with pytest.raises(ValueError):
        key_weights(**a)


@pytest.mark.parametrize("change", [
    dict(last=0), dict(k=torch.zeros(9, 2, 64)), dict(lse=torch.zeros(8, 4)), dict(cu_seqlens=torch.zeros(3)),
    dict(cu_seqlens_k=_i32(0, 1)), dict(out=torch.zeros(8, 2)),
])
def test_packed_key_weights_refuses(as_gpu, change):
    a = dict(q=torch.zeros(8, 4, 64), k=torch.zeros(8, 2, 64), lse=torch.zeros(4, 8), cu_seqlens=_i32(0, 3, 8))
    a.update(change)
    with pytest.raises(ValueError):
        packed_key_weights(**a)


@pytest.mark.parametrize("change", [
    dict(budget=0), dict(budget=4), dict(recent=-1), dict(sink=-1), dict(sink=7), dict(capacity=7),
    dict(v=torch.zeros(2, 2, 8, 64)), dict(v=torch.zeros(2, 2, 9, 64).half()), dict(k=torch.zeros(2, 9, 64)),
    dict(k=torch.zeros(2, 2, 9, 3), v=torch.zeros(2, 2, 9, 3)),
    dict(k=torch.zeros(2, 2, 9, 64).double(), v=torch.zeros(2, 2, 9, 64).double()),
    dict(weights=torch.zeros(2, 2, 8)), dict(weights=torch.zeros(2, 2, 9).half()),
    dict(lengths=_i32(1)), dict(pos=_i32(1, 2)), dict(positions=torch.zeros(2, 2, 9, dtype=torch.int32)),
    dict(positions=torch.zeros(2, 2, 9), pos=_i32(1, 2)), dict(positions=torch.zeros(2, 2, 9, dtype=torch.int32), pos=_i32(1)),
])
def test_evict_kv_refuses(as_gpu, change):
    a = dict(k=torch.zeros(2, 2, 9, 64), v=torch.zeros(2, 2, 9, 64), weights=torch.zeros(2, 2, 9), budget=8, recent=5, sink=2)
    a.update(change)
    with pytest.raises(ValueError):
        evict_kv(**a)


def test_packed_evict_kv_refuses(as_gpu):
    k, w, cu = torch.zeros(9, 2, 64), torch.zeros(2, 9), _i32(0, 9)
    for a in ((k, k, w.t(), cu), (k, k[1:], w, cu), (k, k, w, cu.long()), (k[None], k[None], w, cu)):
        with pytest.raises(ValueError):
            packed_evict_kv(*a, budget=4, recent=1)
    with pytest.raises(ValueError):
        packed_evict_kv(k, k, w, cu, budget=4, recent=4, sink=1)


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(2, 4, 2, 64)), dict(q=torch.zeros(2, 4, 1, 128)), dict(q=torch.zeros(2, 34, 1, 64)),
    dict(q=torch.zeros(2, 3, 1, 64)), dict(k_new=torch.zeros(2, 2, 2, 64)), dict(v_new=torch.zeros(2, 2, 1, 64).half()),
    dict(k_cache=torch.zeros(2, 2, 9, 64).half()), dict(k_cache=torch.zeros(2, 9, 2, 64).transpose(1, 2)),
    dict(v_cache=torch.zeros(2, 2, 8, 64)), dict(weights=torch.zeros(2, 2, 9).double()),
    dict(weights=torch.zeros(2, 2, 18)[..., ::2]), dict(positions=torch.zeros(2, 2, 9)),
    dict(positions=torch.zeros(2, 2, 8, dtype=torch.int32)), dict(lengths=_i32(1)), dict(pos=torch.zeros(2)),
    dict(recent=9), dict(recent=5, sink=4), dict(recent=-1), dict(sink=-1), dict(scale=-1.0),
    dict(out=torch.zeros(2, 4, 1, 63)), dict(out_dtype=torch.float16),
])
def test_evict_decode_step_refuses(as_gpu, change):
    c = torch.zeros(2, 2, 9, 64)
    a = dict(q=torch.zeros(2, 4, 1, 64), k_new=c[:, :, :1].clone(), v_new=c[:, :, :1].clone(), k_cache=c, v_cache=c.clone(),
             weights=torch.zeros(2, 2, 9), positions=torch.zeros(2, 2, 9, dtype=torch.int32), lengths=_i32(1, 2), pos=_i32(1, 2),
             recent=4, sink=2)
    a.update(change)
    with pytest.raises(ValueError):
        evict_decode_step(**a)


def test_arguments_that_share_memory_are_refused(as_gpu):
    c, w = torch.zeros(2, 2, 9, 64), torch.zeros(2, 2, 9)
    new = torch.zeros(2, 2, 1, 64)
    a = dict(q=torch.zeros(2, 2, 1, 64), k_new=new, v_new=new, k_cache=c, v_cache=c.clone(), weights=w,
             positions=torch.zeros(2, 2, 9, dtype=torch.int32), lengths=_i32(1, 2), pos=_i32(1, 2), recent=4, sink=2)
    for change in (dict(v_cache=c), dict(k_new=c[:, :, :1]), dict(v_new=c[:, :, :1]), dict(positions=w.view(torch.int32)),
                   dict(out=a["q"]), dict(out=new), dict(out=torch.zeros(1, 2, 1, 64).expand(2, 2, 1, 64)),
                   dict(out=c.view(-1)[128:384].view(2, 2, 1, 64))):
        with pytest.raises(ValueError, match="share|twice"):
            evict_decode_step(**{**a, **change})
    with pytest.raises(AssertionError, match="not refused"):  # (the same new row twice is only read)
        evict_decode_step(**a)
    q, lse = torch.zeros(2, 2, 9, 64), torch.zeros(2, 2, 9)
    for out in (lse, torch.zeros(2, 1, 9).expand(2, 2, 9)):
        with pytest.raises(ValueError, match="share|twice"):
            key_weights(q, c, lse, out=out)


def test_c_entries_refuse_without_a_gpu():
    L = N.load()
    for call, a in ((L.la_key_weights, N.LaKeyWeightsArgs()), (L.la_evict_kv, N.LaEvictArgs()),
                    (L.la_evict_decode, N.LaEvictDecodeArgs())):
        assert call(ctypes.byref(a), None) == N.LA_ERR_INVALID and L.la_last_error()
    a = N.LaEvictArgs()
    a.B, a.Hkv, a.T, a.D, a.esize, a.budget, a.capacity = 1, 1, 8000, 64, 2, 4, 4
    a.k = a.v = a.weights = a.k_out = a.v_out = a.w_out = a.pos_out = a.len_out = 4096
    a.k_sh = a.k_st = a.v_st = 64
    assert L.la_evict_kv_workspace(ctypes.byref(a)) > 0
    assert L.la_evict_kv(ctypes.byref(a), None) == N.LA_ERR_WORKSPACE
    a.recent = 5
    assert L.la_evict_kv(ctypes.byref(a), None) == N.LA_ERR_INVALID
    d = N.LaEvictDecodeArgs()
    d.B, d.Hq, d.Hkv, d.C, d.D, d.scale, d.dtype, d.out_dtype = 1, 40, 2, 8, 64, 0.1, N.LA_F32, N.LA_F32
    assert L.la_evict_decode(ctypes.byref(d), None) == N.LA_ERR_INVALID
    assert b"16 times" in L.la_last_error()


def test_struct_layouts_match_the_header(tmp_path, monkeypatch):
    monkeypatch.setattr(test_abi, "STRUCTS", {
        "la_dense_attn_args": N.LaDenseAttnArgs, "la_key_weights_args": N.LaKeyWeightsArgs,
        "la_evict_args": N.LaEvictArgs, "la_evict_decode_args": N.LaEvictDecodeArgs})
    test_abi.test_struct_layouts_match_the_header(tmp_path)


def test_plain_selection():
    w = [0.5, 9.0, 1.0, 1.0, math.nan, 1.0, 3.0, 0.1]
    assert keep(w, 8, 4, 1, 1) == [0, 1, 6, 7]
    assert keep(w, 8, 5, 1, 1) == [0, 1, 2, 6, 7]  # of equal ones the first
    assert keep(w, 3, 5, 1, 1) == [0, 1, 2]
    assert keep(w, 8, 3, 2, 0, positions=[7, 6, 0, 1, 2, 3, 4, 5], pos=8) == [0, 1, 6]
    assert victim([1.0, 0.5, 0.5, 0.0], 1, 0, [0, 1, 2, 3], 4) == 2
    assert victim([1.0, math.nan, 0.5, 0.0], 1, 0, [0, 1, 2, 3], 4) == 1
    assert victim([1.0, 0.5], 1, 1, [0, 1], 2) == 1
