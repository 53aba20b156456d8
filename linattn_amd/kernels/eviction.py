"""Eviction of cached keys by the attention weight they gather, on gfx950.

``key_weights`` sums, for each key and KV head, the weights that a prompt's (or a chunk's)
queries give it, from the row sums ``dense_attention`` returned; ``packed_key_weights`` the
same for packed sequences.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from linattn_amd import _native as N
from linattn_amd.kernels.dense import _check_qk, _cu, _int32, _rows, _scale

__all__ = ["key_weights", "packed_key_weights"]


def _last(last: Optional[int]) -> int:
    if last is not None and last <= 0:
        raise ValueError(f"last must be positive, got {last}")
    return last or 0


def _weights_out(what: str, out: Optional[torch.Tensor], shape, dev) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=torch.float32, device=dev)
    if out.dtype != torch.float32 or tuple(out.shape) != tuple(shape) or \
            (out.stride(-1) != 1 and out.shape[-1] > 1):
        raise ValueError(f"{what}: out must be float32 {tuple(shape)} with unit stride over the keys")
    return out


def _lse(what: str, lse: torch.Tensor, shape) -> torch.Tensor:
    if lse.dtype != torch.float32 or tuple(lse.shape) != tuple(shape):
        raise ValueError(f"{what}: lse must be float32 {tuple(shape)}")
    return lse if lse.stride(-1) == 1 else lse.contiguous()


def _run_weights(what: str, a: N.LaKeyWeightsArgs, q, k, lse, out, accumulate, causal, scale,
                 last) -> None:
    dev, D = k.device, q.shape[-1]
    a.q, a.k, a.lse, a.out = q.data_ptr(), k.data_ptr(), lse.data_ptr(), out.data_ptr()
    a.D, a.scale, a.causal, a.last = D, _scale(scale, D), 1 if causal else 0, last
    a.dtype, a.accumulate = N.dtype_code(q.dtype), 1 if accumulate else 0
    L = N.load()
    with torch.cuda.device(dev):
        nbytes = L.la_key_weights_workspace(ctypes.byref(a))
        ws = N.workspace(nbytes, dev)
        a.workspace, a.ws_bytes = N.ptr(ws), nbytes
        N.check(L.la_key_weights(ctypes.byref(a), N.stream_handle(dev)), what)


def key_weights(q: torch.Tensor, k: torch.Tensor, lse: torch.Tensor, *, causal: bool = True,
                scale: Optional[float] = None, last: Optional[int] = None,
                lengths: Optional[torch.Tensor] = None, q_lengths: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The attention weight each key gathers: for key s of KV head h, the sum over the heads
    of its group and the last ``last`` queries (default all) of exp(scale q . k_s - lse).

    q (B, Hq, Tq, D), k (B, Hkv, Tk, D), ``lse`` (B, Hq, Tq) as ``dense_attention`` returned it
    for the same ``causal``, ``scale``, ``lengths`` and ``q_lengths``.  Returns (B, Hkv, Tk)
    in float32, 0 past a sequence's keys; with ``out`` the weights are added to it (the
    weights of chunk after chunk of a prompt).  Sums are in a fixed order."""
    what = "key_weights"
    dev = N.require_gpu(q, k, lse, lengths, q_lengths, out, what=what)
    _check_qk(what, q, k, 4, 1)
    last = _last(last)
    B, Hq, Tq, D = q.shape
    Hkv, Tk = k.shape[1], k.shape[2]
    if k.shape[0] != B:
        raise ValueError(f"{what}: k must be (B, Hkv, Tk, D) in q's batch")
    lse = _lse(what, lse, (B, Hq, Tq))
    lengths = _int32(lengths, (B,), "lengths")
    q_lengths = _int32(q_lengths, (B,), "q_lengths")
    accumulate = out is not None
    out = _weights_out(what, out, (B, Hkv, Tk), dev)
    if B > 0 and Tk > 0:
        q, k = _rows(q), _rows(k)
        a = N.LaKeyWeightsArgs()
        a.q_len, a.k_len = N.ptr(q_lengths), N.ptr(lengths)
        a.B, a.Hq, a.Hkv, a.Tq, a.Tk = B, Hq, Hkv, Tq, Tk
        a.q_sb, a.q_sh, a.q_st = q.stride()[:3]
        a.k_sb, a.k_sh, a.k_st = k.stride()[:3]
        a.l_sb, a.l_sh = lse.stride()[:2]
        a.w_sb, a.w_sh = out.stride()[:2]
        _run_weights(what, a, q, k, lse, out, accumulate, causal, scale, last)
    return out


def packed_key_weights(q: torch.Tensor, k: torch.Tensor, lse: torch.Tensor,
                       cu_seqlens: torch.Tensor, cu_seqlens_k: Optional[torch.Tensor] = None, *,
                       causal: bool = True, scale: Optional[float] = None,
                       last: Optional[int] = None, out: Optional[torch.Tensor] = None
                       ) -> torch.Tensor:
    """``key_weights`` of packed sequences: q (Nq, Hq, D), k (Nk, Hkv, D), ``lse`` (Hq, Nq) of
    ``packed_attention``; ``last`` counts each sequence's own queries.  Returns (Hkv, Nk) in
    float32; keys of no sequence are 0, or left as they were in an ``out`` that is passed."""
    what = "packed_key_weights"
    dev = N.require_gpu(q, k, lse, cu_seqlens, cu_seqlens_k, out, what=what)
    _check_qk(what, q, k, 3, 1)
    last = _last(last)
    Nq, Hq, D = q.shape
    Nk, Hkv = k.shape[:2]
    cu_seqlens = _cu(cu_seqlens, "cu_seqlens")
    B = cu_seqlens.shape[0] - 1
    if cu_seqlens_k is not None:
        cu_seqlens_k = _cu(cu_seqlens_k, "cu_seqlens_k", B)
    elif Nk != Nq:
        raise ValueError(f"{what}: k has other rows than q: pass cu_seqlens_k")
    lse = _lse(what, lse, (Hq, Nq))
    accumulate = out is not None
    out = _weights_out(what, out, (Hkv, Nk), dev)
    if Nk > 0:
        q, k = _rows(q), _rows(k)
        a = N.LaKeyWeightsArgs()
        a.cu_q, a.cu_k = cu_seqlens.data_ptr(), N.ptr(cu_seqlens_k)
        a.B, a.Hq, a.Hkv, a.Tq, a.Tk = B, Hq, Hkv, Nq, Nk
        a.q_st, a.q_sh = q.stride()[:2]
        a.k_st, a.k_sh = k.stride()[:2]
        a.l_sh, a.w_sh = lse.stride(0), out.stride(0)
        a.zero_rest = 0 if accumulate else 1
        _run_weights(what, a, q, k, lse, out, accumulate, causal, scale, last)
    return out
