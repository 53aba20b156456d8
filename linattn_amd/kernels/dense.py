"""Dense causal attention on gfx950: whole prompts, chunks and single tokens.

``dense_attention`` is the attention of core.py:148-181 (softmax of the scaled scores,
causal, grouped heads) over the framework's (B, H, T, D) tensors, ``packed_attention`` the
same over sequences of different lengths packed one behind the other.  Nothing of the
(Tq, Tk) score matrix is stored.  Both can return each row's log sum of exponentials,
which ``linattn_amd.kernels.eviction`` weighs cached keys by.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple, Union

import torch

from linattn_amd import _native as N

__all__ = ["dense_attention", "packed_attention"]

_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def _rows(t: torch.Tensor, token: int = -2) -> torch.Tensor:
    """``t`` with rows the kernels can load 16 bytes at a time (a copy where they are not
    contiguous and 16-byte aligned, or the rows of dimension ``token`` very far apart)."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():  # (head sizes are whole 16-byte chunks)
            return t
        n = 16 // t.element_size()
        st = t.stride()
        if st[-1] == 1 and st[token] < 1 << 24 and \
                all(s % n == 0 for s, d in zip(st[:-1], t.shape) if d > 1):
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _int32(t: Optional[torch.Tensor], shape: Tuple[int, ...], what: str) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.dtype != torch.int32 or tuple(t.shape) != shape:
        raise ValueError(f"{what} must be int32 {shape}")
    return t.contiguous()


def _cu(cu: torch.Tensor, what: str, B: Optional[int] = None) -> torch.Tensor:
    if cu.dtype != torch.int32 or cu.dim() != 1 or cu.shape[0] < 2 or \
            (B is not None and cu.shape[0] != B + 1):
        raise ValueError(f"{what} must be int32 (B + 1,)")
    return cu.contiguous()


def _scale(scale: Optional[float], D: int) -> float:
    s = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < s < 1e30:
        raise ValueError(f"scale must be positive, got {scale}")
    return s


def _check_qk(what: str, q: torch.Tensor, k: torch.Tensor, dims: int, head: int) -> None:
    qs, ks, dt = q.shape, k.shape, q.dtype
    if len(qs) != dims or len(ks) != dims:
        raise ValueError(f"{what}: q and k must have {dims} dimensions")
    if dt != k.dtype or dt not in _TYPES:
        raise ValueError(f"{what}: q, k and v must share one of bfloat16, float16, float32")
    if qs[-1] not in (64, 128) or ks[-1] != qs[-1]:
        raise ValueError(f"{what}: head_dim must be 64 or 128, and the same in q and k")
    if ks[head] == 0 or qs[head] == 0 or qs[head] % ks[head]:
        raise ValueError(f"{what}: the query heads must be a multiple of the KV heads")


def _apart(what: str, out: torch.Tensor, *inputs: torch.Tensor) -> None:
    """Refuses an ``out`` that holds a row twice, starts where an input does, or whose memory
    is part of a contiguous input's (the library looks at what is left, byte by byte: views
    that interleave with ``out`` pass)."""
    if out.numel() == 0:
        return
    if any(s == 0 and d > 1 for s, d in zip(out.stride(), out.shape)):
        raise ValueError(f"{what}: out holds some of its rows twice")
    span = lambda t: t.data_ptr() + t.element_size() * (1 + sum((d - 1) * s for d, s in zip(t.shape, t.stride())))
    a, e, whole = out.data_ptr(), span(out), out.is_contiguous()
    for t in inputs:
        if t.numel() and (t.data_ptr() == a or (t.data_ptr() < e and a < span(t) and whole and t.is_contiguous())):
            raise ValueError(f"{what}: out shares memory with an input")


def _out(what: str, out: Optional[torch.Tensor], q: torch.Tensor,
         out_dtype: Optional[torch.dtype], *inputs: torch.Tensor) -> torch.Tensor:
    """(out, or a new one, checked)."""
    if out is None:
        if out_dtype is not None and out_dtype not in (q.dtype, torch.float32):
            raise ValueError(f"{what}: out_dtype is q's or float32")
        return torch.empty_like(q, dtype=out_dtype, memory_format=torch.contiguous_format)
    if out.shape != q.shape or out.dtype not in (q.dtype, torch.float32) or \
            (out_dtype is not None and out.dtype != out_dtype):
        raise ValueError(f"{what}: out must be q's shape in q's dtype (or float32)")
    n = 16 // out.element_size()
    if out.stride(-1) != 1 or out.data_ptr() % 16 or \
            any(s % n for s, d in zip(out.stride()[:-1], out.shape) if d > 1):
        raise ValueError(f"{what}: rows of out must be contiguous and 16-byte aligned")
    _apart(what, out, q, *inputs)
    return out


def _run(what: str, q, k, v, out, lse, cu_q, cu_k, q_len, k_len, shape, q_s, k_s, v_s, o_s, l_s,
         causal, scale, zero_rest) -> None:
    dev, D = q.device, q.shape[-1]
    a = N.LaDenseAttnArgs(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), N.ptr(lse), N.ptr(cu_q), N.ptr(cu_k),
        N.ptr(q_len), N.ptr(k_len), None, 0, *shape, D, *q_s, *k_s, *v_s, *o_s, *l_s, _scale(scale, D),
        1 if causal else 0, N.dtype_code(q.dtype), N.dtype_code(out.dtype), zero_rest, 0)
    L, ref = N.load(), ctypes.byref(a)
    with N.on_device(dev):
        nbytes = L.la_dense_attention_workspace(ref)
        if nbytes:
            ws = N.workspace(nbytes, dev)
            a.workspace, a.ws_bytes = ws.data_ptr(), nbytes
        N.check(L.la_dense_attention(ref, N.stream_handle(dev)), what)


def dense_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = True,
                    scale: Optional[float] = None, lengths: Optional[torch.Tensor] = None,
                    q_lengths: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                    out_dtype: Optional[torch.dtype] = None, return_lse: bool = False
                    ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """softmax(scale q k^T) v with grouped heads, one pass over k and v.

    q (B, Hq, Tq, D), k/v (B, Hkv, Tk, D), all bfloat16, float16 or float32, D 64 or 128.
    ``lengths`` (int32 (B,), default Tk) gives each sequence's keys, ``q_lengths`` (int32
    (B,), default Tq) its queries: the rest is padding and is never read.  With ``causal``
    the queries are the last of the keys' positions: query t of a sequence sees keys
    0 .. lengths - q_lengths + t (a prompt: both lengths; a chunk or one token behind a
    cache: the keys' alone).  Returns (B, Hq, Tq, D) in ``out_dtype`` (default q's, or
    float32), or in ``out`` (which shares no memory with the inputs), and with ``return_lse``
    also the rows' log sums of exponentials (B, Hq, Tq) in float32.  A query that sees no key, and one past ``q_lengths``, gets
    zeros and -inf.  Infinities and NaN a query does not see do not reach it.  Forward
    only: no gradient is recorded."""
    what = "dense_attention"
    dev = N.require_gpu(q, k, v, lengths, q_lengths, out, what=what)
    _check_qk(what, q, k, 4, 1)
    B, Hq, Tq, D = q.shape
    Hkv, Tk = k.shape[1], k.shape[2]
    if k.shape[0] != B or v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"{what}: k and v must be (B, Hkv, Tk, D) in q's batch and dtype")
    lengths = _int32(lengths, (B,), "lengths")
    q_lengths = _int32(q_lengths, (B,), "q_lengths")
    out = _out(what, out, q, out_dtype, k, v)
    lse = torch.empty(B, Hq, Tq, dtype=torch.float32, device=dev) if return_lse else None
    if B > 0 and Tq > 0:
        q, k, v = _rows(q), _rows(k), _rows(v)
        _run(what, q, k, v, out, lse, None, None, q_lengths, lengths, (B, Hq, Hkv, Tq, Tk), q.stride()[:3],
             k.stride()[:3], v.stride()[:3], out.stride()[:3], (Hq * Tq, Tq), causal, scale, 0)
    return (out, lse) if return_lse else out


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     cu_seqlens_k: Optional[torch.Tensor] = None, *, causal: bool = True,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                     out_dtype: Optional[torch.dtype] = None, return_lse: bool = False
                     ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``dense_attention`` of sequences packed one behind the other.

    q (Nq, Hq, D), k/v (Nk, Hkv, D); ``cu_seqlens`` (int32 (B + 1,), ascending, on the
    device): sequence b's queries are rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1, its keys
    those rows of k and v by ``cu_seqlens_k`` (default ``cu_seqlens``, and then Nk = Nq).
    Sequences may be empty.  Causality as in ``dense_attention`` (the queries end where
    their keys end).  Returns (Nq, Hq, D), and with ``return_lse`` (Hq, Nq) in float32.
    Rows that no sequence holds are left as they were in an ``out`` that is passed, else
    they are zeros; their lse is -inf."""
    what = "packed_attention"
    dev = N.require_gpu(q, k, v, cu_seqlens, cu_seqlens_k, out, what=what)
    _check_qk(what, q, k, 3, 1)
    Nq, Hq, D = q.shape
    Nk, Hkv = k.shape[:2]
    if v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"{what}: k and v must be (Nk, Hkv, D) in q's dtype")
    cu_seqlens = _cu(cu_seqlens, "cu_seqlens")
    B = cu_seqlens.shape[0] - 1
    if cu_seqlens_k is not None:
        cu_seqlens_k = _cu(cu_seqlens_k, "cu_seqlens_k", B)
    elif Nk != Nq:
        raise ValueError(f"{what}: k has other rows than q: pass cu_seqlens_k")
    zero_rest = out is None
    out = _out(what, out, q, out_dtype, k, v)
    lse = None
    if return_lse:  # (where out's rows are left, so would the lse's be)
        lse = torch.empty(Hq, Nq, dtype=torch.float32, device=dev) if zero_rest else \
            torch.full((Hq, Nq), float("-inf"), dtype=torch.float32, device=dev)
    if Nq > 0:
        q, k, v = _rows(q, 0), _rows(k, 0), _rows(v, 0)
        (q_t, q_h, _), (k_t, k_h, _), (v_t, v_h, _), (o_t, o_h, _) = (x.stride() for x in (q, k, v, out))
        _run(what, q, k, v, out, lse, cu_seqlens, cu_seqlens_k, None, None, (B, Hq, Hkv, Nq, Nk), (0, q_h, q_t),
             (0, k_h, k_t), (0, v_h, v_t), (0, o_h, o_t), (0, Nq), causal, scale, 1 if zero_rest else 0)
    return (out, lse) if return_lse else out
