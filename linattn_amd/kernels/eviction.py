"""Eviction of cached keys by the attention weight they gather, on gfx950.

``key_weights`` sums, for each key and KV head, the weights that a prompt's (or a chunk's)
queries give it, from the row sums ``dense_attention`` returned; ``evict_kv`` keeps the first,
the newest and the heaviest entries of each cache up to a budget; ``packed_key_weights`` and
``packed_evict_kv`` do the same for packed sequences.  ``evict_decode_step`` goes on from there
token by token: evict, append, attend and gather weights in one call.  Each KV head keeps
entries of its own.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from linattn_amd import _native as N
from linattn_amd.kernels.dense import _TYPES, _apart, _check_qk, _cu, _int32, _out, _rows, _scale

__all__ = ["key_weights", "packed_key_weights", "evict_kv", "packed_evict_kv", "evict_decode_step"]


def _last(last: Optional[int]) -> int:
    if last is not None and last <= 0:
        raise ValueError(f"last must be positive, got {last}")
    return last or 0


def _weights_out(what: str, out: Optional[torch.Tensor], shape, dev, *inputs) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=torch.float32, device=dev)
    if out.dtype != torch.float32 or tuple(out.shape) != tuple(shape) or \
            (out.stride(-1) != 1 and out.shape[-1] > 1):
        raise ValueError(f"{what}: out must be float32 {tuple(shape)} with unit stride over the keys")
    _apart(what, out, *inputs)
    return out


def _lse(what: str, lse: torch.Tensor, shape) -> torch.Tensor:
    if lse.dtype != torch.float32 or tuple(lse.shape) != tuple(shape):
        raise ValueError(f"{what}: lse must be float32 {tuple(shape)}")
    return lse if lse.stride(-1) == 1 else lse.contiguous()


def _run_weights(what: str, q, k, lse, out, cu_q, cu_k, q_len, k_len, shape, q_s, k_s, l_s, w_s, last,
                 causal, scale, accumulate, zero_rest) -> None:
    dev, D = k.device, q.shape[-1]
    a = N.LaKeyWeightsArgs(
        q.data_ptr(), k.data_ptr(), lse.data_ptr(), out.data_ptr(), N.ptr(cu_q), N.ptr(cu_k), N.ptr(q_len),
        N.ptr(k_len), None, 0, *shape, D, *q_s, *k_s, *l_s, *w_s, last, _scale(scale, D), 1 if causal else 0,
        N.dtype_code(q.dtype), 1 if accumulate else 0, zero_rest, 0)
    L, ref = N.load(), ctypes.byref(a)
    with N.on_device(dev):
        nbytes = L.la_key_weights_workspace(ref)
        if nbytes:
            ws = N.workspace(nbytes, dev)
            a.workspace, a.ws_bytes = ws.data_ptr(), nbytes
        N.check(L.la_key_weights(ref, N.stream_handle(dev)), what)


def key_weights(q: torch.Tensor, k: torch.Tensor, lse: torch.Tensor, *, causal: bool = True,
                scale: Optional[float] = None, last: Optional[int] = None,
                lengths: Optional[torch.Tensor] = None, q_lengths: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The attention weight each key gathers: for key s of KV head h, the sum over the heads
    of its group and the last ``last`` queries (default all) of exp(scale q . k_s - lse).

    q (B, Hq, Tq, D), k (B, Hkv, Tk, D), ``lse`` (B, Hq, Tq) as ``dense_attention`` returned it
    for the same ``causal``, ``scale``, ``lengths`` and ``q_lengths``; a query whose lse is -inf
    adds nothing, whatever its row of q holds.  Returns (B, Hkv, Tk) in float32, 0 past a
    sequence's keys; with ``out`` the weights are added to it (the
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
    out = _weights_out(what, out, (B, Hkv, Tk), dev, q, k, lse)
    if B > 0 and Tk > 0:
        q, k = _rows(q), _rows(k)
        _run_weights(what, q, k, lse, out, None, None, q_lengths, lengths, (B, Hq, Hkv, Tq, Tk), q.stride()[:3],
                     k.stride()[:3], lse.stride()[:2], out.stride()[:2], last, causal, scale, accumulate, 0)
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
    out = _weights_out(what, out, (Hkv, Nk), dev, q, k, lse)
    if Nk > 0:
        q, k = _rows(q, 0), _rows(k, 0)
        (q_t, q_h, _), (k_t, k_h, _) = q.stride(), k.stride()
        _run_weights(what, q, k, lse, out, cu_seqlens, cu_seqlens_k, None, None, (B, Hq, Hkv, Nq, Nk), (0, q_h, q_t),
                     (0, k_h, k_t), (0, lse.stride(0)), (0, out.stride(0)), last, causal, scale, accumulate,
                     0 if accumulate else 1)
    return out


Evicted = Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]


def _budget(what: str, budget: int, recent: int, sink: int, capacity: Optional[int]) -> int:
    if budget <= 0 or recent < 0 or sink < 0 or recent + sink > budget:
        raise ValueError(f"{what}: sink + recent must fit a positive budget, got {sink} + {recent} of {budget}")
    capacity = budget if capacity is None else capacity
    if capacity < budget:
        raise ValueError(f"{what}: capacity {capacity} is less than the budget {budget}")
    return capacity


def _run_evict(what: str, k, v, weights, positions, pos, lengths, cu, B: int, Hkv: int, T: int, k_s, v_s, w_s,
               ps_s, budget, recent, sink, capacity) -> Evicted:
    dev, D = k.device, k.shape[-1]
    k_out = torch.empty(B, Hkv, capacity, D, dtype=k.dtype, device=dev)
    v_out = torch.empty_like(k_out)
    w_out = torch.empty(B, Hkv, capacity, dtype=torch.float32, device=dev)
    pos_out = torch.empty_like(w_out, dtype=torch.int32)
    len_out = torch.empty(B, dtype=torch.int32, device=dev)
    if B > 0:
        a = N.LaEvictArgs(
            k.data_ptr(), v.data_ptr(), weights.data_ptr(), N.ptr(positions), N.ptr(pos), N.ptr(lengths), N.ptr(cu),
            k_out.data_ptr(), v_out.data_ptr(), w_out.data_ptr(), pos_out.data_ptr(), len_out.data_ptr(), None, 0,
            B, Hkv, T, D, k.element_size(), *k_s, *v_s, *w_s, *ps_s, budget, capacity, recent, sink)
        L, ref = N.load(), ctypes.byref(a)
        with N.on_device(dev):
            nbytes = L.la_evict_kv_workspace(ref)
            if nbytes:
                ws = N.workspace(nbytes, dev)
                a.workspace, a.ws_bytes = ws.data_ptr(), nbytes
            N.check(L.la_evict_kv(ref, N.stream_handle(dev)), what)
    return k_out, v_out, w_out, pos_out, len_out


def _check_cache(what: str, k: torch.Tensor, v: torch.Tensor, dims: int) -> None:
    if k.dim() != dims or v.shape != k.shape or v.dtype != k.dtype or k.dtype not in _TYPES:
        raise ValueError(f"{what}: k and v must have {dims} dimensions, one shape and one of "
                         "bfloat16, float16, float32")
    if k.shape[-1] == 0 or k.shape[-1] * k.element_size() % 16:
        raise ValueError(f"{what}: rows of k and v must be whole 16-byte chunks")
    if k.shape[1] == 0:
        raise ValueError(f"{what}: no KV heads")


def evict_kv(k: torch.Tensor, v: torch.Tensor, weights: torch.Tensor, *, budget: int, recent: int,
             sink: int = 0, lengths: Optional[torch.Tensor] = None,
             positions: Optional[torch.Tensor] = None, pos: Optional[torch.Tensor] = None,
             capacity: Optional[int] = None) -> Evicted:
    """Keep ``budget`` entries of each cache: the first ``sink`` and the newest ``recent``
    tokens, then the heaviest by ``weights`` (ties to the lowest index; NaN is lightest).

    k/v (B, Hkv, T, D), ``weights`` (B, Hkv, T) float32 (``key_weights``), ``lengths`` (int32 (B,),
    default T) the entries held.  An entry's token is its index, or ``positions`` (int32
    (B, Hkv, T)) of a cache that was evicted before, with ``pos`` (int32 (B,)) the position
    of the next token.  Returns new tensors (k, v, weights, positions, lengths) with room for
    ``capacity`` (default ``budget``) entries: the kept ones in their order, then zeros with
    weight 0 and position -1; a cache shorter than the budget is kept whole.  A capacity of
    ``budget + 1`` is what ``evict_decode_step`` goes on with."""
    what = "evict_kv"
    dev = N.require_gpu(k, v, weights, lengths, positions, pos, what=what)
    _check_cache(what, k, v, 4)
    capacity = _budget(what, budget, recent, sink, capacity)
    B, Hkv, T, _ = k.shape
    if weights.dtype != torch.float32 or weights.shape != (B, Hkv, T):
        raise ValueError(f"{what}: weights must be float32 (B, Hkv, T)")
    if (positions is None) != (pos is None):
        raise ValueError(f"{what}: pass both positions and pos, or neither")
    if positions is not None and (positions.dtype != torch.int32 or positions.shape != (B, Hkv, T)):
        raise ValueError(f"{what}: positions must be int32 (B, Hkv, T)")
    lengths, pos = _int32(lengths, (B,), "lengths"), _int32(pos, (B,), "pos")
    k, v = _rows(k), _rows(v)
    weights = weights if weights.stride(-1) == 1 else weights.contiguous()
    ps_s = (0, 0)
    if positions is not None:
        positions = positions if positions.stride(-1) == 1 else positions.contiguous()
        ps_s = positions.stride()[:2]
    return _run_evict(what, k, v, weights, positions, pos, lengths, None, B, Hkv, T, k.stride()[:3], v.stride()[:3],
                      weights.stride()[:2], ps_s, budget, recent, sink, capacity)


def packed_evict_kv(k: torch.Tensor, v: torch.Tensor, weights: torch.Tensor,
                    cu_seqlens: torch.Tensor, *, budget: int, recent: int, sink: int = 0,
                    capacity: Optional[int] = None) -> Evicted:
    """``evict_kv`` of packed sequences: k/v (Nk, Hkv, D), ``weights`` (Hkv, Nk) as
    ``packed_key_weights`` returns them, sequence b's entries rows cu_seqlens[b] ..
    cu_seqlens[b + 1] - 1.  Returns caches of their own, as ``evict_kv`` does; positions
    count within each sequence."""
    what = "packed_evict_kv"
    N.require_gpu(k, v, weights, cu_seqlens, what=what)
    _check_cache(what, k, v, 3)
    capacity = _budget(what, budget, recent, sink, capacity)
    Nk, Hkv, _ = k.shape
    if weights.dtype != torch.float32 or weights.shape != (Hkv, Nk):
        raise ValueError(f"{what}: weights must be float32 (Hkv, Nk)")
    cu_seqlens = _cu(cu_seqlens, "cu_seqlens")
    k, v = _rows(k), _rows(v)
    weights = weights if weights.stride(-1) == 1 else weights.contiguous()
    (k_t, k_h, _), (v_t, v_h, _) = k.stride(), v.stride()
    return _run_evict(what, k, v, weights, None, None, None, cu_seqlens, cu_seqlens.shape[0] - 1, Hkv, Nk,
                      (0, k_h, k_t), (0, v_h, v_t), (0, weights.stride(0)), (0, 0), budget, recent, sink, capacity)


def evict_decode_step(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                      k_cache: torch.Tensor, v_cache: torch.Tensor, weights: torch.Tensor,
                      positions: torch.Tensor, lengths: torch.Tensor, pos: torch.Tensor, *,
                      recent: int, sink: int = 0, scale: Optional[float] = None,
                      out: Optional[torch.Tensor] = None,
                      out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """One token over caches that evict, updated in place.

    q (B, Hq, 1, D), k_new/v_new (B, Hkv, 1, D), caches (B, Hkv, C, D) in the same dtype,
    ``weights`` float32 and ``positions`` int32 (B, Hkv, C), ``lengths`` and ``pos`` int32 (B,):
    the entries each cache holds and the new token's position.  For each (sequence, KV
    head): a full cache loses its lightest entry that is neither among the first ``sink``
    nor the newest ``recent`` tokens (position >= sink and < pos - recent; of equal weights
    the highest slot; NaN is lightest; the highest slot if nothing else is left); the new
    token takes its slot (or the next free one); the query heads attend the cache with it;
    every entry's weight grows by the weights they gave it.  Returns (B, Hq, 1, D) in
    ``out_dtype`` (default q's, or float32), or in ``out``.

    The caller advances ``lengths`` (to at most C) and ``pos``.  Caches are contiguous, share
    no memory with one another or with other arguments, and a call's are not another's: two
    streams may run two calls on caches of their own."""
    what = "evict_decode_step"
    dev = N.require_gpu(q, k_new, v_new, k_cache, v_cache, weights, positions, lengths, pos, out,
                        what=what)
    _check_qk(what, q, k_cache, 4, 1)
    B, Hq, Tq, D = q.shape
    Hkv, C = k_cache.shape[1], k_cache.shape[2]
    if Tq != 1 or k_cache.shape[0] != B:
        raise ValueError(f"{what}: one token of each sequence: q (B, Hq, 1, D)")
    if Hq // Hkv > 16:
        raise ValueError(f"{what}: at most 16 query heads per KV head")
    if v_cache.shape != k_cache.shape or v_cache.dtype != q.dtype or \
            not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError(f"{what}: caches must be contiguous (B, Hkv, C, D) in q's dtype")
    kp, vp, wp, pp = k_cache.data_ptr(), v_cache.data_ptr(), weights.data_ptr(), positions.data_ptr()
    if kp % 16 or vp % 16:
        raise ValueError(f"{what}: caches must be 16-byte aligned")
    for t in (k_new, v_new):
        if t.shape != (B, Hkv, 1, D) or t.dtype != q.dtype:
            raise ValueError(f"{what}: k_new and v_new must be (B, Hkv, 1, D) in q's dtype")
    if weights.dtype != torch.float32 or weights.shape != (B, Hkv, C) or not weights.is_contiguous():
        raise ValueError(f"{what}: weights must be contiguous float32 (B, Hkv, C)")
    if positions.dtype != torch.int32 or positions.shape != (B, Hkv, C) or \
            not positions.is_contiguous():
        raise ValueError(f"{what}: positions must be contiguous int32 (B, Hkv, C)")
    lengths, pos = _int32(lengths, (B,), "lengths"), _int32(pos, (B,), "pos")
    if recent < 0 or sink < 0 or recent + sink >= C:
        raise ValueError(f"{what}: sink + recent must leave an entry of the cache to evict")
    if B > 0 and (kp == vp or wp == pp or k_new.data_ptr() in (kp, vp) or v_new.data_ptr() in (kp, vp)):
        raise ValueError(f"{what}: caches, weights, positions and the new rows share memory")
    out = _out(what, out, q, out_dtype, k_new, v_new, k_cache, v_cache, weights, positions)
    if B == 0:
        return out
    q, k_new, v_new = _rows(q), _rows(k_new), _rows(v_new)
    a = N.LaEvictDecodeArgs(
        q.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), kp, vp, wp, pp, lengths.data_ptr(), pos.data_ptr(),
        out.data_ptr(), None, 0,
        B, Hq, Hkv, C, D, *q.stride()[:2], *k_new.stride()[:2], *v_new.stride()[:2], *out.stride()[:2], recent,
        sink, _scale(scale, D), N.dtype_code(q.dtype), N.dtype_code(out.dtype), 0)
    L, ref = N.load(), ctypes.byref(a)
    with N.on_device(dev):
        nbytes = L.la_evict_decode_workspace(ref)
        if nbytes:
            ws = N.workspace(nbytes, dev)
            a.workspace, a.ws_bytes = ws.data_ptr(), nbytes
        N.check(L.la_evict_decode(ref, N.stream_handle(dev)), what)
    return out
