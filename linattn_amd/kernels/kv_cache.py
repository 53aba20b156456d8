"""Paged KV cache maintenance on gfx950: append with Quest page bounds.

``paged_kv_append`` writes the new keys / values of a decode (or chunked
prefill) step into a paged pool and, in the same kernel, folds them into the
Quest page bounds -- the KV concatenation of AttentionVariant.push_kv
(core.py:219-220) plus QuestAttention._refresh_pages (variants/selection.py:
181-201) -- so that a serving loop needs no recompute pass over touched
pages.  For an fp8 pool the codec of kv/quant.py:76-93 (per-token scales,
group = head_dim) runs in the same kernel.  Sequences may sit at different
positions (ragged batches).

``rotary_kv_append`` does this for whole prompts, chunks and single tokens together, and
turns the new queries and keys by their rotary positions on the way.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from linattn_amd import _native as N
from linattn_amd.kernels.block_sparse import _paged_scale_stride
from linattn_amd.kernels.dense import _cu, _pools, _table
from linattn_amd.kernels.rotary import _TYPES, _frequencies, _out_rows, _positions, _strides, _unit_rows

__all__ = ["paged_kv_append", "rotary_kv_append"]

_pack, _library = N.by_bytes(N.LaRotaryAppendArgs, "la_rotary_append")


def paged_kv_append(k_new: torch.Tensor, v_new: torch.Tensor, k_pool: torch.Tensor,
                    v_pool: torch.Tensor, page_table: torch.Tensor, positions: torch.Tensor, *,
                    page_min: Optional[torch.Tensor] = None,
                    page_max: Optional[torch.Tensor] = None, page_size: Optional[int] = None,
                    k_scale: Optional[torch.Tensor] = None,
                    v_scale: Optional[torch.Tensor] = None) -> None:
    """Append (B, Hkv, Tn, D) keys / values at per-sequence ``positions`` (B,).

    Token t of sequence b goes to slot t % pool_page of physical page
    ``page_table[b, t // pool_page]`` of the pools (n_phys, Hkv, pool_page, D).
    With ``page_min`` / ``page_max`` (B, Hkv, n_pages, D) in the key dtype (as
    ``page_update_hip`` returns them) the bounds of every Quest page of
    ``page_size`` tokens that the new tokens touch are updated in place; for an
    append at the end of each sequence the result equals ``page_update_hip``
    over the grown cache bit for bit.  An fp8 (``torch.float8_e4m3fn``) pool
    takes ``k_scale`` / ``v_scale`` (n_phys, Hkv, pool_page) fp32 (contiguous,
    or the interleaved halves of ``fp8_scale_pairs``) and stores
    codes = e4m3(x / scale), scale = max(|x|, 1e-8) / 448 per token (no page
    bounds for fp8 pools).  Runs on the current stream; inputs are not
    modified."""
    dev = N.require_gpu(k_new, v_new, k_pool, v_pool, page_table, positions,
                        page_min, page_max, k_scale, v_scale, what="paged_kv_append")
    if k_new.dim() != 4 or v_new.shape != k_new.shape or k_new.stride() != v_new.stride():
        raise ValueError("k_new / v_new must be (B, Hkv, Tn, D) with equal shapes and strides")
    if k_new.dtype != v_new.dtype or k_new.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("k_new / v_new must both be float32 or bfloat16")
    B, Hkv, Tn, D = k_new.shape
    if k_new.stride(3) != 1:
        raise ValueError("k_new / v_new rows must be contiguous")
    if k_pool.dim() != 4 or v_pool.shape != k_pool.shape or k_pool.shape[1] != Hkv \
            or k_pool.shape[3] != D:
        raise ValueError("pools must be (n_phys, Hkv, pool_page, D) matching k_new")
    if not (k_pool.is_contiguous() and v_pool.is_contiguous()):
        raise ValueError("pools must be contiguous")
    if k_pool.dtype != v_pool.dtype:
        raise ValueError("k_pool / v_pool dtype mismatch")
    fp8 = k_pool.dtype == torch.float8_e4m3fn
    if not fp8 and k_pool.dtype != k_new.dtype:
        raise ValueError("the pool stores k_new's dtype (or float8_e4m3fn codes)")
    n_phys, _, pool_page, _ = k_pool.shape
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != B \
            or page_table.stride(1) != 1:
        raise ValueError("page_table must be int32 (B, pages) with unit column stride")
    if positions.dtype != torch.int32 or positions.shape != (B,) or not positions.is_contiguous():
        raise ValueError("positions must be contiguous int32 (B,)")
    a = N.LaKvAppendArgs()
    a.k_new, a.v_new = k_new.data_ptr(), v_new.data_ptr()
    a.k_pool, a.v_pool = k_pool.data_ptr(), v_pool.data_ptr()
    if fp8:
        for s in (k_scale, v_scale):
            if s is None or s.dtype != torch.float32:
                raise ValueError("fp8 pools need fp32 k_scale / v_scale (n_phys, Hkv, pool_page)")
        if k_scale.stride() != v_scale.stride():
            raise ValueError("k_scale / v_scale must share strides")
        a.s_stride = _paged_scale_stride(k_scale, k_pool)
        a.k_scale, a.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
    a.page_table, a.positions = page_table.data_ptr(), positions.data_ptr()
    if (page_min is None) != (page_max is None):
        raise ValueError("pass both page_min and page_max, or neither")
    if page_min is not None:
        if fp8:
            raise ValueError("fp8 pools take no page bounds")
        if page_size is None or page_size <= 0:
            raise ValueError("page bounds need page_size")
        P = page_min.shape[2] if page_min.dim() == 4 else -1
        if page_min.shape != (B, Hkv, P, D) or page_max.shape != page_min.shape \
                or page_min.stride() != page_max.stride():
            raise ValueError("page_min / page_max must be (B, Hkv, n_pages, D) with equal strides")
        if page_min.dtype != k_new.dtype or page_max.dtype != k_new.dtype:
            raise ValueError("page bounds are stored in the key dtype")
        a.page_min, a.page_max = page_min.data_ptr(), page_max.data_ptr()
        a.meta_page, a.n_pages = int(page_size), P
        a.m_sb, a.m_sh, a.m_sp, a.m_sd = page_min.stride()
    a.B, a.Hkv, a.Tn, a.D = B, Hkv, Tn, D
    a.n_sb, a.n_sh, a.n_st = k_new.stride(0), k_new.stride(1), k_new.stride(2)
    a.n_phys, a.pool_page = n_phys, pool_page
    a.pt_sb, a.pt_pages = page_table.stride(0), page_table.shape[1]
    a.in_dtype = N.dtype_code(k_new.dtype)
    a.pool_dtype = N.dtype_code(k_pool.dtype)
    N.check(N.load().la_paged_kv_append(ctypes.byref(a), N.stream_handle(dev)), "paged_kv_append")


def rotary_kv_append(q: Optional[torch.Tensor], k_new: torch.Tensor, v_new: torch.Tensor, k_pool: torch.Tensor,
                     v_pool: torch.Tensor, page_table: torch.Tensor, positions: torch.Tensor,
                     inv_freq: torch.Tensor, *, cu_seqlens: Optional[torch.Tensor] = None,
                     rotary_positions: Optional[torch.Tensor] = None, axes: Optional[torch.Tensor] = None,
                     interleaved: bool = False, q_out: Optional[torch.Tensor] = None,
                     page_min: Optional[torch.Tensor] = None, page_max: Optional[torch.Tensor] = None,
                     page_size: Optional[int] = None, k_scale: Optional[torch.Tensor] = None,
                     v_scale: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Turns the queries and keys of new tokens by their rotary positions and stores the keys
    and their values in the pages of their sequences; returns the turned queries.

    q (B, Hq, Tn, D), k_new / v_new (B, Hkv, Tn, D), or packed (N, H, D) with ``cu_seqlens``
    (int32 (B + 1,), ascending, on the device): sequence b's tokens are rows cu_seqlens[b] ..
    cu_seqlens[b + 1] - 1, none to many; q may be None.  bfloat16, float16 or float32.
    New token i of sequence b goes to place ``positions[b]`` + i (int32 (B,)), that is to slot
    place % pool_page of page ``page_table[b, place // pool_page]`` of the pools (n_phys, Hkv,
    pool_page, D); a token whose place lies outside of the table, or whose page outside of the
    pool, is not stored.  The pools hold k_new's dtype, or float8_e4m3fn codes with ``k_scale`` /
    ``v_scale`` (as ``paged_kv_append``; codes are of the row as it was turned in fp32; of D above
    128 only where D, n and all rows are whole fours of values, and pools begin at whole fours).
    Angles: ``inv_freq``, ``axes`` and ``interleaved`` as in ``rotary``, by the tokens' places, or by
    ``rotary_positions`` (int32, (B, Tn) or (N,); with ``axes`` (A, B, Tn) or (A, N)).
    ``page_min`` / ``page_max`` (B, Hkv, n_pages, D) in k_new's dtype, with ``page_size``: Quest's
    bounds of the pages that the new tokens touch are kept as in ``paged_kv_append`` (the keys
    as they are stored).  Queries go to a new tensor (rows of no sequence are zeros), or to
    ``q_out`` (those rows are left), which may be q itself.  Forward only."""
    what = "rotary_kv_append"
    dev = N.require_gpu(k_new, v_new, q, k_pool, v_pool, page_table, positions, inv_freq, cu_seqlens,
                        rotary_positions, axes, q_out, page_min, page_max, k_scale, v_scale, what=what)
    packed, shape, dtype = cu_seqlens is not None, k_new.shape, k_new.dtype
    if len(shape) != (3 if packed else 4) or v_new.shape != shape:
        raise ValueError(f"{what}: k_new / v_new must be (B, Hkv, Tn, D), or with cu_seqlens (N, Hkv, D)")
    if dtype not in _TYPES or v_new.dtype != dtype:
        raise ValueError(f"{what}: k_new / v_new must both be bfloat16, float16 or float32")
    Hkv, D, Hq = shape[1], shape[-1], 0
    if Hkv == 0:
        raise ValueError(f"{what}: no KV heads")
    if q is not None:
        qs = q.shape
        if len(qs) != len(shape) or q.dtype != dtype or qs[0] != shape[0] or qs[2:] != shape[2:] or qs[1] % Hkv:
            raise ValueError(f"{what}: q must have k_new's dtype, tokens and head_dim, and a multiple of its heads")
        Hq = qs[1]
    elif q_out is not None:
        raise ValueError(f"{what}: q_out without q")
    if packed:
        cu_seqlens = _cu(cu_seqlens, "cu_seqlens")
        B, T = cu_seqlens.shape[0] - 1, shape[0]
    else:
        B, T = shape[0], shape[2]
    pool, fp8, s_stride = _pools(what, k_pool, v_pool, dtype, Hkv, D, k_scale, v_scale)
    pt_stride, pt_pages = _table(what, page_table, B)
    if positions.dtype != torch.int32 or positions.shape != (B,):
        raise ValueError(f"{what}: positions must be int32 ({B},)")
    n = _frequencies(what, inv_freq, axes, D)
    A, p_s, rp = 1, (0, 0, 0), 0
    if rotary_positions is not None:
        A, p_s = _positions(what, rotary_positions, axes, (T,) if packed else (B, T))
        rp = rotary_positions.data_ptr()
    elif axes is not None:
        raise ValueError(f"{what}: axes need rotary_positions")
    mn = mx = 0
    meta = (0, 0, 0, 0, 0, 0)
    if page_min is not None and page_max is not None:
        if fp8:
            raise ValueError(f"{what}: fp8 pools take no page bounds")
        if page_size is None or not 0 < int(page_size) < 1 << 30:
            raise ValueError(f"{what}: page bounds need page_size")
        ms, m_s = page_min.shape, page_min.stride()
        if len(ms) != 4 or ms[0] != B or ms[1] != Hkv or ms[3] != D or page_max.shape != ms or page_max.stride() != m_s:
            raise ValueError(f"{what}: page_min / page_max must be (B, Hkv, n_pages, D) with equal strides")
        if page_min.dtype != dtype or page_max.dtype != dtype:
            raise ValueError(f"{what}: page bounds are stored in the key dtype")
        if ms[2] > 0:
            mn, mx, meta = page_min.data_ptr(), page_max.data_ptr(), (int(page_size), ms[2], *m_s)
    elif page_min is not None or page_max is not None:
        raise ValueError(f"{what}: pass both page_min and page_max, or neither")
    elif page_size is not None:
        raise ValueError(f"{what}: page_size is for page bounds")
    zero_rest = q_out is None
    if q is not None:
        q_out = _out_rows(what, "q_out", q_out, q)
    if B == 0 or T == 0:
        return q_out
    k_new, v_new, inv_freq, positions = _unit_rows(k_new), _unit_rows(v_new), inv_freq.contiguous(), positions.contiguous()
    axes = None if axes is None else axes.contiguous()
    qp = qo = 0
    q_s = o_s = (0, 0, 0)
    if Hq:
        q = _unit_rows(q)
        qp, qo, q_s, o_s = q.data_ptr(), q_out.data_ptr(), _strides(q), _strides(q_out)
    a = _pack(qp, k_new.data_ptr(), v_new.data_ptr(), qo, k_pool.data_ptr(), v_pool.data_ptr(),
              k_scale.data_ptr() if fp8 else 0, v_scale.data_ptr() if fp8 else 0, page_table.data_ptr(),
              positions.data_ptr(), cu_seqlens.data_ptr() if packed else 0, rp, inv_freq.data_ptr(),
              0 if axes is None else axes.data_ptr(), mn, mx, B, T, Hq, Hkv, D, n, A, *q_s, *_strides(k_new),
              *_strides(v_new), *o_s, *p_s, pool[0], pool[2], pt_stride, pt_pages, s_stride, *meta,
              N.dtype_code(dtype), N.dtype_code(k_pool.dtype), interleaved, zero_rest)
    run, = _library()
    with N.on_device(dev):
        N.check(run(a, N.stream_handle(dev)), what)
    return q_out
