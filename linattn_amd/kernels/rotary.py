"""Rotary positions on gfx950, on one axis or on several (time, height and width of a video).

``rotary`` turns the rows of q and k by their tokens' positions before
``linattn_amd.kernels.dense`` or ``linattn_amd.kernels.prefill`` attends over them;
``linattn_amd.kernels.kv_cache.rotary_kv_append`` does it on the way into a paged cache.
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch

from linattn_amd import _native as N
from linattn_amd.kernels.dense import _apart

__all__ = ["rotary", "rotary_axes"]

_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def rotary_axes(sections: Sequence[int], interleaved: bool = False,
                device: Optional[torch.device] = None) -> torch.Tensor:
    """Which axis each frequency goes by, int32: ``sections[a]`` frequencies on axis a, one
    section behind the other, or the axes in turn, as long as each has some left."""
    if not sections or any(int(s) != s or s < 0 for s in sections) or sum(sections) == 0:
        raise ValueError(f"sections must be whole numbers that are not negative, got {sections}")
    if not interleaved:
        axes = [a for a, s in enumerate(sections) for _ in range(int(s))]
    else:
        axes = [a for i in range(int(max(sections))) for a, s in enumerate(sections) if i < s]
    return torch.tensor(axes, dtype=torch.int32, device=device)


_pack, _library = N.by_bytes(N.LaRotaryArgs, "la_rotary")


def _unit_rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride()[-1] == 1 or t.shape[-1] == 1 else t.contiguous()


def _frequencies(what: str, inv_freq: torch.Tensor, axes: Optional[torch.Tensor], D: int) -> int:
    """How many there are, checked."""
    shape = inv_freq.shape
    if inv_freq.dtype != torch.float32 or len(shape) != 1 or not 0 < 2 * shape[0] <= D <= 512:
        raise ValueError(f"{what}: inv_freq must be float32 (n,) with 2 n <= head_dim <= 512")
    if axes is not None and (axes.dtype != torch.int32 or axes.shape != shape):
        raise ValueError(f"{what}: axes must be int32 with an entry for each frequency")
    return shape[0]


def _positions(what: str, positions: torch.Tensor, axes: Optional[torch.Tensor],
               tokens: Tuple[int, ...]) -> Tuple[int, Tuple[int, int, int]]:
    """(axes, strides by axis, sequence and token) of positions (*tokens) or (A, *tokens)."""
    if positions.dtype != torch.int32:
        raise ValueError(f"{what}: positions must be int32")
    shape, st = positions.shape, positions.stride()
    if axes is None:
        if shape != tokens:
            raise ValueError(f"{what}: positions must be {tokens} (with several axes, pass `axes`), got {tuple(shape)}")
        return 1, (0, *st) if len(st) == 2 else (0, 0, st[0])
    if len(shape) != len(tokens) + 1 or shape[1:] != tokens or shape[0] == 0:
        raise ValueError(f"{what}: positions must be (axes, {', '.join(map(str, tokens))}), got {tuple(shape)}")
    return shape[0], st if len(st) == 3 else (st[0], 0, st[1])


def _out_rows(what: str, name: str, out: Optional[torch.Tensor], x: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty_like(x, memory_format=torch.contiguous_format)
    if out.shape != x.shape or out.dtype != x.dtype or (out.shape[-1] > 1 and out.stride(-1) != 1):
        raise ValueError(f"{what}: {name} must have its input's shape and dtype, and contiguous rows")
    if out.data_ptr() != x.data_ptr():
        _apart(what, out, x)
    elif any(s == 0 and d > 1 for s, d in zip(out.stride(), out.shape)):
        raise ValueError(f"{what}: {name} holds some of its rows twice")
    elif out is x:
        return out
    elif out.numel() and any(a != b for a, b, d in zip(out.stride(), x.stride(), x.shape) if d > 1):
        raise ValueError(f"{what}: {name} shares memory with its input, but does not hold the same rows")
    return out


def _strides(t: torch.Tensor) -> Tuple[int, int, int]:
    """(sequence, head, token) of (B, H, T, D), or packed (T, H, D)."""
    s = t.stride()
    return s[:3] if len(s) == 4 else (0, s[1], s[0])


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor, *,
           axes: Optional[torch.Tensor] = None, interleaved: bool = False, inverse: bool = False,
           q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None
           ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """The rows of q and k turned by their tokens' positions.

    q (B, Hq, T, D) and k (B, Hkv, T, D), or packed (N, Hq, D) and (N, Hkv, D), bfloat16,
    float16 or float32, D up to 512; k may be None.  ``inv_freq`` (float32 (n,), 2 n <= D):
    frequency i turns the pair (i, n + i) of a row, or with ``interleaved`` (2 i, 2 i + 1), by
    the angle position * inv_freq[i]; what is behind the first 2 n values is copied.
    ``positions`` (int32) is (B, T) or (N,); with ``axes`` (int32 (n,), see ``rotary_axes``) it
    is (A, B, T) or (A, N), and frequency i goes by positions[axes[i]].  ``inverse`` turns back:
    the gradient of a turn is the turn back of its output's gradient (no gradient is recorded).
    Angles are counted in 64 bits, so far positions keep their phase; rows are turned in 32 and
    rounded once.  Returns new tensors (q alone where k is None), or ``q_out`` / ``k_out``, which
    may be q and k themselves (in place)."""
    what = "rotary"
    dev = N.require_gpu(q, k, positions, inv_freq, axes, q_out, k_out, what=what)
    shape, dtype = q.shape, q.dtype
    batched = len(shape) == 4
    if not (batched or len(shape) == 3) or dtype not in _TYPES:
        raise ValueError(f"{what}: q must be (B, Hq, T, D) or (N, Hq, D) in bfloat16, float16 or float32")
    B, Hq, T, D = shape if batched else (1, shape[1], shape[0], shape[2])
    Hkv = 0
    if k is not None:
        ks = k.shape
        if len(ks) != len(shape) or k.dtype != dtype or ks[0] != shape[0] or ks[2:] != shape[2:]:
            raise ValueError(f"{what}: k must have q's dtype, tokens and head_dim")
        Hkv = ks[1]
    elif k_out is not None:
        raise ValueError(f"{what}: k_out without k")
    n = _frequencies(what, inv_freq, axes, D)
    A, p_s = _positions(what, positions, axes, (B, T) if batched else (T,))
    q_out = _out_rows(what, "q_out", q_out, q)
    if k is not None:
        k_out = _out_rows(what, "k_out", k_out, k)
    if B * T * (Hq + Hkv) * D > 0:
        q, inv_freq = _unit_rows(q), inv_freq.contiguous()
        axes = None if axes is None else axes.contiguous()
        kp = ko = 0
        k_s = ko_s = (0, 0, 0)
        if Hkv:
            k = _unit_rows(k)
            kp, ko, k_s, ko_s = k.data_ptr(), k_out.data_ptr(), _strides(k), _strides(k_out)
        if Hq == 0:  # (the rows of k alone)
            rotary(k, None, positions, inv_freq, axes=axes, interleaved=interleaved, inverse=inverse, q_out=k_out)
            return q_out, k_out
        a = _pack(q.data_ptr(), kp, q_out.data_ptr(), ko, positions.data_ptr(), inv_freq.data_ptr(),
                  0 if axes is None else axes.data_ptr(), B, T, Hq, Hkv, D, n, A, *_strides(q), *k_s, *_strides(q_out),
                  *ko_s, *p_s, N.dtype_code(dtype), interleaved, inverse, 0)
        run, = _library()
        with N.on_device(dev):
            N.check(run(a, N.stream_handle(dev)), what)
    return q_out if k is None else (q_out, k_out)
