"""Memory that an output shares with an input, in any layout, is refused by the library before
it touches a GPU; views that interleave without a common byte are not.  The addresses are
made up: a call that is not refused ends at the workspace it lacks."""

from __future__ import annotations

import ctypes
import random

import numpy as np
import pytest

from linattn_amd import _native as N

BASE = 1 << 40
FAR = 1 << 36  # from one tensor to the next that is meant to be apart


def _bytes(at, run, dims):
    """The 16-byte units of runs of `run` bytes from `at` on, dims of (stride in bytes, count)."""
    x = np.arange(at // 16, (at + run) // 16)
    for stride, count in dims:
        x = (x[None] + (np.arange(count) * (stride // 16))[:, None]).ravel()
    return set(x.tolist())


def _dense(out, o, k, ks, Tk=512, Tq=2, B=2, H=2):
    """A call of fp32 tensors at addresses out and k with strides o and ks (values), D = 64."""
    a = N.LaDenseAttnArgs()
    a.B, a.Hq, a.Hkv, a.Tq, a.Tk, a.D, a.scale, a.dtype, a.out_dtype = B, H, H, Tq, Tk, 64, 0.1, N.LA_F32, N.LA_F32
    a.q, a.k, a.v, a.out = BASE + FAR, k, BASE + 2 * FAR, out
    a.q_sb, a.q_sh, a.q_st = H * Tq * 64, Tq * 64, 64
    a.v_sb, a.v_sh, a.v_st = H * Tk * 64, Tk * 64, 64
    (a.o_sb, a.o_sh, a.o_st), (a.k_sb, a.k_sh, a.k_st) = o, ks
    rc = N.load().la_dense_attention(ctypes.byref(a), None)
    assert rc in (N.LA_ERR_WORKSPACE, N.LA_ERR_INVALID)
    assert rc == N.LA_ERR_WORKSPACE or b"shares memory" in N.load().la_last_error()
    return rc == N.LA_ERR_INVALID


@pytest.mark.parametrize("seed", range(6))
def test_any_strides(seed):
    """Against the sets of what both cover."""
    r = random.Random(seed)
    seen = [0, 0]
    for _ in range(150):
        Tk, pad = 512, 4 * r.randint(0, 40)
        row = 64 + pad  # keys in rows with gaps, heads side by side, behind one another or apart
        heads = r.choice([(row, 2 * row), (row * Tk, row), (row * Tk + 4 * r.randint(0, 99), row)])
        ks = (2 * row * Tk + 4 * r.randint(0, 99), *heads)
        o = r.choice([ks, (ks[0], ks[1], ks[2] * r.randint(1, 3)), (4 * r.randint(16, 9999), 4 * r.randint(16, 999), 4 * r.randint(16, 99))])
        at = BASE + 16 * r.choice([r.randint(-300, 300), r.randint(-2 * row * Tk // 4, row * Tk)])
        covers = [_bytes(p, 256, [(4 * s[0], 2), (4 * s[1], 2), (4 * s[2], n)]) for p, s, n in ((at, o, 2), (BASE, ks, Tk))]
        want = bool(covers[0] & covers[1])
        assert _dense(at, o, BASE, ks) == want, (at - BASE, o, ks)
        seen[want] += 1
    assert min(seen) > 10


def test_slices_of_one_buffer():
    """Columns of one buffer: the output beside the keys, and over half of them."""
    s = (2 * 512 * 128, 512 * 128, 128)
    assert not _dense(BASE + 4 * 64, s, BASE, s)
    assert _dense(BASE + 4 * 8, s, BASE, s) and _dense(BASE + 4 * 124, s, BASE, s)
    s = (512 * 6 * 64, 64, 6 * 64)  # heads of the queries, keys and values of a token side by side
    assert not _dense(BASE, s, BASE + 4 * 2 * 64, s) and _dense(BASE, s, BASE + 4 * 64, s)


def _step(**change):
    a, C, D, B, H, G = N.LaEvictDecodeArgs(), 9, 64, 2, 2, 2
    a.B, a.Hq, a.Hkv, a.C, a.D, a.scale, a.dtype, a.out_dtype = B, H * G, H, C, D, 0.1, N.LA_F32, N.LA_F32
    for i, n in enumerate(("q", "k_new", "v_new", "k", "v", "weights", "positions", "lengths", "pos", "out")):
        setattr(a, n, BASE + i * FAR)
    a.q_sb, a.q_sh = a.o_sb, a.o_sh = H * G * D, D
    a.kn_sb, a.kn_sh = a.vn_sb, a.vn_sh = H * D, D
    for n, x in change.items():
        setattr(a, n, x(a) if callable(x) else x)
    rc = N.load().la_evict_decode(ctypes.byref(a), None)
    assert rc == N.LA_ERR_WORKSPACE or (rc == N.LA_ERR_INVALID and b"share memory" in N.load().la_last_error())
    return rc == N.LA_ERR_INVALID


def test_decode_step():
    """Caches that are slices of one buffer and overlap, rows of the new token, bookkeeping."""
    size = 2 * 2 * 9 * 64 * 4
    assert not _step()
    assert _step(v=lambda a: a.k + size // 2) and _step(v=lambda a: a.k - size + 16) and not _step(v=lambda a: a.k + size)
    assert _step(weights=lambda a: a.v + 64) and _step(positions=lambda a: a.weights + 4 * 2 * 2 * 9 - 4)
    assert not _step(positions=lambda a: a.weights + 4 * 2 * 2 * 9)
    assert _step(k_new=lambda a: a.k + size - 256) and _step(v_new=lambda a: a.k + 64 * 4)
    assert _step(lengths=lambda a: a.positions + 8) and _step(pos=lambda a: a.weights)
    assert _step(out=lambda a: a.q) and _step(out=lambda a: a.v_new + 256) and _step(q=lambda a: a.v)
    # q, k_new and v_new beside one another in the rows of one buffer, and the output there
    width = 64 * 8
    fused = dict(k_new=lambda a: a.q + 4 * 4 * 64, v_new=lambda a: a.q + 4 * 6 * 64, q_sb=width, kn_sb=width, vn_sb=width)
    assert not _step(**fused)
    assert not _step(**fused, out=lambda a: a.q + 4 * 8 * 64 * 2)
    assert _step(**fused, out=lambda a: a.q + 4 * 7 * 64, o_sb=width)


def test_key_weights():
    def call(out, lse=BASE + 4 * FAR, sb=2 * 600, sh=600):
        a = N.LaKeyWeightsArgs()
        a.B, a.Hq, a.Hkv, a.Tq, a.Tk, a.D, a.scale, a.dtype = 2, 2, 2, 600, 600, 64, 0.1, N.LA_F32
        a.q, a.k, a.lse, a.out = BASE, BASE + FAR, lse, out
        a.q_sb, a.q_sh, a.q_st = a.k_sb, a.k_sh, a.k_st = 2 * 600 * 64, 600 * 64, 64
        a.l_sb, a.l_sh, a.w_sb, a.w_sh = sb, 600, sb, sh
        rc = N.load().la_key_weights(ctypes.byref(a), None)
        assert rc == N.LA_ERR_WORKSPACE or (rc == N.LA_ERR_INVALID and b"shares memory" in N.load().la_last_error())
        return rc == N.LA_ERR_INVALID

    at = BASE + 3 * FAR
    assert not call(at) and call(BASE + 640) and call(BASE + FAR - 16) and call(at, lse=at + 4 * 600)
    assert not call(at, lse=at + 4 * 2400)
    assert not call(at, lse=at + 4 * 1200, sb=2400) and call(at, lse=at + 4 * 600, sb=2400)
