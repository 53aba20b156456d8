"""Calls of more threads than a launch may have (2^32) are refused, not handed to the device.
The addresses are made up: nothing is launched."""

from __future__ import annotations

import ctypes

import pytest

from linattn_amd import _native as N

BASE, FAR = 1 << 44, 1 << 40


@pytest.mark.parametrize("B,Hkv,Tq,Tk", [(1 << 21, 8, 1, 1), (1 << 20, 8, 130, 1)])
def test_dense_attention(B, Hkv, Tq, Tk):
    a = N.LaDenseAttnArgs()
    a.B, a.Hq, a.Hkv, a.Tq, a.Tk, a.D, a.scale, a.dtype, a.out_dtype = B, Hkv, Hkv, Tq, Tk, 64, 0.1, N.LA_BF16, N.LA_BF16
    a.q, a.k, a.v, a.out = (BASE + i * FAR for i in range(4))
    a.q_sb, a.q_sh, a.q_st = a.o_sb, a.o_sh, a.o_st = Hkv * Tq * 64, Tq * 64, 64
    a.k_sb, a.k_sh, a.k_st = a.v_sb, a.v_sh, a.v_st = Hkv * Tk * 64, Tk * 64, 64
    assert N.load().la_dense_attention(ctypes.byref(a), None) == N.LA_ERR_INVALID
    assert b"too many" in N.load().la_last_error()


def test_key_weights():
    a = N.LaKeyWeightsArgs()
    a.B, a.Hq, a.Hkv, a.Tq, a.Tk, a.D, a.scale, a.dtype = 1 << 21, 8, 8, 1, 1, 64, 0.1, N.LA_F32
    a.q, a.k, a.lse, a.out = (BASE + i * FAR for i in range(4))
    a.q_sb, a.q_sh, a.q_st = a.k_sb, a.k_sh, a.k_st = 8 * 64, 64, 64
    a.l_sb, a.l_sh, a.w_sb, a.w_sh = 8, 1, 8, 1
    assert N.load().la_key_weights(ctypes.byref(a), None) == N.LA_ERR_INVALID
    assert b"too many" in N.load().la_last_error()


@pytest.mark.parametrize("B,T,budget,capacity", [
    (1 << 20, 4, 4, 64 * 16),              # one kernel: 2^24 workgroups of 256 threads
    (1 << 10, 4096, 100, 64 * 4100),       # slots beside the selecting workgroups, of 1024 threads
    (1 << 18, 4096, 4096, 4096),           # chosen slots
    (1 << 14, 20000, 100, 64 * (1 << 12)),  # slices
])
def test_evict_kv(B, T, budget, capacity):
    a = N.LaEvictArgs()
    a.B, a.Hkv, a.T, a.D, a.esize, a.budget, a.capacity = B, 1, T, 8, 2, budget, capacity
    a.k, a.v, a.weights, a.k_out, a.v_out, a.w_out, a.pos_out, a.len_out = (BASE + i * FAR for i in range(8))
    a.k_sb, a.k_sh, a.k_st = a.v_sb, a.v_sh, a.v_st = T * 8, T * 8, 8
    a.w_sb, a.w_sh = T, T
    a.ws_bytes = N.load().la_evict_kv_workspace(ctypes.byref(a))
    a.workspace = BASE + 9 * FAR
    assert N.load().la_evict_kv(ctypes.byref(a), None) == N.LA_ERR_INVALID
    assert b"too many" in N.load().la_last_error()
