"""What ``la_rotary``, ``la_rotary_append`` and ``la_paged_attention`` write shares no memory with itself or
with anything else that they read or write: refused before anything is launched.  The addresses
are made up; calls whose memory is apart end at something else that they lack."""

from __future__ import annotations

import ctypes

import pytest

from linattn_amd import _native as N

BASE, FAR = 1 << 40, 1 << 32


def _said(fn, a):
    lib = N.load()
    rc = getattr(lib, fn)(ctypes.byref(a), None)
    assert rc in (N.LA_ERR_INVALID, N.LA_ERR_UNSUPPORTED, N.LA_ERR_WORKSPACE), (rc, lib.la_last_error())
    return lib.la_last_error().decode()


# ------------------------------------------------------------- page bounds ----
B, HKV, P, D, PAGES = 2, 2, 5, 64, 6 * 2 * 16  # PAGES: rows of the pools


def _append(minor=False):
    """An fp32 call with page bounds, pages (or dims) side by side, whose k_new is not aligned: what
    is refused for nothing else is refused for that."""
    a = N.LaRotaryAppendArgs()
    names = ("q", "k_new", "v_new", "q_out", "k_pool", "v_pool", "page_table", "positions", "inv_freq", "page_min", "page_max")
    at = {name: BASE + i * FAR for i, name in enumerate(names)}
    for name, x in at.items():
        setattr(a, name, x)
    a.k_new += 2
    a.B, a.T, a.Hq, a.Hkv, a.D, a.n, a.A = B, 8, 4, HKV, D, 32, 1
    a.q_sb, a.q_sh, a.q_st = a.o_sb, a.o_sh, a.o_st = 2048, 512, 64
    a.kn_sb, a.kn_sh, a.kn_st = a.vn_sb, a.vn_sh, a.vn_st = 1024, 512, 64
    a.n_phys, a.pool_page, a.pt_sb, a.pt_pages, a.s_stride = 6, 16, 4, 4, 1
    a.meta_page, a.n_pages = 16, P
    a.m_sb, a.m_sh, a.m_sp, a.m_sd = (HKV * P * D, P * D, 1, P) if minor else (HKV * P * D, P * D, D, 1)
    return a, at


@pytest.mark.parametrize("minor", [False, True])
def test_page_bounds_apart(minor):
    a, at = _append(minor)
    assert "unaligned" in _said("la_rotary_append", a)
    # halves of one buffer, value by value, page by page, and one behind the other
    size = 4 * B * HKV * P * D
    a.page_max = a.page_min + size
    assert "unaligned" in _said("la_rotary_append", a)
    a, at = _append(minor)
    a.m_sb, a.m_sh, a.m_sp, a.m_sd = (2 * x for x in (a.m_sb, a.m_sh, a.m_sp, a.m_sd))
    a.page_max = a.page_min + 4
    assert "unaligned" in _said("la_rotary_append", a)
    a, at = _append()
    a.m_sb, a.m_sh, a.m_sp = 2 * a.m_sb, 2 * a.m_sh, 2 * a.m_sp
    a.page_max = a.page_min + 4 * D
    assert "unaligned" in _said("la_rotary_append", a)


@pytest.mark.parametrize("minor", [False, True])
@pytest.mark.parametrize("change", [
    lambda a, at: dict(page_max=at["page_min"]),
    lambda a, at: dict(page_max=at["page_min"] + 4 * B * HKV * P * D - 4),
    lambda a, at: dict(page_max=at["page_min"] - 4),
    lambda a, at: dict(page_min=at["k_pool"] + PAGES * D * 4 - 4),
    lambda a, at: dict(page_max=at["v_pool"]),
    lambda a, at: dict(page_min=at["q_out"] + 256),
    lambda a, at: dict(page_max=at["q"]),
    lambda a, at: dict(page_min=at["k_new"] + 4096),
    lambda a, at: dict(page_max=at["v_new"]),
    lambda a, at: dict(page_min=at["page_table"]),
    lambda a, at: dict(page_max=at["positions"]),
    lambda a, at: dict(page_max=at["inv_freq"] + 31 * 4),
    lambda a, at: dict(m_sb=0),                     # rows held twice
    lambda a, at: dict(m_sh=0),
    lambda a, at: dict(m_sp=0),
    lambda a, at: dict(m_sd=0),
    lambda a, at: dict(m_sb=a.m_sh),
])
def test_page_bounds_over_others(minor, change):
    a, at = _append(minor)
    for name, x in change(a, at).items():
        setattr(a, name, x)
    assert "shares memory" in _said("la_rotary_append", a)


def test_what_else_an_append_writes():
    for change in (dict(k_pool="page_table"), dict(v_pool="positions"), dict(q_out="inv_freq"), dict(v_pool="k_pool")):
        a, at = _append()
        for name, of in change.items():
            setattr(a, name, at[of])
        assert "shares memory" in _said("la_rotary_append", a), change
    for extra in ("cu", "axes", "rot_positions"):
        a, at = _append()
        a.p_sb, a.p_st = 8, 1
        setattr(a, extra, at["k_pool"] + 64)
        assert "shares memory" in _said("la_rotary_append", a), extra
    for name in ("o_sb", "o_sh", "o_st"):  # rows of q_out held twice, in place too
        for place in ("q_out", "q"):
            a, at = _append()
            a.q_out = at[place]
            setattr(a, name, 0)
            setattr(a, name.replace("o_", "q_"), 0)
            assert "shares memory" in _said("la_rotary_append", a), (name, place)
    a, at = _append()
    a.q_out = a.q  # (in place)
    assert "unaligned" in _said("la_rotary_append", a)


# --------------------------------------------------------------- attention ----
def _attend(fp8=False):
    """An fp16 call over a cache of 6 pages, which ends at its workspace."""
    a = N.LaPagedAttnArgs()
    names = ("q", "k_pool", "v_pool", "out", "lse", "page_table", "lengths", "workspace", "k_scale", "v_scale")
    at = {name: BASE + i * FAR for i, name in enumerate(names)}
    for name, x in at.items():
        if fp8 or not name.endswith("scale"):
            setattr(a, name, x)
    a.B, a.Hq, a.Hkv, a.Tq, a.D = 2, 4, 2, 8, 64
    a.q_sb, a.q_sh, a.q_st = a.o_sb, a.o_sh, a.o_st = 2048, 512, 64
    a.l_sb, a.l_sh = 32, 8
    a.n_phys, a.page, a.pt_sb, a.pt_pages, a.s_stride = 6, 16, 4, 4, 1
    a.scale, a.causal, a.dtype, a.kv_dtype, a.out_dtype = 0.125, 1, N.LA_F16, N.LA_FP8_E4M3 if fp8 else N.LA_F16, N.LA_F16
    return a, at


@pytest.mark.parametrize("change", [
    lambda a, at: dict(out=at["k_scale"] + PAGES * 4 - 16),
    lambda a, at: dict(out=at["v_scale"]),
    lambda a, at: dict(out=at["lse"]),
    lambda a, at: dict(out=at["lengths"]),
    lambda a, at: dict(out=at["page_table"] + 16),
    lambda a, at: dict(lse=at["out"] + 4096),
    lambda a, at: dict(lse=at["q"]),
    lambda a, at: dict(lse=at["k_pool"] + 64),
    lambda a, at: dict(lse=at["v_pool"] + PAGES * 64 - 4),
    lambda a, at: dict(lse=at["k_scale"]),
    lambda a, at: dict(lse=at["v_scale"] + 8),
    lambda a, at: dict(lse=at["page_table"]),
    lambda a, at: dict(lse=at["lengths"]),
    lambda a, at: dict(cu_q=at["lse"], Tq=16),
    lambda a, at: dict(q_len=at["out"]),
    lambda a, at: dict(lse=at["workspace"], ws_bytes=256),
    lambda a, at: dict(workspace=at["q"], ws_bytes=256),
    lambda a, at: dict(workspace=at["out"] + 256, ws_bytes=256),
    lambda a, at: dict(o_sb=0),                     # rows held twice
    lambda a, at: dict(o_sh=0),
    lambda a, at: dict(o_st=0),
    lambda a, at: dict(l_sb=0),
    lambda a, at: dict(l_sh=0),
    lambda a, at: dict(l_sh=7),
])
def test_attention_over_others(change):
    a, at = _attend(True)
    for name, x in change(a, at).items():
        setattr(a, name, x)
    assert "shares memory" in _said("la_paged_attention", a)


@pytest.mark.parametrize("fp8", [False, True])
def test_attention_apart(fp8):
    a, at = _attend(fp8)
    assert "workspace" in _said("la_paged_attention", a)
    a.lse = None
    a.l_sb = a.l_sh = 0
    assert "workspace" in _said("la_paged_attention", a)
    # out beside q, row by row; the halves of the scales' pairs
    a, at = _attend(fp8)
    a.out = a.q + 128
    a.q_sb, a.q_sh, a.q_st = a.o_sb, a.o_sh, a.o_st = 4096, 1024, 128
    if fp8:
        a.s_stride, a.v_scale = 2, a.k_scale + 4
    assert "workspace" in _said("la_paged_attention", a)
    # packed: one row of lse a head
    a, at = _attend(fp8)
    a.cu_q, a.l_sb, a.q_sb, a.o_sb = BASE + 20 * FAR, 0, 0, 0
    assert "workspace" in _said("la_paged_attention", a)


# ------------------------------------------------------------------ rotary ----
def _rotary():
    a = N.LaRotaryArgs()
    names = ("q", "k", "q_out", "k_out", "positions", "inv_freq", "axes")
    at = {name: BASE + i * FAR for i, name in enumerate(names)}
    for name, x in at.items():
        setattr(a, name, x)
    a.B, a.T, a.Hq, a.Hkv, a.D, a.n, a.A = 2, 8, 4, 2, 64, 32, 3
    a.q_sb, a.q_sh, a.q_st = a.qo_sb, a.qo_sh, a.qo_st = 2048, 512, 64
    a.k_sb, a.k_sh, a.k_st = a.ko_sb, a.ko_sh, a.ko_st = 1024, 512, 64
    a.p_sa, a.p_sb, a.p_st = 16, 8, 1
    a.dtype = N.LA_F32
    return a, at


@pytest.mark.parametrize("change", [
    lambda at: dict(q_out=at["positions"] + 188),
    lambda at: dict(k_out=at["positions"] - 256),
    lambda at: dict(q_out=at["inv_freq"]),
    lambda at: dict(k_out=at["axes"] + 124),
    lambda at: dict(q_out=at["k_out"]),
    lambda at: dict(k_out=at["q"] + 4),
    lambda at: dict(qo_sb=0),
    lambda at: dict(qo_sh=0),
    lambda at: dict(qo_st=32),
    lambda at: dict(ko_sb=0),
    lambda at: dict(ko_sh=0),
    lambda at: dict(ko_st=0),
    lambda at: dict(q_out=at["q"], qo_sh=0, q_sh=0),  # (in place)
    lambda at: dict(k_out=at["k"], ko_st=0, k_st=0),
])
def test_rotary_over_others(change):
    a, at = _rotary()
    for name, x in change(at).items():
        setattr(a, name, x)
    assert "shares memory" in _said("la_rotary", a)


@pytest.mark.parametrize("off", [1, 2, 3])
def test_codes_of_unaligned_pools_are_not_written_four_at_a_time(off):
    """Chunks of four 16-bit values (n = 36: rows of 256 have 64 of them) need pools at whole fours."""
    a, at = _append()
    a.page_min = a.page_max = None
    a.k_new -= 2
    a.dtype, a.pool_dtype, a.D, a.n = N.LA_BF16, N.LA_FP8_E4M3, 256, 36
    a.k_scale, a.v_scale = BASE + 20 * FAR, BASE + 21 * FAR
    for s in ("q_s", "o_s", "kn_s", "vn_s"):
        for d in "bht":
            setattr(a, s + d, 4 * getattr(a, s + d))
    for name in ("k_pool", "v_pool"):
        setattr(a, name, at[name] + off)
        assert "aligned chunks" in _said("la_rotary_append", a)
        setattr(a, name, at[name])
