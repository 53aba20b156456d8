"""What ``rotary`` and ``rotary_kv_append`` refuse, and the 64-bit references they are tested
against, on the CPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from linattn_amd import _native as N
from linattn_amd.kernels.kv_cache import rotary_kv_append
from linattn_amd.kernels.rotary import rotary, rotary_axes
from rotary_reference import turn


@pytest.fixture
def as_gpu(monkeypatch):
    """Lets CPU tensors past the device check, so that what follows it can be tested here."""
    monkeypatch.setattr(N, "require_gpu", lambda *t, what: torch.device("cpu"))

    def never(*a):
        raise AssertionError("the call was not refused")

    monkeypatch.setattr(N, "load", never)


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_cpu_tensors_are_rejected():
    q = torch.zeros(3, 2, 64)
    with pytest.raises(RuntimeError, match="GPU"):
        rotary(q, None, _i32(3), torch.zeros(32))
    with pytest.raises(RuntimeError, match="GPU"):
        rotary_kv_append(None, q, q, torch.zeros(2, 2, 16, 64), torch.zeros(2, 2, 16, 64), _i32(1, 2), _i32(1),
                         torch.zeros(32), cu_seqlens=_i32(2))


Q = torch.zeros(2, 4, 8, 64)


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(8, 64)),
    dict(q=Q.double()),
    dict(q=torch.zeros(2, 4, 8, 514)),
    dict(k=torch.zeros(2, 2, 9, 64)),
    dict(k=torch.zeros(2, 2, 8, 32)),
    dict(k=torch.zeros(1, 2, 8, 64)),
    dict(k=torch.zeros(2, 2, 8, 64).half()),
    dict(k=torch.zeros(8, 2, 64)),
    dict(positions=_i32(2, 8).long()),
    dict(positions=_i32(8)),
    dict(positions=_i32(3, 2, 8)),
    dict(inv_freq=torch.zeros(33)),
    dict(inv_freq=torch.zeros(0)),
    dict(inv_freq=torch.zeros(32).double()),
    dict(inv_freq=torch.zeros(1, 32)),
    dict(axes=_i32(32)),
    dict(axes=_i32(31), positions=_i32(2, 2, 8)),
    dict(axes=_i32(32).long(), positions=_i32(2, 2, 8)),
    dict(axes=_i32(32), positions=_i32(0, 2, 8)),
    dict(k=None, k_out=torch.zeros(2, 2, 8, 64)),
    dict(q_out=torch.zeros(2, 4, 8, 32)),
    dict(q_out=torch.zeros(2, 4, 8, 64).half()),
    dict(q_out=torch.zeros(2, 4, 64, 8).transpose(2, 3)),
    dict(q_out=Q[:, :1].expand(2, 4, 8, 64)),
    dict(q=Q, q_out=Q.view(2, 8, 4, 64).transpose(1, 2)),
    dict(q=torch.zeros(2 * 4 * 8 * 64 + 8)[:4096].view(2, 4, 8, 64), q_out=None, overlap=True),
])
def test_rotary_refuses(as_gpu, change):
    a = dict(q=Q.clone(), k=torch.zeros(2, 2, 8, 64), positions=_i32(2, 8), inv_freq=torch.zeros(32))
    change = dict(change)
    if change.pop("overlap", False):
        buf = torch.zeros(4096 + 8)
        change = dict(q=buf[:4096].view(2, 4, 8, 64), q_out=buf[8:].view(2, 4, 8, 64))
    a.update(change)
    with pytest.raises(ValueError):
        rotary(a.pop("q"), a.pop("k"), a.pop("positions"), a.pop("inv_freq"), **a)


P = torch.zeros(6, 2, 16, 64)


@pytest.mark.parametrize("change", [
    dict(k_new=torch.zeros(2, 2, 3, 64)),
    dict(v_new=torch.zeros(5, 2, 32)),
    dict(v_new=torch.zeros(5, 2, 64).half()),
    dict(k_new=torch.zeros(5, 2, 64).double(), v_new=torch.zeros(5, 2, 64).double()),
    dict(k_new=torch.zeros(5, 0, 64), v_new=torch.zeros(5, 0, 64)),
    dict(q=torch.zeros(5, 3, 64)),
    dict(q=torch.zeros(4, 4, 64)),
    dict(q=torch.zeros(5, 4, 64).half()),
    dict(k_pool=torch.zeros(6, 3, 16, 64), v_pool=torch.zeros(6, 3, 16, 64)),
    dict(k_pool=torch.zeros(6, 2, 16, 32), v_pool=torch.zeros(6, 2, 16, 32)),
    dict(k_pool=torch.zeros(0, 2, 16, 64), v_pool=torch.zeros(0, 2, 16, 64)),
    dict(v_pool=torch.zeros(5, 2, 16, 64)),
    dict(k_pool=P.half(), v_pool=P.half()),
    dict(k_pool=torch.zeros(6, 16, 2, 64).transpose(1, 2)),
    dict(k_scale=torch.zeros(6, 2, 16), v_scale=torch.zeros(6, 2, 16)),
    dict(k_pool=P.to(torch.float8_e4m3fn), v_pool=P.to(torch.float8_e4m3fn)),
    dict(k_pool=P.to(torch.float8_e4m3fn), v_pool=P.to(torch.float8_e4m3fn), k_scale=torch.zeros(6, 2, 15), v_scale=torch.zeros(6, 2, 15)),
    dict(k_pool=P.to(torch.float8_e4m3fn), v_pool=P.to(torch.float8_e4m3fn), k_scale=torch.zeros(6, 2, 16), v_scale=torch.zeros(6, 2, 16),
         page_min=torch.zeros(2, 2, 4, 64), page_max=torch.zeros(2, 2, 4, 64), page_size=16),
    dict(page_table=_i32(3, 4)),
    dict(page_table=_i32(2, 0)),
    dict(page_table=_i32(2, 4).long()),
    dict(page_table=_i32(4, 2).t()),
    dict(positions=_i32(3)),
    dict(positions=_i32(2).long()),
    dict(cu_seqlens=_i32(3).long()),
    dict(cu_seqlens=_i32(1)),
    dict(inv_freq=torch.zeros(33)),
    dict(axes=_i32(32)),
    dict(rotary_positions=_i32(4)),
    dict(rotary_positions=_i32(2, 5)),
    dict(page_min=torch.zeros(2, 2, 4, 64)),
    dict(page_size=16),
    dict(page_min=torch.zeros(2, 2, 4, 64), page_max=torch.zeros(2, 2, 4, 64)),
    dict(page_min=torch.zeros(2, 2, 4, 64), page_max=torch.zeros(2, 2, 4, 64), page_size=0),
    dict(page_min=torch.zeros(2, 2, 4, 64), page_max=torch.zeros(2, 2, 5, 64), page_size=16),
    dict(page_min=torch.zeros(2, 2, 4, 64).half(), page_max=torch.zeros(2, 2, 4, 64).half(), page_size=16),
    dict(q=None, q_out=torch.zeros(5, 4, 64)),
    dict(q_out=torch.zeros(5, 4, 32)),
])
def test_append_refuses(as_gpu, change):
    a = dict(q=torch.zeros(5, 4, 64), k_new=torch.zeros(5, 2, 64), v_new=torch.zeros(5, 2, 64), k_pool=P.clone(),
             v_pool=P.clone(), page_table=_i32(2, 4), positions=_i32(2), inv_freq=torch.zeros(32), cu_seqlens=_i32(3))
    a.update(change)
    names = ("q", "k_new", "v_new", "k_pool", "v_pool", "page_table", "positions", "inv_freq")
    with pytest.raises(ValueError):
        rotary_kv_append(*[a.pop(n) for n in names], **a)


def _rotary_args():
    base, far = 1 << 40, 1 << 32
    a = N.LaRotaryArgs(base, base + far, base + 2 * far, base + 3 * far, base + 4 * far, base + 5 * far, None,
                       2, 8, 4, 2, 64, 32, 1, 2048, 512, 64, 1024, 512, 64, 2048, 512, 64, 1024, 512, 64, 0, 8, 1,
                       N.LA_F32, 0, 0, 0)
    return a, base, far


def _refused(fn, a):
    lib = N.load()
    rc = getattr(lib, fn)(ctypes.byref(a), None)
    assert rc in (N.LA_ERR_INVALID, N.LA_ERR_UNSUPPORTED), (rc, lib.la_last_error())
    return lib.la_last_error().decode()


def test_the_library_refuses():
    """Through the C ABI, before anything is launched."""
    for change, said in ((dict(q=None), "null"), (dict(inv_freq=None), "null"), (dict(A=2), "axes"), (dict(n=33), "frequencies"),
                         (dict(D=520, n=32), "head_dim"), (dict(Hq=0), "positive"), (dict(dtype=N.LA_F64), "dtype"),
                         (dict(B=1 << 20, T=1 << 20), "too many"), (dict(Hq=65000, Hkv=1000), "heads")):
        a, base, far = _rotary_args()
        for name, x in change.items():
            setattr(a, name, x)
        assert said in _refused("la_rotary", a), change
    # outputs over inputs: a row lower, the other tensor, one another
    for change in (dict(q_out=lambda b, f: b + 256), dict(q_out=lambda b, f: b + f), dict(k_out=lambda b, f: b),
                   dict(k_out=lambda b, f: b + 2 * f + 256)):
        a, base, far = _rotary_args()
        for name, x in change.items():
            setattr(a, name, x(base, far))
        assert "shares memory" in _refused("la_rotary", a)
    a = N.LaRotaryAppendArgs()
    assert "positive" in _refused("la_rotary_append", a)


def _append_args():
    base, far = 1 << 40, 1 << 32
    a = N.LaRotaryAppendArgs()
    for i, name in enumerate(("q", "k_new", "v_new", "q_out", "k_pool", "v_pool", "page_table", "positions", "inv_freq")):
        setattr(a, name, base + i * far)
    a.B, a.T, a.Hq, a.Hkv, a.D, a.n, a.A = 2, 8, 4, 2, 64, 32, 1
    a.q_sb, a.q_sh, a.q_st = a.o_sb, a.o_sh, a.o_st = 2048, 512, 64
    a.kn_sb, a.kn_sh, a.kn_st = a.vn_sb, a.vn_sh, a.vn_st = 1024, 512, 64
    a.n_phys, a.pool_page, a.pt_sb, a.pt_pages, a.s_stride = 6, 16, 4, 4, 1
    return a, base, far


def test_the_library_refuses_appends():
    for change, said in ((dict(Hq=3), "multiple"), (dict(pool_dtype=N.LA_F16), "pool stores"), (dict(k_pool=None), "null"),
                         (dict(pt_pages=1 << 28), "bad pool"), (dict(n_phys=0), "bad pool"), (dict(q_out=None), "null"),
                         (dict(pool_dtype=N.LA_FP8_E4M3), "scales"), (dict(page_min=1 << 45), "both"),
                         (dict(page_min=1 << 45, page_max=1 << 46), "bad page bounds"), (dict(A=3), "axes"),
                         (dict(T=1 << 30), "too many"), (dict(k_new=(1 << 40) + (1 << 32) + 2), "unaligned")):
        a, base, far = _append_args()
        for name, x in change.items():
            setattr(a, name, x)
        assert said in _refused("la_rotary_append", a), change
    for change in (dict(v_pool=lambda b, f: b + 4 * f + 1024), dict(q_out=lambda b, f: b + f), dict(k_pool=lambda b, f: b + 2 * f + 64),
                   dict(q_out=lambda b, f: b + 256), dict(v_pool=lambda b, f: b + 3 * f)):
        a, base, far = _append_args()
        for name, x in change.items():
            setattr(a, name, x(base, far))
        assert "shares memory" in _refused("la_rotary_append", a)


def test_axes_of_sections():
    assert rotary_axes((2, 1, 3)).tolist() == [0, 0, 1, 2, 2, 2]
    assert rotary_axes((2, 1, 3), interleaved=True).tolist() == [0, 1, 2, 0, 2, 2]
    for bad in ((), (0, 0), (-1, 3), (1.5, 2)):
        with pytest.raises(ValueError):
            rotary_axes(bad)


def test_the_reference_turns():
    """Known turns, lengths kept, and back again."""
    x = torch.tensor([[[1.0, 2.0, 0.0, 4.0, 9.0]]])
    quarter = torch.tensor([torch.pi / 2, torch.pi]).float()
    y, _ = turn(x, torch.tensor([1]), quarter)
    assert torch.allclose(y, torch.tensor([[[0.0, -2.0, 1.0, -4.0, 9.0]]]).double(), atol=1e-6)
    y, _ = turn(x, torch.tensor([1]), quarter, interleaved=True)
    assert torch.allclose(y, torch.tensor([[[-2.0, 1.0, 0.0, -4.0, 9.0]]]).double(), atol=1e-6)
    z, p, f = torch.randn(7, 3, 64), torch.randint(0, 9999, (7,)), torch.rand(32)
    y, tol = turn(z, p, f)
    assert torch.allclose(y.norm(dim=-1), z.double().norm(dim=-1)) and (tol > 0).all()
    assert torch.allclose(turn(y, p, f, inverse=True)[0], z.double(), atol=1e-12)
    # only the distance of two positions shows in their product
    a, b = turn(z, p, f)[0], turn(z.flip(0), p + 5, f)[0]
    c, d = turn(z, p - p, f)[0], turn(z.flip(0), p - p + 5, f)[0]
    assert torch.allclose((a * b).sum(-1), (c * d).sum(-1), atol=1e-9)


def test_outputs_that_are_inputs_hold_their_rows_once(as_gpu):
    """In place: rows of unit stride, each once."""
    for x in (torch.zeros(5, 64, 4).transpose(1, 2), torch.zeros(5, 1, 64).expand(5, 4, 64)):
        with pytest.raises(ValueError):
            rotary(x, None, _i32(5), torch.zeros(32), q_out=x)
        with pytest.raises(ValueError):
            rotary(torch.zeros(5, 4, 64), x, _i32(5), torch.zeros(32), k_out=x)
        with pytest.raises(ValueError):
            rotary_kv_append(x, torch.zeros(5, 2, 64), torch.zeros(5, 2, 64), P.clone(), P.clone(), _i32(2, 4), _i32(2),
                             torch.zeros(32), cu_seqlens=_i32(3), q_out=x)


def test_the_library_refuses_scales_over_others():
    def with_scales():
        a, base, far = _append_args()
        a.pool_dtype, a.k_scale, a.v_scale = N.LA_FP8_E4M3, base + 20 * far, base + 21 * far
        return a, base, far

    rows = 6 * 2 * 16
    for change in (dict(k_scale=lambda b, f: b + 4 * f + rows * 64 - 4), dict(v_scale=lambda b, f: b + 5 * f),
                   dict(v_scale=lambda b, f: b + 20 * f + rows * 4 - 4), dict(k_scale=lambda b, f: b + 3 * f + 64),
                   dict(v_scale=lambda b, f: b + f), dict(k_scale=lambda b, f: b + 2 * f + 128), dict(k_scale=lambda b, f: b)):
        a, base, far = with_scales()
        for name, x in change.items():
            setattr(a, name, x(base, far))
        assert "shares memory" in _refused("la_rotary_append", a), change
