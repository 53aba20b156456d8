"""What ``paged_attention`` refuses, on the CPU: by its wrapper, and by the library through the C ABI
before anything is launched."""

from __future__ import annotations

import ctypes

import pytest
import torch

from linattn_amd import _native as N
from linattn_amd.kernels.dense import paged_attention


@pytest.fixture
def as_gpu(monkeypatch):
    """Lets CPU tensors past the device check, so that what follows it can be tested here."""
    monkeypatch.setattr(N, "require_gpu", lambda *t, what: torch.device("cpu"))

    def never(*a):
        raise AssertionError("the call was not refused")

    monkeypatch.setattr(N, "on_device", never)


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


P = torch.zeros(6, 2, 16, 64)
P8 = P.to(torch.float8_e4m3fn)
S = torch.zeros(6, 2, 16)
Q = torch.zeros(9, 4, 64)


def test_cpu_tensors_are_rejected():
    with pytest.raises(RuntimeError, match="GPU"):
        paged_attention(Q, P, P, _i32(3, 4), _i32(3), _i32(4))


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(9, 4, 32)),
    dict(q=torch.zeros(9, 4, 96), k_pool=torch.zeros(6, 2, 16, 96), v_pool=torch.zeros(6, 2, 16, 96)),
    dict(q=torch.zeros(9, 3, 64)),
    dict(q=torch.zeros(9, 0, 64)),
    dict(q=Q.double()),
    dict(q=Q.half()),
    dict(q=torch.zeros(3, 4, 3, 64)),
    dict(q=torch.zeros(3, 4, 3, 64), cu_seqlens=None, q_lengths=_i32(2)),
    dict(q=torch.zeros(3, 4, 3, 64), cu_seqlens=None, q_lengths=_i32(3).long()),
    dict(q=Q, cu_seqlens=None),
    dict(q_lengths=_i32(3)),
    dict(cu_seqlens=_i32(4).long()),
    dict(cu_seqlens=_i32(1)),
    dict(cu_seqlens=_i32(5)),
    dict(k_pool=torch.zeros(6, 16, 64)),
    dict(k_pool=torch.zeros(6, 0, 16, 64), v_pool=torch.zeros(6, 0, 16, 64)),
    dict(v_pool=torch.zeros(6, 2, 17, 64)),
    dict(v_pool=P.half()),
    dict(k_pool=P.transpose(1, 2).contiguous().transpose(1, 2)),
    dict(k_scale=S, v_scale=S),
    dict(k_pool=P8, v_pool=P8),
    dict(k_pool=P8, v_pool=P8, k_scale=S, v_scale=S),  # (fp32 q)
    dict(q=Q.half(), k_pool=P8, v_pool=P8, k_scale=S),
    dict(q=Q.half(), k_pool=P8, v_pool=P8, k_scale=S, v_scale=S.half()),
    dict(q=Q.half(), k_pool=P8, v_pool=P8, k_scale=S, v_scale=torch.zeros(6, 2, 16, 2)[..., 0]),
    dict(q=Q.half(), k_pool=P8, v_pool=P8, k_scale=torch.zeros(6, 16, 2).transpose(1, 2), v_scale=torch.zeros(6, 16, 2).transpose(1, 2)),
    dict(page_table=_i32(2, 4)),
    dict(page_table=_i32(3, 0)),
    dict(page_table=_i32(3, 4).long()),
    dict(page_table=_i32(4, 3).t()),
    dict(lengths=None),
    dict(lengths=_i32(4)),
    dict(lengths=_i32(3).long()),
    dict(scale=0.0),
    dict(scale=-1.0),
    dict(scale=float("nan")),
    dict(out=torch.zeros(9, 4, 32)),
    dict(out=torch.zeros(9, 4, 64).half()),
    dict(out=torch.zeros(9, 4, 65)[..., 1:]),
    dict(out=torch.zeros(9, 64, 4).transpose(1, 2)),
    dict(out=torch.zeros(9, 4, 64), out_dtype=torch.bfloat16),
    dict(out_dtype=torch.float16),
    dict(out=torch.zeros(1, 4, 64).expand(9, 4, 64)),
    dict(out=Q),
    dict(out=P.view(-1)[:9 * 4 * 64].view(9, 4, 64)),
])
def test_the_wrapper_refuses(as_gpu, change):
    a = dict(q=Q, k_pool=P, v_pool=P.clone(), page_table=_i32(3, 4), lengths=_i32(3), cu_seqlens=_i32(4))
    a.update(change)
    names = ("q", "k_pool", "v_pool", "page_table", "lengths", "cu_seqlens")
    with pytest.raises(ValueError):
        paged_attention(*[a.pop(n) for n in names], **a)


def _args():
    base, far = 1 << 40, 1 << 32
    a = N.LaPagedAttnArgs()
    for i, name in enumerate(("q", "k_pool", "v_pool", "out", "page_table", "lengths", "workspace")):
        setattr(a, name, base + i * far)
    a.B, a.Hq, a.Hkv, a.Tq, a.D = 2, 4, 2, 8, 64
    a.q_sb, a.q_sh, a.q_st = a.o_sb, a.o_sh, a.o_st = 2048, 512, 64
    a.n_phys, a.page, a.pt_sb, a.pt_pages, a.s_stride = 6, 16, 4, 4, 1
    a.scale, a.causal, a.dtype, a.kv_dtype, a.out_dtype = 0.125, 1, N.LA_BF16, N.LA_BF16, N.LA_BF16
    return a, base, far


def _call(a):
    lib = N.load()
    rc = lib.la_paged_attention(ctypes.byref(a), None)
    return rc, lib.la_last_error().decode()


@pytest.mark.parametrize("change,said", [
    (dict(B=0), "positive"), (dict(Hq=3), "multiple"), (dict(D=96), "head_dim"), (dict(dtype=N.LA_F64), "dtype"),
    (dict(kv_dtype=N.LA_F16), "cache has"), (dict(dtype=N.LA_F32, kv_dtype=N.LA_FP8_E4M3), "cache has"),
    (dict(out_dtype=N.LA_F16), "out_dtype"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(pt_pages=1 << 26), "bad cache"), (dict(n_phys=0), "bad cache"), (dict(page=0), "bad cache"),
    (dict(n_phys=1 << 27), "2^32 rows"), (dict(Tq=1 << 29), "2^30 rows"), (dict(q=(1 << 40) + 2), "aligned"),
    (dict(out=None), "aligned"), (dict(o_sh=513), "aligned"), (dict(k_pool=(1 << 40) + (1 << 32) + 8), "aligned"),
    (dict(lengths=None), "null"), (dict(page_table=None), "null"), (dict(kv_dtype=N.LA_FP8_E4M3), "scales"),
    (dict(cu_q=1 << 45, q_len=1 << 46), "batched"),
])
def test_the_library_refuses(change, said):
    a, base, far = _args()
    for name, x in change.items():
        setattr(a, name, x)
    rc, text = _call(a)
    assert rc == N.LA_ERR_INVALID and said in text, (rc, text)


def test_shared_memory_and_workspace():
    for at in (0, 256, 2 * 4 * 8 * 128 - 128, (1 << 32), (1 << 32) + 1024, (2 << 32) + 6 * 2 * 16 * 128 - 16):
        a, base, far = _args()
        a.out = base + at
        rc, text = _call(a)
        assert rc == N.LA_ERR_INVALID and "shares memory" in text, (at, rc, text)
    a, base, far = _args()
    a.ws_bytes = N.load().la_paged_attention_workspace(ctypes.byref(a)) - 1
    rc, text = _call(a)
    assert a.ws_bytes > 0 and rc == N.LA_ERR_WORKSPACE and "workspace" in text
    a.ws_bytes += 1
    a.workspace += 16
    rc, text = _call(a)
    assert rc == N.LA_ERR_INVALID and "alignment" in text
    a.Tq = 0  # (nothing to do, whatever the rest is)
    assert _call(a)[0] == N.LA_OK and N.load().la_paged_attention_workspace(ctypes.byref(a)) == 0


def test_struct_layouts_match_the_header(tmp_path):
    import subprocess
    from pathlib import Path

    header = Path(__file__).resolve().parents[1] / "include" / "linattn_hip.h"
    structs = {"la_rotary_args": N.LaRotaryArgs, "la_rotary_append_args": N.LaRotaryAppendArgs, "la_paged_attn_args": N.LaPagedAttnArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void){"]
    for c, py in structs.items():
        lines.append(f'printf("{c} size %zu\\n", sizeof({c}));')
        lines += [f'printf("{c} {f} %zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
    (tmp_path / "probe.c").write_text("\n".join([*lines, "return 0;}"]))
    subprocess.run(["gcc", "-std=c99", "-o", str(tmp_path / "probe"), str(tmp_path / "probe.c")], check=True)
    for line in subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout.splitlines():
        c, f, at = line.split()
        py = structs[c]
        assert int(at) == (ctypes.sizeof(py) if f == "size" else getattr(py, f).offset), line
        pack, _ = N.by_bytes(py)
        if f == "size":
            assert len(pack(*[0] * len(py._fields_))) == int(at)


def test_more_work_than_can_be_counted():
    """The lengths are on the device: sizes whose longest tiles would pass 64-bit places are refused."""
    a, base, far = _args()
    a.Hq, a.Tq, a.page, a.pt_pages = 2 * 1024, 1 << 19, 1 << 14, 1 << 15
    a.q_sb, a.q_sh, a.q_st = a.o_sb, a.o_sh, a.o_st = 0, 64, 64 * a.Hq
    a.cu_q = 1 << 50
    rc, text = _call(a)
    assert rc == N.LA_ERR_INVALID and "more products" in text, (rc, text)
    assert N.load().la_paged_attention_workspace(ctypes.byref(a)) == 0
