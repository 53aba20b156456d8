"""``rotary_kv_append`` into fp8 pools that begin anywhere: the codes and scales are those of pools that
begin at whole chunks, bit for bit, and nothing beside the pools is written."""

from __future__ import annotations

import pytest
import torch

from linattn_amd.kernels.kv_cache import rotary_kv_append

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,n", [(72, 36), (128, 64), (80, 20)])
@pytest.mark.parametrize("off", [1, 2, 3, 4])
def test_pools_that_begin_anywhere(dev, dtype, D, n, off):
    lq, before, page, Hq, Hkv, n_phys = [21, 1, 9], [5, 16, 0], 16, 4, 2, 8
    g = torch.Generator().manual_seed(50)
    q, k, v = (torch.randn(sum(lq), h, D, generator=g).to(dtype).to(dev) for h in (Hq, Hkv, Hkv))
    table = torch.randperm(n_phys, generator=g)[:6].int().view(3, 2).to(dev)
    freq = torch.rand(n, generator=g).to(dev)
    pos, cu = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (before, [0, 21, 22, 31]))
    shape, size = (n_phys, Hkv, page, D), n_phys * Hkv * page * D
    got = []
    for at in (16, off):
        whole = [torch.full((size + 32,), 0x55, dtype=torch.uint8, device=dev) for _ in "kv"]
        pools = [x[at:at + size].view(torch.float8_e4m3fn).view(shape) for x in whole]
        scales = [torch.zeros(shape[:3], device=dev) for _ in "kv"]
        gq = rotary_kv_append(q, k, v, *pools, table, pos, freq, cu_seqlens=cu, k_scale=scales[0], v_scale=scales[1])
        for x in whole:
            assert (x[:at] == 0x55).all() and (x[at + size:] == 0x55).all()
        got.append([gq, *scales, *(x[at:at + size].clone() for x in whole)])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert (got[0][1] > 0).sum() == Hkv * sum(lq)
