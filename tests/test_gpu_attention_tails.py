"""CTAs of attention that follow one another on an SM at once: each leaves only when its copies have landed and its
products have reported, so a long row of short calls gives the same bits every time, and no wait gives up."""
from __future__ import annotations

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens", [[17], [97] * 40, [20] * 300, [1, 130, 257, 96, 33] * 30], ids=lambda x: f"{len(x)}x{max(x)}")
def test_calls_in_a_row(lens, dtype):
    from proteus_b200 import _lib
    from proteus_b200 import kernels as KN
    n = sum(lens)
    g = torch.Generator(device=DEV).manual_seed(len(lens))
    q, k, v, do = (torch.randn(1, h, n, 64, generator=g, device=DEV).to(dtype) for h in (8, 4, 4, 8))
    plan = KN.seq_maps(torch.tensor(lens, device=DEV), n).plan(0)

    def both():
        out, lse = KN.attention(q, k, v, plan)
        return (out, lse, *KN.attention_grad(do, q, k, v, out, lse, plan))

    want = both()
    for got in [both() for _ in range(30)]:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    status = ctypes.c_int(-1)
    assert _lib.load().atlas_device_status(ctypes.byref(status), 0) == 0 and status.value == 0
