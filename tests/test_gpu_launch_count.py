"""The count of launched kernels behind the bench line, for attention's gradient: by the kernels that a call's types and
strides choose."""
from __future__ import annotations

import pytest
import torch

DEV = "cuda"


def test_a_refused_call_counts_nothing():
    from proteus_b200 import _lib
    before = _lib.LAUNCHES["count"]
    with pytest.raises(_lib.AtlasKernelError, match="bad shape"):
        _lib.call("atlas_seq_maps", None, 0, 0, 0, 0, 0, 0, None, None, None, None, None, None, None, 0, None)
    assert _lib.LAUNCHES["count"] == before


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D,scale,kernels", [(torch.bfloat16, 64, None, 2), (torch.float16, 24, None, 2), (torch.float32, 64, None, 3),
                                                   (torch.bfloat16, 13, None, 3), (torch.float16, 64, -1.0, 3), (torch.bfloat16, 64, 0.0, 3)])
def test_kernels_of_the_gradient(dtype, D, scale, kernels):
    from proteus_b200 import _lib
    from proteus_b200 import kernels as KN
    lens = [40, 150]
    q, k, v, do = (torch.randn(1, 2, sum(lens), D, device=DEV).to(dtype) for _ in range(4))
    plan = KN.seq_maps(torch.tensor(lens, device=DEV), sum(lens)).plan(0)
    out, lse = KN.attention(q, k, v, plan, scale)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        before = _lib.LAUNCHES["count"]
        KN.attention_grad(do, q, k, v, out, lse, plan, scale)
        counted = _lib.LAUNCHES["count"] - before
        torch.cuda.synchronize()
    assert counted == kernels
    seen = sum(e.count for e in prof.key_averages() if "attn_" in e.key)
    assert seen in (0, kernels)  # 0: no tracing on this machine
