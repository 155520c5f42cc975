"""How far the 16-bit results of attention's gradient are from the 64-bit ones, by their norms."""
from __future__ import annotations

import pytest
import torch

from .test_gpu_attention_fp16_range import _want
from .test_gpu_batch_ops import _batch, _half

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,H,Hk,D", [([290, 302, 271], 4, 4, 64), ([1366, 700], 4, 1, 64), ([90, 61, 40, 17], 4, 2, 32), ([513], 2, 2, 8)],
                         ids=str)
def test_norms_of_the_errors(lens, H, Hk, D, dtype):
    """The results are rounded to within half a step, h, uniformly: h / sqrt(3) of the norm at most. For dk and dv the
    rounding of dS or P comes on top, independent of that one: sqrt(2 / 3) h. dq's dS is two 16-bit values, which together
    are off by h^2: its own rounding alone, h / sqrt(3), and 3 % for that. The 64-bit form takes delta from the given output,
    whose roundings are the forward's."""
    from proteus_b200 import kernels as KN
    q, k, v, do, plan, where, _ = _batch(lens, True, H, Hk, D, dtype, seed=D, poison=False)
    out, lse = KN.attention(q, k, v, plan)
    got = KN.attention_grad(do, q, k, v, out, lse, plan)
    h, sub = _half(dtype), 2.0 ** -25 if dtype == torch.float16 else 0.0
    for _, r in where:
        for name, x, w, limit in zip(("dq", "dk", "dv"), got, _want(q, k, v, do, out, r, D ** -0.5), (1.03 / 3 ** 0.5, (2 / 3) ** 0.5, (2 / 3) ** 0.5)):
            err = (x[0, :, r].double() - w).norm()
            assert err <= limit * h * w.norm() + sub * w.numel() ** 0.5, (name, r, (err / w.norm() / h).item())
