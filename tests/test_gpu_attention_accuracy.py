"""How far the 16-bit results of attention's gradient are from the 64-bit ones, by their norms."""
from __future__ import annotations

import pytest
import torch

from .test_gpu_attention_fp16_range import _want
from .test_gpu_batch_ops import _batch, _half

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,H,Hk,D", [([290, 302, 271], 4, 4, 64), ([1366, 700], 4, 1, 64), ([90, 61, 40, 17], 4, 2, 32), ([513], 2, 2, 8),
                                         ([255, 256, 257, 128, 129], 4, 2, 8), ([17, 30, 33, 63, 64, 65, 18] * 4, 2, 1, 16)],
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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [8, 13, 64])
@pytest.mark.parametrize("packed", [True, False])
def test_one_row_is_its_value(packed, D, dtype):
    """A sequence of one row: its weight is 1, its output the value, bit for bit; so it is where every other key's weight
    vanishes (scores 200 lower). Its log-sum-exp is the score: D products, the scale and two roundings of 2^-24 of it."""
    from proteus_b200 import kernels as KN
    q, k, v, _, plan, where, _ = _batch([1] * 40, packed, 4, 2, D, dtype, seed=D)
    out, lse = KN.attention(q, k, v, plan)
    for o, r in where:
        assert torch.equal(out[o, :, r], v[o, :, r].repeat_interleave(2, 0))
        s = (q[o, :, r].double() * k[o, :, r].double().repeat_interleave(2, 0)).sum(-1) * D ** -0.5
        a = (q[o, :, r].double() * k[o, :, r].double().repeat_interleave(2, 0)).abs().sum(-1) * D ** -0.5
        assert ((lse[o, :, r].double() - s).abs() <= 2.0 ** -24 * ((D + 4) * a + 4 * s.abs())).all()
    q, k, v, _, plan, _, _ = _batch([150, 33], True, 4, 2, D, dtype, seed=D)
    q.zero_()
    k.zero_()
    q[..., 0] = 1.0
    k[:, :, 70, 0] = k[:, :, 150, 0] = 200.0
    out, _ = KN.attention(q, k, v, plan, 1.0)
    for r, at in ((slice(0, 150), 70), (slice(150, 183), 150)):
        assert torch.equal(out[0, :, r], v[0, :, at].repeat_interleave(2, 0)[:, None].expand(4, r.stop - r.start, D))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n", [2, 3, 10, 40, 300])
def test_log_sum_exp_keeps_its_digits(n, dtype):
    """Off by a score's roundings (D products and 3, of |q| |k| scale) and 2^-22 or so of a weight's exponential, on average over
    its keys: an absolute error, however large or small the log-sum-exp is."""
    from proteus_b200 import kernels as KN
    D = 32
    q, k, v, _, plan, where, _ = _batch([n] * 30, True, 2, 2, D, dtype, seed=n)
    _, lse = KN.attention(q, k, v, plan)
    for o, r in where:
        s = q[o, :, r].double() @ k[o, :, r].double().transpose(1, 2) * D ** -0.5
        a = (q[o, :, r].double().abs() @ k[o, :, r].double().abs().transpose(1, 2) * D ** -0.5).amax(-1)
        w = torch.logsumexp(s, -1)
        err = (lse[o, :, r].double() - w).abs()
        assert (err <= 2.0 ** -24 * ((D + 3) * a + 2 * s.abs().amax(-1) + 8 + n / 8 + 2 * w.abs())).all()
        assert err.norm() <= 2.0 ** -22 * (1 + w.norm())
