"""Attention over values near the ends of their type: the output is a mean of values, and finite as they are, however the
scores lie."""
from __future__ import annotations

import pytest
import torch

from .test_gpu_batch_ops import DEV, U, _batch, _half

pytestmark = pytest.mark.gpu


def _mean(q, k, v, r, scale):
    """The output of rows r of a packed batch in 64 bits, the mean of |v|, the log-sum-exp, and the largest score."""
    H, Hk = q.shape[1], k.shape[1]
    S = q[0, :, r].double() @ k[0, :, r].double().repeat_interleave(H // Hk, 0).transpose(1, 2) * scale
    P = torch.softmax(S, -1)
    V = v[0, :, r].double().repeat_interleave(H // Hk, 0)
    return P @ V, P @ V.abs(), torch.logsumexp(S, -1), S.abs().max()


def _check(out, lse, q, k, v, where, scale):
    """h of each weight and of the result; a weight's score is some D + 6 + 16 roundings of fp32 of |q| |k| scale (twice: in the
    weight and in its sum), and a sum of n terms n."""
    D = q.shape[3]
    h = U if q.dtype == torch.float32 else _half(q.dtype)
    for _, r in where:
        want, mean, wl, top = _mean(q, k, v, r, scale)
        n = want.shape[1]
        fp = 2 * U * ((D + 24) * (top + 2) + n + 8)
        # fp16 weights below 2^-14 are off by 2^-25, with a largest of 2^-15 or more: 2^-10 of a mean value at most together
        assert torch.isfinite(out[0, :, r]).all()
        tol = (2 * h + fp) * mean
        if q.dtype == torch.float16:
            tol = tol + n * 2.0 ** -25 * v[0, :, r].double().abs().max()
        assert ((out[0, :, r].double() - want).abs() <= tol).all()
        assert ((lse[0, :, r].double() - wl).abs() <= fp + 4 * U * wl.abs()).all()


SIZES = {torch.bfloat16: [2.0 ** 124, 2.0 ** 70, 2.0 ** -90], torch.float32: [2.0 ** 124, 2.0 ** 70, 2.0 ** -90], torch.float16: [2.0 ** 13]}


@pytest.mark.parametrize("dtype,size", [(t, s) for t, ss in SIZES.items() for s in ss])
@pytest.mark.parametrize("D", [16, 13, 64])
@pytest.mark.parametrize("rise", [8.0, 2.0, 0.0, -8.0])
def test_values_of_any_size(dtype, size, D, rise):
    """Each 16 keys' scores `rise` above the 16 before; values of `size` and up to 5 times that."""
    from proteus_b200 import kernels as KN
    q, k, v, _, plan, where, _ = _batch([800, 40, 5, 161, 1, 16, 97], True, 2, 1, D, dtype, seed=7)
    v = (v.float() * size).to(dtype)
    for o, r in where:
        n = r.stop - r.start
        q[o, :, r, 0] = 1.0
        k[o, :, r, 0] = (torch.arange(n, device=DEV).div(16, rounding_mode="floor") * rise).to(dtype)
    assert torch.isfinite(v).all()
    out, lse = KN.attention(q, k, v, plan, 1.0)
    _check(out, lse, q, k, v, where, 1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [1, 5, 64, 700, 9000])
def test_the_largest_values(dtype, n):
    """Values of one sign, 2^127 throughout, under equal scores: the mean of n of them is 2^127, their sum is not finite."""
    from proteus_b200 import kernels as KN
    x = torch.ones(1, 1, n, 16, dtype=dtype, device=DEV)
    plan = KN.seq_maps(torch.tensor([n], device=DEV), n).plan(0)
    out, lse = KN.attention(x, x, x * 2.0 ** 127, plan)
    # sums of equal terms in fp32: n roundings of half a step at most
    assert ((out.double() * 2.0 ** -127 - 1).abs() <= (n + 4) * U + (0 if dtype == torch.float32 else _half(dtype))).all()
    assert (lse.double() - (4 + torch.tensor(float(n)).double().log())).abs().max() <= (n + 40) * U
