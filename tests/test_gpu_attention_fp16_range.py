"""The fp16 gradient of attention over fp16's range: small and large values and gradients, long sequences, rows whose
gradients differ by orders of magnitude. The 64-bit form takes delta from the output that the call is given, as the
formula does.

What may be left, h = 2^-11 being the largest relative rounding error: that of dS (of P for dv) and that of the result, each
uniform within half a step, h / sqrt(3) of the norm at most, independent of one another: 0.82 h together, and the limit is h
of a sequence's and head's norm. Where one row's gradient stands for nearly all of dk and dv, few roundings make their error
and do not even out: h for P or dS, h for the result, and a third of them for the fp32 parts. A single row of dq may be off by
h of each term that it sums, |dS| |k|, and h of itself, 1 % more for the fp32 parts (a score's 70 roundings of 2^-24 at
|q| |k| scale of 6 or so: 0.01 h). A result below 2^-14 is off by up to 2^-25 whatever its size."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
H_STEP, SUB = 2.0 ** -11, 2.0 ** -25


def _case(lens, H, Hk, D, seed, size_v=1.0, size_do=1.0, rows_do=None):
    from proteus_b200 import kernels as KN
    g = torch.Generator(device=DEV).manual_seed(seed)
    n = sum(lens)
    mk = lambda h, s: torch.randn(1, h, n, D, generator=g, device=DEV) * s  # noqa: E731
    q, k, v, do = mk(H, 1.5), mk(Hk, 1.0), mk(Hk, size_v), mk(H, size_do)
    if rows_do is not None:
        do *= rows_do(n).to(DEV)[None, None, :, None]
    q, k, v, do = (t.half() for t in (q, k, v, do))
    assert all(torch.isfinite(t).all() for t in (q, k, v, do))
    plan = KN.seq_maps(torch.tensor(lens, device=DEV), n).plan(0)
    out, lse = KN.attention(q, k, v, plan)
    return (q, k, v, do, out), KN.attention_grad(do, q, k, v, out, lse, plan)


def _want(q, k, v, do, out, r, scale):
    """dq [H, n, D], dk, dv [Hk, n, D] of rows r in 64 bits, and the sizes of the terms of dq."""
    H, Hk = q.shape[1], k.shape[1]
    dq, dk, dv, terms = [], [], [], []
    for j in range(Hk):
        K, V = k[0, j, r].double(), v[0, j, r].double()
        sk, sv = torch.zeros_like(K), torch.zeros_like(K)
        for h in range(j * (H // Hk), (j + 1) * (H // Hk)):
            Q, G = q[0, h, r].double(), do[0, h, r].double()
            P = torch.softmax(Q @ K.T * scale, -1)
            dS = P * (G @ V.T - (G * out[0, h, r].double()).sum(-1, keepdim=True))
            dq.append(dS @ K * scale)
            terms.append(dS.abs() @ K.abs() * scale)
            sk += dS.T @ Q * scale
            sv += P.T @ G
        dk.append(sk)
        dv.append(sv)
    return torch.stack(dq), torch.stack(dk), torch.stack(dv), torch.stack(terms)


def _check(lens, inputs, grads, scale, rows=False, limit=H_STEP):
    c = 0
    for n in lens:
        r = slice(c, c + n)
        c += n
        *wants, terms = _want(*inputs, r, scale)
        for name, got, want in zip(("dq", "dk", "dv"), grads, wants):
            err = got[0, :, r].double() - want
            assert torch.isfinite(err).all(), (name, n)
            # every element's own limit would be larger: here lost or zero gradients fail
            a, b = err.norm(dim=(1, 2)), want.norm(dim=(1, 2))
            assert (a <= limit * b + SUB * want[0].numel() ** 0.5).all(), (name, n, (a / b / H_STEP).tolist())
            if rows and name == "dq":
                tol = 1.01 * H_STEP * (terms + want.abs()).norm(dim=2) + SUB * want.shape[2] ** 0.5
                worst = (err.norm(dim=2) / tol).max().item()
                assert worst <= 1, (n, worst)


@pytest.mark.parametrize("lens,size_v,size_do", [([4096], 0.1, 64.0), ([4096], 0.01, 256.0), ([300, 77], 1e-3, 1000.0), ([300, 1000], 1.0, 1.0),
                                                 ([300, 65], 2.0 ** 13, 2.0 ** -10), ([300], 2.0 ** -10, 2.0 ** 11), ([129], 2.0 ** -8, 2.0 ** -4),
                                                 ([2000], 2.0 ** 13, 2.0 ** -8)], ids=str)
@pytest.mark.parametrize("D,H,Hk", [(64, 2, 2), (24, 4, 2), (64, 4, 1)])
def test_sizes_of_values_and_gradients(lens, size_v, size_do, D, H, Hk):
    inputs, grads = _case(lens, H, Hk, D, len(lens) + D, size_v, size_do)
    _check(lens, inputs, grads, D ** -0.5)


@pytest.mark.parametrize("size", [2.0 ** -12, 2.0 ** -9, 1.0, 2.0 ** 9])
def test_small_and_large_gradients(size):
    """The results of the smallest lie below fp16's normal range, where they are held to 2^-25."""
    lens = [300, 65, 140]
    inputs, grads = _case(lens, 4, 2, 64, 11, 1.0, size)
    _check(lens, inputs, grads, 0.125)


@pytest.mark.parametrize("n", [70, 300, 2000])
@pytest.mark.parametrize("large", [1e3, 1e4])
@pytest.mark.parametrize("D", [64, 40])
def test_one_row_of_much_larger_gradients(n, large, D):
    """An attribution's usual gradient: one row's answer, and little elsewhere. Each row of dq keeps its own range."""
    def rows(m):
        x = torch.ones(m)
        x[m // 3] = large
        return x
    inputs, grads = _case([n], 2, 1, D, 5, 0.5, 1.0, rows)
    _check([n], inputs, grads, D ** -0.5, rows=True, limit=3 * H_STEP)


def test_rows_of_every_size():
    """Gradients from 2^-8 to 2^7 of their mean, by rows, and a row of zeros."""
    def rows(m):
        x = 2.0 ** (torch.arange(m) % 16 - 8.0)
        x[5] = 0.0
        return x
    inputs, grads = _case([500, 33], 4, 2, 64, 6, 1.0, 4.0, rows)
    _check([500, 33], inputs, grads, 0.125, rows=True)
    assert (grads[0][0, :, 5] == 0).all()


def test_probabilities_below_the_normal_range():
    """17000 equal scores: each probability is below 2^-14, the smallest normal number, and all round the same way.
    With queries of zero P = 1 / n: dv is the mean of dout, and dq = scale / n (dout (V^T K) - delta sum K)."""
    from proteus_b200 import kernels as KN
    n, D = 17000, 64
    g = torch.Generator(device=DEV).manual_seed(2)
    k, v, do = ((torch.randn(1, 1, n, D, generator=g, device=DEV) + 1).half() for _ in range(3))
    q = torch.zeros_like(k)
    plan = KN.seq_maps(torch.tensor([n], device=DEV), n).plan(0)
    out, lse = KN.attention(q, k, v, plan)
    dq, dk, dv = KN.attention_grad(do, q, k, v, out, lse, plan)
    K, V, G = k[0, 0].double(), v[0, 0].double(), do[0, 0].double()
    mean = V.mean(0)
    assert (out[0, 0].double() - mean).norm(dim=1).max() <= 2 * H_STEP * mean.norm()
    want = G.mean(0)
    assert (dv[0, 0].double() - want).norm(dim=1).max() <= 2 * H_STEP * want.norm()
    assert (dk == 0).all()
    # dP - delta of a query is dout (v_j - mean): the output's rounding moves all of a query's by |dout| h |out| at most
    want = D ** -0.5 / n * (G @ (V.T @ K) - (G @ mean)[:, None] * K.sum(0))
    off = D ** -0.5 * H_STEP * (G.abs() @ mean.abs())[:, None] * K.mean(0).abs()
    assert ((dq[0, 0].double() - want).norm(dim=1) <= 3 * H_STEP * want.norm(dim=1) + off.norm(dim=1) + SUB * 8).all()


@pytest.mark.parametrize("n", [3000, 17000])
def test_output_of_many_small_weights(n):
    """One key of weight near 1 and a value of zero, n others whose weights of e^-12 (2^-17.3) round alike: the output is their
    share. h for each weight, h for the result, and a few roundings of fp32 at scores of 12."""
    from proteus_b200 import kernels as KN
    D = 16
    g = torch.Generator(device=DEV).manual_seed(n)
    k = torch.zeros(1, 1, n, D, dtype=torch.float16, device=DEV)
    k[:, :, 0, 0] = 12.0
    q = torch.zeros_like(k)
    q[..., 0] = 1.0
    v = (torch.rand(1, 1, n, D, generator=g, device=DEV) + 1).half()
    v[:, :, 0] = 0.0
    plan = KN.seq_maps(torch.tensor([n], device=DEV), n).plan(0)
    out, lse = KN.attention(q, k, v, plan, 1.0)
    w = torch.full((n,), -12.0, dtype=torch.float64, device=DEV).exp()
    w[0] = 1.0
    want = (w @ v[0, 0].double()) / w.sum()
    assert ((out[0, 0].double() - want).abs() <= 2.1 * H_STEP * want + SUB).all()
    assert (lse[0, 0].double() - (12 + w.sum().log())).abs().max() <= (n / 64 + 100) * 2.0 ** -24
