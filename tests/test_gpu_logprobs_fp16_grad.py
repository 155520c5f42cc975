"""The fp16 gradient of the log probabilities below the type's normal range, where it is held to 2^-25."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV, U, H_STEP, SUB = "cuda", 2.0 ** -24, 2.0 ** -11, 2.0 ** -25


@pytest.mark.parametrize("size", [2.0 ** -10, 2.0 ** -4, 1.0, 2.0 ** 8])
@pytest.mark.parametrize("N,V", [(40, 33), (9, 300), (5, 5000), (3, 20001)])
def test_small_results(N, V, size):
    """dx = (one - p) g - h p (log p + H): half a step of the result, 2^-25 below the normal range, and fp32's part, of the
    terms p g, p h |log p| and p h H (their exponent's and the log-sum-exp's roundings: V / 512 + 120 of 2^-24, and 4 of
    |log p|). Norms too, so that lost gradients fail."""
    from proteus_b200 import kernels as KN
    g = torch.Generator(device=DEV).manual_seed(V)
    x = (torch.randn(N, V, generator=g, device=DEV) * 3).half()
    t = torch.randint(0, V, (N,), generator=g, device=DEV)
    gl, gh = torch.randn(N, generator=g, device=DEV) * size, torch.randn(N, generator=g, device=DEV) * size
    r = KN.token_logprobs(x, t)
    dx = KN.token_logprobs_grad(x, t, r.lse, r.entropy, gl, gh).double()
    logp = torch.log_softmax(x.double(), 1)
    p, G, E = logp.exp(), gl.double()[:, None], gh.double()[:, None]
    H = -(p * logp).sum(1, keepdim=True)
    want = -p * G - E * p * (logp + H)
    want.scatter_add_(1, t[:, None], G)
    part = p * (G.abs() + E.abs() * (logp.abs() + H))
    tol = H_STEP * want.abs() + SUB + U * (V / 512 + 120 + 4 * logp.abs()) * part + 4 * U * G.abs() * (torch.arange(V, device=DEV) == t[:, None])
    assert ((dx - want).abs() <= tol).all()
    assert ((dx - want).norm(dim=1) <= H_STEP * want.norm(dim=1) + SUB * V ** 0.5).all()
