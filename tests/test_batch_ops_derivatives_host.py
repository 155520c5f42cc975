"""Forward-mode derivatives of the operators on a model's batches and answers: refused (on any device), since the
results would come without their tangents."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from proteus_b200 import kernels as KN
from proteus_b200._lib import AtlasKernelError

PLAN = KN.SeqPlan(torch.tensor([0, 8], dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int64), 0)


def _calls():
    x, lse = torch.randn(1, 2, 8, 16), torch.randn(1, 2, 8)
    logits, row = torch.randn(4, 9), torch.randn(4)
    tokens = torch.zeros(4, dtype=torch.int64)
    return {"attention": (lambda q, k, v: KN.attention(q, k, v, PLAN), [x, x, x]),
            "attention_grad": (lambda *t: KN.attention_grad(*t, PLAN), [x, x, x, x, x, lse]),
            "token_logprobs": (lambda t: KN.token_logprobs(t, tokens), [logits]),
            "token_logprobs_grad": (lambda a, *t: KN.token_logprobs_grad(a, tokens, *t), [logits, row, row, row, row])}


@pytest.mark.parametrize("name,arg", [(n, i) for n, (_, a) in _calls().items() for i in range(len(a))])
def test_a_tangent_is_refused(name, arg):
    call, args = _calls()[name]
    with forward_ad.dual_level():
        with pytest.raises(AtlasKernelError):  # without a tangent: as far as the device
            call(*args)
        args[arg] = forward_ad.make_dual(args[arg], torch.ones_like(args[arg]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(*args)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(*args)
