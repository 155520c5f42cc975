"""Attention with block tables that a caller made: what is not an entry of the row maps is passed over. Each bad
entry stands behind the sequence's own, among the spare ones, so that every row has its entry."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("entry", [(1, 1), (1, 5), (1, 64), (1, 127), (0, 130), (2, 200), (3, 0), (-1, 0), (-2, 7), (1 << 30, 0), (1, -128),
                                   (1, 1 << 30)], ids=str)
def test_entries_that_are_none(entry, dtype):
    from proteus_b200 import kernels as KN
    lens = [140, 300, 90]
    n = sum(lens)
    g = torch.Generator(device=DEV).manual_seed(3)
    q, k, v, do = (torch.randn(1, h, n, 32, generator=g, device=DEV).to(dtype) for h in (4, 2, 2, 4))
    plan = KN.seq_maps(torch.tensor(lens, device=DEV), n + 300).plan(0)
    out, lse = KN.attention(q, k, v, plan)
    want = (out, lse, *KN.attention_grad(do, q, k, v, out, lse, plan))
    blocks, counts = plan.blocks.clone(), plan.counts.clone()
    at = int(counts[1])
    assert at < blocks.shape[0]
    blocks[at] = torch.tensor(entry, dtype=torch.int32, device=DEV)
    counts[1] += 1
    other = plan._replace(blocks=blocks, counts=counts)
    o2, l2 = KN.attention(q, k, v, other)
    for a, b in zip(want, (o2, l2, *KN.attention_grad(do, q, k, v, o2, l2, other))):
        assert torch.equal(a, b)
