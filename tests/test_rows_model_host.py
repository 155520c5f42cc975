"""CPU checks of the model side: what attention over the valid rows refuses, and how long a batch's plan lives.
On the CPU an accepted call ends at the kernel's wrapper (AtlasKernelError), or at a stand-in for it."""
from __future__ import annotations

import pytest
import torch

from proteus_b200 import esm
from proteus_b200._lib import AtlasKernelError


def _tiny(seed=0):
    from transformers import EsmConfig, EsmModel
    torch.manual_seed(seed)
    cfg = EsmConfig(vocab_size=33, hidden_size=16, num_hidden_layers=2, num_attention_heads=2, intermediate_size=32,
                    max_position_embeddings=64, position_embedding_type="rotary", pad_token_id=1, mask_token_id=32,
                    token_dropout=True, hidden_dropout_prob=0.0, attention_probs_dropout_prob=0.0)
    return EsmModel(cfg, add_pooling_layer=False).eval()


@pytest.mark.parametrize("dtype", [torch.int64, torch.float32])
@pytest.mark.parametrize("row", [[2, 1, 1, 0], [2, 0, 0, 0], [3, 0, 0, 0], [2, 2, 2, 2], [-1, -1, -1, -1], [1, 0, 1, 0], [0, 1, 1, 1],
                                 [1, 1, 1, 2]], ids=str)
def test_masks_that_are_not_ones_followed_by_zeros(row, dtype):
    """The first column counts as the others do: [2, 1, 1, 0] would be taken for a sequence of 4 rows."""
    model = _tiny()
    esm.attach_attention(model)
    ids = torch.full((2, 4), 5)
    mask = torch.tensor([[1, 1, 0, 0], row], dtype=dtype)
    with pytest.raises(ValueError, match="ones followed by zeros"):
        model(input_ids=ids, attention_mask=mask)


def test_masks_of_one_column_and_good_ones():
    model = _tiny()
    esm.attach_attention(model)
    with pytest.raises(ValueError, match="ones followed by zeros"):
        model(input_ids=torch.full((3, 1), 5), attention_mask=torch.full((3, 1), 2))
    for mask in ([[1, 1, 1]], [[1, 0, 0]], [[0, 0, 0]], [[True, True, False]], [[1.0, 1.0, 0.0]]):
        mask = torch.tensor(mask)
        with pytest.raises(AtlasKernelError):
            model(input_ids=torch.full((1, 3), 5), attention_mask=mask)
