"""CPU checks of the model side: what attention over the valid rows refuses, and how long a batch's plan lives.
On the CPU an accepted call ends at the kernel's wrapper (AtlasKernelError), or at a stand-in for it."""
from __future__ import annotations

import pytest
import torch

from proteus_b200 import esm
from proteus_b200._lib import AtlasKernelError


def _tiny(seed=0, **kw):
    from transformers import EsmConfig, EsmModel
    torch.manual_seed(seed)
    cfg = EsmConfig(vocab_size=33, hidden_size=16, num_hidden_layers=2, num_attention_heads=2, intermediate_size=32,
                    max_position_embeddings=64, position_embedding_type="rotary", pad_token_id=1, mask_token_id=32,
                    token_dropout=True, hidden_dropout_prob=0.0, attention_probs_dropout_prob=0.0, **kw)
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


@pytest.fixture
def plans(monkeypatch):
    """Attention and row maps replaced by stand-ins that run on the CPU: the list gets the lengths that each layer's
    attention was given."""
    seen = []

    class Maps:
        def __init__(self, lengths):
            self.lengths = lengths.tolist()

        def plan(self, stride):
            return self.lengths

    def attention(q, k, v, plan, scale=None):
        seen.append(plan)
        return torch.zeros_like(q), None

    monkeypatch.setattr(esm.KN, "seq_maps", lambda lengths, rows, stride: Maps(lengths))
    monkeypatch.setattr(esm.KN, "attention", attention)
    return seen


def _mask(*lens, width=6):
    return (torch.arange(width) < torch.tensor(lens)[:, None]).long()


IDS = torch.full((2, 6), 5)


def test_a_copy_of_the_model_has_its_own_plan(plans):
    """Made after a forward, the copy's attention follows the copy's batches, and the other way round."""
    import copy
    import io
    model = _tiny()
    esm.attach_attention(model)
    model(input_ids=IDS, attention_mask=_mask(6, 6))
    other = copy.deepcopy(model)
    plans.clear()
    other(input_ids=IDS, attention_mask=_mask(3, 3))
    model(input_ids=IDS, attention_mask=_mask(2, 5))
    other(input_ids=IDS, attention_mask=_mask(1, 4))
    assert plans == [[3, 3]] * 2 + [[2, 5]] * 2 + [[1, 4]] * 2
    f = io.BytesIO()
    torch.save(other, f)
    f.seek(0)
    plans.clear()
    torch.load(f, weights_only=False)(input_ids=IDS, attention_mask=_mask(5, 1))
    assert plans == [[5, 1]] * 2


def test_the_plan_ends_with_the_forward(plans):
    """What runs a layer outside the model's forward has no batch's plan, least of all the last batch's."""
    model = _tiny()
    hook = esm.attach_attention(model)
    model(input_ids=IDS, attention_mask=_mask(6, 2))
    plans.clear()
    states = torch.zeros(2, 6, 16)
    for call in (lambda: model.encoder(states), lambda: model.encoder.layer[1](states)):
        with pytest.raises(RuntimeError, match="outside a forward"):
            call()
    hook.remove()
    with pytest.raises(RuntimeError, match="outside a forward"):
        model(input_ids=IDS, attention_mask=_mask(3, 3))
    model.set_attn_implementation("sdpa")
    model(input_ids=IDS, attention_mask=_mask(3, 3))
    assert not plans
    with esm.attach_attention(model):
        model(input_ids=IDS, attention_mask=_mask(3, 3))
    assert plans == [[3, 3]] * 2


def test_a_failed_forward_leaves_no_plan(plans, monkeypatch):
    model = _tiny()
    esm.attach_attention(model)
    with monkeypatch.context() as m:
        m.setattr(model.encoder.layer[1].output, "forward", lambda *a: 1 / 0)
        with pytest.raises(ZeroDivisionError):
            model(input_ids=IDS, attention_mask=_mask(6, 6))
    with pytest.raises(RuntimeError, match="outside a forward"):
        model.encoder(torch.zeros(2, 6, 16))
    with pytest.raises(ValueError):
        model(input_ids=IDS, attention_mask=_mask(6, 6, width=7))
    with pytest.raises(RuntimeError, match="outside a forward"):
        model.encoder(torch.zeros(2, 6, 16))


def test_a_checkpoint_that_runs_a_layer_again_raises(plans):
    """torch.utils.checkpoint around a layer: its second run comes in the backward pass, after the forward."""
    from torch.utils.checkpoint import checkpoint
    model = _tiny()
    esm.attach_attention(model)
    layer = model.encoder.layer[0]
    first = layer.forward
    layer.forward = lambda *a, **k: checkpoint(first, *a, use_reentrant=False, **k)
    out = model(input_ids=IDS, attention_mask=_mask(6, 6)).last_hidden_state
    with pytest.raises(RuntimeError, match="outside a forward"):
        out.sum().backward()


@pytest.mark.parametrize("kw", [{"is_decoder": True}, {"is_decoder": True, "add_cross_attention": True}], ids=str)
def test_decoders_are_refused(kw):
    """Their scores are causal, which attention over all rows of a sequence is not."""
    model = _tiny(**kw)
    with pytest.raises(ValueError, match="decoder"):
        esm.attach_attention(model)
    assert model.config._attn_implementation != "atlas_rows"


def test_a_layer_made_causal_afterwards(plans):
    model = _tiny()
    esm.attach_attention(model)
    model.encoder.layer[1].attention.self.is_causal = True
    with pytest.raises(ValueError, match="causal"):
        model(input_ids=IDS, attention_mask=_mask(6, 6))


@pytest.mark.parametrize("tied", [True, False])
def test_the_head_of_a_checkpoint_projects_with_the_models_embeddings(tmp_path, tied):
    """Of a control too, whose embeddings are not the checkpoint's any more; a checkpoint with a projection of its own keeps it."""
    from transformers import EsmForMaskedLM
    torch.manual_seed(3)
    cfg = _tiny().config
    cfg.tie_word_embeddings = tied
    whole = EsmForMaskedLM(cfg).eval()
    with torch.no_grad():
        whole.lm_head.bias.normal_()
    whole.save_pretrained(tmp_path / "m")
    own = whole.lm_head.decoder.weight
    for control in ("none", "shuffled"):
        model, _, _ = esm.load(str(tmp_path / "m"), control, dtype=torch.float32)
        head = esm.lm_head(model, str(tmp_path / "m"))
        w = model.get_input_embeddings().weight
        assert (head.decoder.weight is w) == tied
        assert torch.equal(head.decoder.weight, w if tied else own)
        assert torch.equal(head.dense.weight, whole.lm_head.dense.weight) and torch.equal(head.bias, whole.lm_head.bias)
    x = torch.randn(4, 16)
    model, _, _ = esm.load(str(tmp_path / "m"), dtype=torch.float32)
    assert torch.equal(esm.lm_head(model, str(tmp_path / "m"))(x), whole.lm_head(x))
