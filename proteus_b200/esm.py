"""ESM-2 models and the forward hooks that feed the atlas — drop-in for haelyons/proteus
atlas/esm.py.

Hook point (esm.py:52-63 of the reference): encoder.layer[i].intermediate.dense output, the
pre-GELU FFN activation [B, L, d_ff], handed to the sink flattened to [B*L, d_ff] — a view of
the live activation, consumed by the sink's kernels on the current stream before the forward
moves on.

Attention: PyTorch's (sdpa), or with `attn="rows"` this library's kernels over the valid rows of the
batch (kernels.attention): they plan nothing per batch shape, read no padding, and are differentiable,
for gradients of an answer by the units. `lm_head` and `readout` give the model's answers at chosen rows.

Weights: this build has no network, so `load` builds the architecture from its published
configuration with a seeded random init (the reference's `control="random"`), unless a local
HuggingFace checkpoint directory is given.
"""
from __future__ import annotations

import os

import torch

from . import kernels as KN

# name -> (layers, d_model, d_ff, heads)
ARCH = {
    "8M": (6, 320, 1280, 20),
    "35M": (12, 480, 1920, 20),
    "150M": (30, 640, 2560, 20),
    "650M": (33, 1280, 5120, 20),
    "3B": (36, 2560, 10240, 40),
}
MODELS = {"8M": "facebook/esm2_t6_8M_UR50D", "35M": "facebook/esm2_t12_35M_UR50D",
          "150M": "facebook/esm2_t30_150M_UR50D", "650M": "facebook/esm2_t33_650M_UR50D",
          "3B": "facebook/esm2_t36_3B_UR50D"}

# ESM-2 alphabet: specials, residues in the model's order, then the rest (33 tokens)
ESM_TOKENS = ["<cls>", "<pad>", "<eos>", "<unk>", "L", "A", "G", "V", "S", "E", "R", "T", "I", "D", "P", "K", "Q",
              "N", "F", "Y", "M", "H", "W", "C", "X", "B", "U", "Z", "O", ".", "-", "<null_1>", "<mask>"]


class Vocab:
    """The tokenizer surface the batcher needs (get_vocab)."""

    def __init__(self):
        self._v = {t: i for i, t in enumerate(ESM_TOKENS)}

    def get_vocab(self) -> dict:
        return dict(self._v)


def esm_config(name: str):
    from transformers import EsmConfig
    L, d, ff, heads = ARCH[name]
    return EsmConfig(vocab_size=33, hidden_size=d, num_hidden_layers=L, num_attention_heads=heads,
                     intermediate_size=ff, max_position_embeddings=1026, position_embedding_type="rotary",
                     pad_token_id=1, mask_token_id=32, token_dropout=True, emb_layer_norm_before=False,
                     layer_norm_eps=1e-5, hidden_act="gelu", hidden_dropout_prob=0.0,
                     attention_probs_dropout_prob=0.0)


def load(name: str, control: str = "none", dtype=torch.bfloat16, device="cpu", seed: int = 0, attn: str = "sdpa"):
    """Returns (model, tokenizer-like vocab, info) as the reference's load() (esm.py:21-49). attn: "sdpa",
    or "rows" for attention by this library's kernels (attach_attention)."""
    if attn not in ("sdpa", "rows"):
        raise ValueError(f"unknown attention {attn!r} (sdpa, rows)")
    from transformers import EsmModel
    local = name if os.path.isdir(str(name)) else None
    if local:
        model = EsmModel.from_pretrained(local, add_pooling_layer=False, attn_implementation="sdpa")
        arch = os.path.basename(local)
    else:
        if name not in ARCH:
            raise ValueError(f"unknown model {name!r} (known: {sorted(ARCH)})")
        torch.manual_seed(seed)
        cfg = esm_config(name)
        cfg._attn_implementation = "sdpa"
        dev = torch.device(device)
        with torch.device(dev):  # initialise on the target device (seconds instead of minutes for 650M+)
            model = EsmModel(cfg, add_pooling_layer=False)
        arch = MODELS.get(name, name)
    if control == "shuffled":
        g = torch.Generator().manual_seed(seed)
        with torch.no_grad():
            for _, p in model.named_parameters():
                flat = p.data.view(-1)
                flat.copy_(flat[torch.randperm(flat.numel(), generator=g).to(flat.device)])
    elif control not in ("none", "random"):
        raise ValueError(control)
    model = model.to(device=device, dtype=dtype).eval()
    if attn == "rows":
        attach_attention(model)
    info = {"hf": arch, "control": control if local else "random",
            "attn": getattr(model.config, "_attn_implementation", "eager"),
            "n_layers": model.config.num_hidden_layers, "d_model": model.config.hidden_size,
            "d_ff": model.config.intermediate_size, "n_params": sum(p.numel() for p in model.parameters())}
    return model, Vocab(), info


def ffn_modules(model):
    return [layer.intermediate.dense for layer in model.encoder.layer]


def attach(model, sink):
    """sink(l, H[B*L, d_ff]) from each FFN pre-activation hook; returns the hook handles."""
    handles = []
    for i, mod in enumerate(ffn_modules(model)):
        def hook(_m, _inp, out, i=i):
            sink(i, out.reshape(-1, out.shape[-1]))
        handles.append(mod.register_forward_hook(hook))
    return handles


class _RowsPlan:
    """The plan of the forward that is under way, shared by a model's attention modules; None between forwards."""
    plan = None


def _rows_attention(module, query, key, value, attention_mask, scaling=None, dropout=0.0, **kw):
    """transformers' attention interface over kernels.attention: [B, H, L, D] in, [B, L, H, D] out."""
    if dropout or kw.get("is_causal") or getattr(module, "is_causal", False):
        raise ValueError("attention over the valid rows has neither dropout nor a causal mask")
    plan = module.atlas_plan.plan
    if plan is None:
        raise RuntimeError("attention over the valid rows outside a forward of the model that attach_attention was given: "
                           "no batch's rows are known here (a layer called alone, run again by a checkpoint, or after the handle's remove)")
    out, _ = KN.attention(query, key, value, plan, scaling)
    return out.transpose(1, 2), None


def batch_plan(attention_mask: torch.Tensor) -> "KN.SeqPlan":
    """The plan of a padded batch from its [B, L] mask, whose rows must be ones followed by zeros."""
    B, L = attention_mask.shape
    return KN.seq_maps(attention_mask.sum(1, dtype=torch.int64), B * L, stride=L).plan(L)


def _plan_of(model) -> _RowsPlan:
    """The plan that the layers of `model` read: found through the model, so that a copy of it has its own."""
    return model.encoder.layer[0].attention.self.atlas_plan


def _set_plan(check, model, args, kwargs):
    x = args[0] if args else kwargs.get("input_ids")
    if x is None:
        x = kwargs["inputs_embeds"]
    mask = args[1] if len(args) > 1 else kwargs.get("attention_mask")
    if mask is None:
        mask = torch.ones(x.shape[:2], dtype=torch.int64, device=x.device)
    if getattr(model, "is_gradient_checkpointing", False) and model.training and torch.is_grad_enabled():
        raise ValueError("attention over the valid rows: a checkpointed layer would run again after the batch's plan is gone")
    if mask.dim() != 2 or mask.shape != x.shape[:2]:
        raise ValueError(f"attention over the valid rows: attention_mask must be {list(x.shape[:2])}, got {list(mask.shape)}")
    if check and bool((mask * mask != mask).any() | (mask[:, 1:] > mask[:, :-1]).any()):
        raise ValueError("attention over the valid rows: attention_mask must be ones followed by zeros in every row")
    _plan_of(model).plan = batch_plan(mask)


def _clear_plan(model, args, output):
    _plan_of(model).plan = None


class AttentionHandle:
    """The hooks of attach_attention. remove() takes them off; until model.set_attn_implementation puts another
    attention back, a forward then raises."""

    def __init__(self, *handles):
        self._handles = handles

    def remove(self):
        for h in self._handles:
            h.remove()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.remove()


def attach_attention(model, check: bool = True) -> AttentionHandle:
    """Let every attention layer of `model` run kernels.attention over the valid rows of its batch; returns
    the hooks' handle (model.set_attn_implementation puts another attention back). The batch's attention_mask
    has to be ones followed by zeros, as Batch's are; `check` looks at it, which waits for the device once a
    forward, so a loop that builds its masks so itself turns it off. Rows of padding come out of attention
    as zeros. The plan of a batch is the model's, from the start of its forward to the end: one forward at a
    time, and a layer that runs outside one raises (called alone, or again by a checkpoint in the backward pass;
    gradient checkpointing of the model is refused at once). A copy of the model has a plan of its own. A decoder
    (causal scores, or cross-attention) is refused."""
    from functools import partial
    from transformers import AttentionInterface, AttentionMaskInterface
    if model.config.is_decoder or model.config.add_cross_attention:
        raise ValueError("attention over the valid rows: every row attends to every row of its sequence, and this model is a decoder")
    AttentionInterface.register("atlas_rows", _rows_attention)
    AttentionMaskInterface.register("atlas_rows", lambda *a, **k: None)  # the plan says which rows are valid
    holder = _RowsPlan()
    for layer in model.encoder.layer:
        layer.attention.self.atlas_plan = holder
    model.set_attn_implementation("atlas_rows")
    return AttentionHandle(model.register_forward_pre_hook(partial(_set_plan, check), with_kwargs=True),
                           model.register_forward_hook(_clear_plan, always_call=True))


def lm_head(model, name: str | None = None, seed: int = 0):
    """The language-model head of an EsmModel (hidden states -> logits over its alphabet), in its dtype and on
    its device: of a local HuggingFace checkpoint directory `name`, else of the architecture with a seeded
    random init. Its projection is the model's own embedding matrix (unless the checkpoint's two are not tied)."""
    import copy
    from transformers import EsmForMaskedLM
    w = model.get_input_embeddings().weight
    if name is not None and os.path.isdir(str(name)):
        whole = EsmForMaskedLM.from_pretrained(name)
        head, tied = whole.lm_head, whole.config.tie_word_embeddings
    else:
        cfg = copy.deepcopy(model.config)
        cfg.num_hidden_layers = 1
        cfg._attn_implementation = "eager"
        torch.manual_seed(seed)
        with torch.device(w.device):
            head, tied = EsmForMaskedLM(cfg).lm_head, True
    if tied:  # as the checkpoint's own projection is; the model's embeddings may be a control's
        head.decoder.weight = w
    return head.to(device=w.device, dtype=w.dtype).eval()


def readout(hidden: torch.Tensor, head, rows: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> "KN.TokenLogprobs":
    """What the model answers at `rows` (int64, of the flattened [B*L] positions) of its last hidden states
    [B, L, d]: kernels.token_logprobs of the head's logits there, for `tokens` ([N] or [N, J] ids)."""
    return KN.token_logprobs(head(hidden.reshape(-1, hidden.shape[-1]).index_select(0, rows)), tokens, top=top)


def flops_per_batch(info: dict, n_rows: int, Lmax: int) -> float:
    """Dense matmul FLOPs of one forward over n_rows padded positions (esm.py:66-70 convention)."""
    d, f, L = info["d_model"], info["d_ff"], info["n_layers"]
    return n_rows * L * (2 * (4 * d * d + 2 * d * f) + 4 * Lmax * d)


@torch.no_grad()
def pilot(model, batches, device, max_tokens: int, store_device="cpu", layers=None):
    """Valid-token FFN activations per layer from the first batches -> list[[N, d_ff]] (esm.py:73-98).
    `layers` restricts the capture to a subset (the others are returned as None), which bounds the
    memory of large pilots."""
    L = model.config.num_hidden_layers
    keep = set(range(L)) if layers is None else set(layers)
    bufs = [[] for _ in range(L)]
    cur = {}

    def sink(l, H):
        if l in keep:
            bufs[l].append(H.index_select(0, cur["rows"]).to(store_device))

    hs = attach(model, sink)
    n = 0
    toks = []
    try:
        for b in batches:
            cur["rows"] = b.valid_rows.to(device)
            model(input_ids=b.input_ids.to(device), attention_mask=b.attention_mask.to(device))
            n += b.valid_rows.numel()
            toks.append(b.tok)
            if n >= max_tokens:
                break
    finally:
        for h in hs:
            h.remove()
    pilot.last_tok = torch.cat(toks) if toks else torch.zeros(0, dtype=torch.long)
    return [torch.cat(x) if x else None for x in bufs], n
