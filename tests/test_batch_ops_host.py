"""CPU checks around the operators on a model's batches and answers: what the C ABI and the wrappers refuse
before any CUDA call, the model-side pieces, and the driver's flags."""
from __future__ import annotations

import ctypes
import struct

import pytest
import torch

from proteus_b200 import _lib
from proteus_b200._lib import AtlasKernelError


def _buf(n=4096):
    b = ctypes.create_string_buffer(n + 64)
    return (ctypes.addressof(b) + 63) // 64 * 64, b


def test_seq_maps_refusals():
    lib = _lib.load()
    p, keep = _buf()

    def call(B=4, rows=100, stride=0, lead=0, trail=0, ptr=p, ws=None, ws_bytes=0, slots=p):
        return lib.atlas_seq_maps(ptr, 0, B, rows, stride, lead, trail, None, p, slots, p, p, p, ws, ws_bytes, None)

    for kw, word in (({"B": 0}, b"bad shape"), ({"rows": 0}, b"bad shape"), ({"rows": 2 ** 31}, b"bad shape"),
                     ({"stride": -1}, b"must not be negative"), ({"lead": -1}, b"must not be negative"),
                     ({"trail": -1}, b"must not be negative"), ({"stride": 26}, b"do not fit"), ({"ptr": None}, b"null pointer"),
                     ({"slots": p + 8}, b"aligned"), ({"B": 2000}, b"workspace")):
        assert call(**kw) == 1 and word in lib.atlas_last_error(), kw
    assert lib.atlas_seq_maps_ws_bytes(1024) == 0 and lib.atlas_seq_maps_ws_bytes(1025) >= 8 * 1025


def test_attention_refusals():
    lib = _lib.load()
    p, keep = _buf()
    strides = struct.pack("24q", *[1] * 24)

    def args(dtype=1, outer=2, rows=8, H=4, Hk=2, D=16, B=2, cap=3, packed=0, ptr=p):
        return [dtype, strides, outer, rows, H, Hk, D, p, ptr, p, B, cap, packed, 1.0]

    bad = (({"dtype": 7}, b"dtype"), ({"rows": 0}, b"bad shape"), ({"outer": 3}, b"outer must be"), ({"packed": 1}, b"outer must be"),
           ({"Hk": 3}, b"multiple"), ({"H": 0}, b"multiple"), ({"Hk": 0}, b"multiple"), ({"D": 65}, b"head dimension"),
           ({"D": 0}, b"head dimension"), ({"cap": 0}, b"block table"), ({"ptr": None}, b"null pointer"), ({"ptr": p + 4}, b"aligned"))
    for kw, word in bad:
        assert lib.atlas_attention(p, p, p, *args(**kw), p, p, None) == 1 and word in lib.atlas_last_error(), kw
        a = args(**kw)
        assert lib.atlas_attention_grad(p, p, p, p, p, p, *a, p, p, p, p, 1 << 20, None) == 1
        assert word in lib.atlas_last_error(), kw
    # 2 x 200 rows: the row maps' table has 400 / 128 + 2 + 1 entries, and with fewer some rows would be left out
    assert lib.atlas_attention(p, p, p, *args(rows=200, cap=5), p, p, None) == 1 and b"too few" in lib.atlas_last_error()
    assert lib.atlas_attention(None, p, p, *args(), p, p, None) == 1 and b"null pointer" in lib.atlas_last_error()
    assert lib.atlas_attention(p, p, p, 1, None, 2, 8, 4, 2, 16, p, p, p, 2, 3, 0, 1.0, p, p, None) == 1
    need = lib.atlas_attention_grad_ws_bytes(2, 8, 4, 2, 2)
    assert need >= 4 * 2 * 8 * 4
    for ws, size in ((p, need - 1), (p + 4, need)):
        assert lib.atlas_attention_grad(p, p, p, p, p, p, *args(), p, p, p, ws, size, None) == 1
        assert b"workspace" in lib.atlas_last_error()


def test_token_logprobs_refusals():
    lib = _lib.load()
    p, keep = _buf()

    def fwd(dtype=1, N=2, V=10, ld=10, J=1, top=2, x=p, tok=p):
        return lib.atlas_token_logprobs(x, dtype, N, V, ld, tok, J, top, p, p, p, p, p, p, None)

    def grad(dtype=1, N=2, V=10, ld=10, J=1, x=p, tok=p, ldd=10):
        return lib.atlas_token_logprobs_grad(x, dtype, N, V, ld, tok, J, p, p, p, p, p, ldd, None)

    for kw, word in (({"dtype": 5}, b"dtype"), ({"V": 0}, b"bad shape"), ({"ld": 9}, b"bad shape"), ({"N": -1}, b"bad shape"),
                     ({"J": 65}, b"tokens a row"), ({"x": None}, b"null pointer"), ({"tok": None}, b"null pointer")):
        assert fwd(**kw) == 1 and word in lib.atlas_last_error(), kw
        assert grad(**kw) == 1 and word in lib.atlas_last_error(), kw
    assert fwd(top=11) == 1 and b"top must be" in lib.atlas_last_error()
    assert fwd(V=100, ld=100, top=33) == 1 and b"top must be" in lib.atlas_last_error()
    assert grad(ldd=9) == 1 and b"bad shape" in lib.atlas_last_error()
    assert fwd(N=0) == 0 and grad(N=0) == 0  # nothing to do


def test_wrappers_refuse_cpu_tensors():
    from proteus_b200 import kernels as KN
    with pytest.raises(AtlasKernelError):
        KN.seq_maps(torch.ones(3, dtype=torch.int32), 8)
    x = torch.zeros(1, 2, 8, 16)
    with pytest.raises(AtlasKernelError):
        KN.attention(x, x, x, KN.SeqPlan(torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32),
                                         torch.zeros(3, dtype=torch.int64), 0))
    with pytest.raises(AtlasKernelError):
        KN.token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))


def test_model_side_on_the_cpu():
    """The head is tied to the embeddings; attention over the valid rows has no CPU path."""
    from proteus_b200 import esm
    with pytest.raises(ValueError):
        esm.load("8M", attn="other")
    model, _, _ = esm.load("8M", dtype=torch.float32)
    head = esm.lm_head(model, seed=3)
    logits = head(torch.randn(5, model.config.hidden_size))
    assert logits.shape == (5, 33) and head.decoder.weight is model.get_input_embeddings().weight
    assert torch.equal(head.dense.weight, esm.lm_head(model, seed=3).dense.weight)
    ids, mask = torch.full((2, 6), 5), torch.ones(2, 6, dtype=torch.int64)
    before = model(input_ids=ids, attention_mask=mask).last_hidden_state
    hook = esm.attach_attention(model)
    with pytest.raises(AtlasKernelError):
        model(input_ids=ids, attention_mask=mask)
    mask[0, 2] = 0
    with pytest.raises(ValueError, match="ones followed by zeros"):
        model(input_ids=ids, attention_mask=mask)
    mask[0] = 2
    with pytest.raises(ValueError, match="ones followed by zeros"):
        model(input_ids=ids, attention_mask=mask)
    with pytest.raises(ValueError, match="attention_mask must be"):
        model(input_ids=ids, attention_mask=torch.ones(2, 5, dtype=torch.int64))
    model.train()
    model.gradient_checkpointing_enable()
    with pytest.raises(ValueError, match="checkpointed"):
        model(input_ids=ids, attention_mask=torch.ones_like(ids))
    model.gradient_checkpointing_disable()
    model.eval()
    hook.remove()
    model.set_attn_implementation("sdpa")
    assert torch.equal(model(input_ids=ids, attention_mask=torch.ones_like(mask)).last_hidden_state, before)


def test_driver_flags():
    from proteus_b200 import run_atlas as R
    base = ["--data", "synthetic:4", "--out", "x"]
    a = R.parser().parse_args(base)
    assert a.attn == "sdpa" and a.readout == -1 and "attn" not in R._args_key(a)
    b = R.parser().parse_args(base + ["--attn", "rows", "--readout", "3"])
    assert R._args_key(b)["attn"] == "rows" and b.readout == 3  # attention rounds differently; a read-out changes nothing
