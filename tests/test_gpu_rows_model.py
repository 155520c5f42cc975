"""The operators together, as the model path and the driver use them: ESM-2 with attention over the valid
rows against PyTorch's, gradients of an answer by the FFN units, graphs, streams, and run_atlas's read-out."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROOT = Path(__file__).resolve().parents[1]


def _batch(model_vocab, idx=(3, 0, 7, 11, 5), seed=4):
    from proteus_b200.data import SwissProt, synthetic_dataset
    ds = SwissProt(synthetic_dataset(12, seed=seed))
    return ds.make_batch(list(idx), model_vocab)


@pytest.mark.parametrize("name", ["8M", "35M"])
def test_model_with_rows_attention_matches_sdpa(name):
    """fp32: hidden states of every valid row agree to the roundings of two fp32 forwards (each layer's
    attention, projections and norms, a few hundred steps of 2^-24 relative on states of order 1)."""
    from proteus_b200 import esm
    model, vocab, _ = esm.load(name, dtype=torch.float32, device=DEV)
    b = _batch(vocab.get_vocab())
    ids, am = b.input_ids.to(DEV), b.attention_mask.to(DEV)
    with torch.no_grad():
        want = model(input_ids=ids, attention_mask=am).last_hidden_state
        hook = esm.attach_attention(model)
        got = model(input_ids=ids, attention_mask=am).last_hidden_state
        whole = model(input_ids=ids[:1, :50]).last_hidden_state  # no mask: every row is valid
        hook.remove()
        model.set_attn_implementation("sdpa")
        want_whole = model(input_ids=ids[:1, :50]).last_hidden_state
    on = am.bool()
    assert torch.isfinite(got).all()
    tol = 500 * 2.0 ** -24 * want[on].abs().max()
    assert (got[on] - want[on]).abs().max() <= tol
    assert (whole - want_whole).abs().max() <= tol


def test_gradient_of_an_answer_by_the_units():
    """d log p(residue) / d FFN pre-activations through lm_head, attention and the log probabilities, against
    PyTorch's own attention and log_softmax, fp32."""
    from proteus_b200 import esm
    model, vocab, _ = esm.load("8M", dtype=torch.float32, device=DEV)
    head = esm.lm_head(model, seed=1)
    b = _batch(vocab.get_vocab(), idx=(3, 5))
    ids, am, rows = b.input_ids.to(DEV), b.attention_mask.to(DEV), b.valid_rows.to(DEV)
    tokens = ids.view(-1)[rows]

    def grads(plain):
        acts = []

        def keep(_m, _i, out):
            out.retain_grad()
            acts.append(out)

        hooks = [m.register_forward_hook(keep) for m in esm.ffn_modules(model)]
        h = model(input_ids=ids, attention_mask=am).last_hidden_state
        if plain:
            logits = head(h.reshape(-1, h.shape[-1]).index_select(0, rows))
            logp = torch.log_softmax(logits, 1)
            loss = logp.gather(1, tokens[:, None]).sum() - (logp.exp() * logp).sum()
        else:
            r = esm.readout(h, head, rows, tokens, top=3)
            loss = r.logprob.sum() + r.entropy.sum()
        loss.backward()
        for x in hooks:
            x.remove()
        model.zero_grad(set_to_none=True)
        return loss.detach(), [a.grad.reshape(-1, a.shape[-1])[rows] for a in acts]

    want_loss, want = grads(True)
    hook = esm.attach_attention(model, check=False)
    loss, got = grads(False)
    hook.remove()
    assert abs(loss - want_loss) <= 1e-5 * abs(want_loss)
    for x, y in zip(got, want):
        assert (x - y).norm() <= 1e-4 * y.norm()


def _ops(q, k, v, lengths, logits, tokens, rows):
    from proteus_b200 import kernels as KN
    m = KN.seq_maps(lengths, rows, lead=1, trail=1)
    plan = m.plan(0)
    out, lse = KN.attention(q, k, v, plan)
    g = KN.attention_grad(out, q, k, v, out, lse, plan)
    r = KN.token_logprobs(logits, tokens, top=4)
    return [*m, out, lse, *g, *r, KN.token_logprobs_grad(logits, tokens, r.lse, r.entropy, r.logprob, r.entropy)]


def _inputs(seed, dtype, V, lens=(40, 1, 300, 0, 129)):
    g = torch.Generator(device=DEV).manual_seed(seed)
    n = sum(lens) + 7
    mk = lambda h: torch.randn(1, h, n, 32, generator=g, device=DEV).to(dtype)  # noqa: E731
    return [mk(4), mk(2), mk(2), torch.tensor(lens, device=DEV), torch.randn(50, V, generator=g, device=DEV).to(dtype),
            torch.randint(0, V, (50, 2), generator=g, device=DEV), n]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [33, 9000])
def test_captured_replayed_and_side_stream(dtype, V):
    """A graph of all of them replayed on new inputs, two graphs replayed at once on two streams, and a call
    on a side stream give what plain calls give, bit for bit."""
    a, b = _inputs(1, dtype, V), _inputs(2, dtype, V, (7, 290, 2, 64, 107))
    assert a[-1] == b[-1]
    want_a, want_b = _ops(*a), _ops(*b)
    statics = [[t.clone() if torch.is_tensor(t) else t for t in a] for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _ops(*b)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want_b))
    graphs, outs = [], []
    for s in statics:
        _ops(*s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_ops(*s))
        graphs.append(g)
    for t, src in zip(statics[1], b):
        if torch.is_tensor(t):
            t.copy_(src)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    for _ in range(3):
        graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(outs[0], want_a))
    assert all(torch.equal(x, y) for x, y in zip(outs[1], want_b))


def test_no_wait_gave_up():
    """The bounded waits of the attention kernels recorded nothing."""
    import ctypes
    from proteus_b200 import _lib
    _ops(*_inputs(3, torch.bfloat16, 33))
    torch.cuda.synchronize()
    v = ctypes.c_int(-1)
    assert _lib.load().atlas_device_status(ctypes.byref(v), 0) == 0 and v.value == 0


def test_run_atlas_with_rows_attention_and_readout(tmp_path):
    """--attn rows --readout: the files hold every residue of the plan once, with what a forward by hand
    gives, and a stopped and resumed run writes the same."""
    from proteus_b200 import esm
    from proteus_b200.run_atlas import _dataset
    base = ["--model", "8M", "--data", "synthetic:60:3", "--device", "cuda:0", "--dtype", "fp32", "--tokens-per-batch", "4096",
            "--pilot-tokens", "4096", "--K", "8", "--Kr", "4", "--ckpt-every", "2", "--attn", "rows", "--readout", "3"]

    def run(out, *more):
        r = subprocess.run([sys.executable, "-m", "proteus_b200.run_atlas", *base, "--out", str(out), *more], cwd=ROOT,
                           capture_output=True, text=True, timeout=600)
        assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-3000:]

    run(tmp_path / "a")
    run(tmp_path / "b", "--stop-after", "3")
    run(tmp_path / "b", "--resume")
    files = sorted((tmp_path / "a" / "readout").glob("*.pt"), key=lambda p: int(p.stem))
    ds = _dataset("synthetic:60:3")
    toks = []
    model, vocab, _ = esm.load("8M", dtype=torch.float32, device=DEV)
    head = esm.lm_head(model)
    for f in files:
        r = torch.load(f)
        other = torch.load(tmp_path / "b" / "readout" / f.name)
        assert all(torch.equal(r[k], other[k]) for k in r)
        toks.append(r["tok"])
    assert torch.equal(torch.cat(toks).sort().values,
                       torch.cat([i * 1024 + torch.arange(min(int(n), ds.max_res)) for i, n in enumerate(ds.len)]).sort().values)
    r = torch.load(files[0])
    seqs = list(dict.fromkeys((r["tok"] // 1024).tolist()))
    b = ds.make_batch(seqs, vocab.get_vocab())
    rows = b.valid_rows.to(DEV)
    with torch.no_grad():
        h = model(input_ids=b.input_ids.to(DEV), attention_mask=b.attention_mask.to(DEV)).last_hidden_state
        logp = torch.log_softmax(head(h.reshape(-1, h.shape[-1])[rows]).double(), 1)
    assert torch.equal(b.tok, r["tok"])
    own = logp.gather(1, b.input_ids.view(-1)[b.valid_rows].to(DEV)[:, None])[:, 0].cpu()
    assert (r["logprob"].double() - own).abs().max() <= 1e-4
    assert (r["entropy"].double() + (logp.exp() * logp).sum(1).cpu()).abs().max() <= 1e-4
    assert (r["top_logprob"].double() - logp.topk(3).values.cpu()).abs().max() <= 1e-4
