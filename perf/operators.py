"""Cases that time the operators on a model's batches and answers: the row maps of a batch built from its
lengths, attention over the valid rows with its gradient, and the log probabilities of given tokens with
theirs.

`own` chooses what `run` calls: the plain form in elementary torch operations, or the functions of
proteus_b200.kernels. Both take the state that `prepare` makes."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TILE = 128  # rows of one entry of a batch's block table
SEQ_STRIDE = 1024  # token id = sequence * SEQ_STRIDE + position


def listed():
    return [
        # the maps of one 32768-token batch of the 650M stream: sequences of nearly one length, <cls> and <eos> unscored
        {"name": "maps, one batch", "op": "maps", "batch": 109, "shortest": 271, "longest": 302, "packed": False, "lead": 1, "trail": 1},
        # many short peptides at once, packed end to end
        {"name": "maps, many peptides", "op": "maps", "batch": 65536, "shortest": 1, "longest": 64, "packed": True, "lead": 0, "trail": 0},
        # one layer's attention of the 650M architecture over the same batch
        {"name": "attention, 650M batch", "op": "attention", "dtype": "bf16", "batch": 109, "shortest": 271, "longest": 302, "packed": False, "heads": 20, "kv_heads": 20, "dim": 64},
        # the 8M architecture in fp32, lengths 30 to 400 and two specials
        {"name": "attention, 8M fp32", "op": "attention", "dtype": "fp32", "batch": 40, "shortest": 32, "longest": 402, "packed": False, "heads": 20, "kv_heads": 20, "dim": 16},
        # one short sequence alone: latency
        {"name": "attention, one peptide", "op": "attention", "dtype": "fp16", "batch": 1, "shortest": 37, "longest": 37, "packed": True, "heads": 20, "kv_heads": 20, "dim": 24},
        # forward and backward of that layer, for attributions
        {"name": "attention grad, 650M batch", "op": "attention_grad", "dtype": "bf16", "batch": 109, "shortest": 271, "longest": 302, "packed": False, "heads": 20, "kv_heads": 20, "dim": 64},
        # long and very ragged sequences, packed, four query heads to a key head
        {"name": "attention grad, long ragged", "op": "attention_grad", "dtype": "bf16", "batch": 4, "shortest": 1, "longest": 4096, "packed": True, "heads": 16, "kv_heads": 4, "dim": 64},
        # every residue of a 32768-token batch scored against the 33-token alphabet
        {"name": "logprobs, residues", "op": "logprobs", "dtype": "bf16", "rows": 30973, "vocab": 33, "given": 1, "top": 5},
        # the twenty residues scored at every position (substitution scores), fp32 logits
        {"name": "logprobs, substitutions", "op": "logprobs", "dtype": "fp32", "rows": 8191, "vocab": 33, "given": 20, "top": 0},
        # one answer over a large vocabulary: latency
        {"name": "logprobs, one answer", "op": "logprobs", "dtype": "bf16", "rows": 1, "vocab": 65537, "given": 1, "top": 20},
        # a loss and its gradient over the residues of a batch
        {"name": "logprobs grad, residues", "op": "logprobs_grad", "dtype": "bf16", "rows": 30973, "vocab": 33, "given": 1, "top": 0},
        # the same over a large vocabulary
        {"name": "logprobs grad, large", "op": "logprobs_grad", "dtype": "bf16", "rows": 4095, "vocab": 50003, "given": 1, "top": 0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["maps", "attention", "attention", "attention_grad", "attention_grad", "logprobs", "logprobs_grad"])
    if op == "maps":
        longest = _log_int(rng, 1, 8192)
        batch = _log_int(rng, 1, min(65536, max(1, 4_000_000 // longest)))
        lead, trail = rng.choice([(0, 0), (1, 1), (1, 0)])
        return {"op": op, "batch": batch, "shortest": rng.randint(0, longest), "longest": longest, "packed": rng.random() < 0.5, "lead": lead, "trail": trail}
    if op.startswith("attention"):
        kv = rng.choice([1, 2, 5, 8, 20])
        heads = min(40, kv * rng.choice([1, 1, 1, 2, 4]) if kv < 20 else kv * rng.choice([1, 1, 2]))
        # over one row alone the gradients by queries and keys are zero: nothing to compare
        longest = _log_int(rng, 2 if op.endswith("grad") else 1, 4096)
        batch = _log_int(rng, 1, max(1, min(400, 1_000_000_000 // (heads * longest * longest), 262144 // longest)))
        return {"op": op, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "batch": batch, "shortest": rng.randint(0, longest), "longest": longest,
                "packed": rng.random() < 0.5, "heads": heads, "kv_heads": kv, "dim": rng.choice([8, 16, 24, 32, 40, 48, 56, 64, 64, 64])}
    vocab = _log_int(rng, 2, 150000)
    rows = _log_int(rng, 1, min(32768, 200_000_000 // vocab))
    return {"op": op, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "rows": rows, "vocab": vocab, "given": rng.choice([1, 1, 1, 3, 20]),
            "top": 0 if op.endswith("grad") else min(vocab, rng.choice([0, 1, 5, 20]))}


def _lengths(case):
    """The batch's lengths, evenly from the longest to the shortest."""
    b, lo, hi = case["batch"], case["shortest"], case["longest"]
    return [hi - (hi - lo) * i // max(1, b - 1) for i in range(b)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kw = {"device": "cuda", "generator": g}
    s = {"case": case}
    if case["op"].startswith("logprobs"):
        n, v, j = case["rows"], case["vocab"], case["given"]
        s["logits"] = (torch.randn(n, v, **kw) * 3).to(DTYPES[case["dtype"]])
        s["tokens"] = torch.randint(0, v, (n, j), **kw)
        s["g_logprob"] = torch.randn(n, j, **kw)
        s["g_entropy"] = torch.randn(n, **kw)
        return s
    n = torch.tensor(_lengths(case), device="cuda")[torch.randperm(case["batch"], **kw)]
    s["stride"] = 0 if case["packed"] else max(1, case["longest"])
    s["rows"] = max(1, sum(_lengths(case))) if case["packed"] else case["batch"] * s["stride"]
    if case["op"] == "maps":
        s["lengths"] = n.to(torch.int32)
        s["seq"] = torch.randint(0, 500000, (case["batch"],), **kw)
        return s
    # the plan that a program makes once for all layers: prefix sums and the table of 128-row blocks
    s["cu"] = torch.cat([n.new_zeros(1), n.cumsum(0)]).to(torch.int32)
    per = ((n + TILE - 1) // TILE).clamp(min=1)
    cap = s["rows"] // TILE + case["batch"] + 1
    at = torch.arange(cap, device="cuda")
    b = torch.searchsorted(per.cumsum(0), at, right=True)
    c = b.clamp(max=case["batch"] - 1)
    first = (at - (per.cumsum(0) - per)[c]) * TILE
    s["blocks"] = torch.where((b < case["batch"])[:, None], torch.stack([c, first], 1), -1).to(torch.int32)
    s["counts"] = torch.stack([n.sum(), per.sum(), n.sum() * 0])
    outer, rows = (1, s["rows"]) if case["packed"] else (case["batch"], s["stride"])
    dt, h, hk, d = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    # queries and keys as the rotary embedding leaves them, values and the incoming gradient as a projection's columns
    s["q"] = (torch.randn(outer, h, rows, d, **kw) * 1.5).to(dt)
    s["k"] = torch.randn(outer, hk, rows, d, **kw).to(dt)
    s["v"] = torch.randn(outer, rows, hk, d, **kw).to(dt).transpose(1, 2)
    s["dout"] = torch.randn(outer, rows, h, d, **kw).to(dt).transpose(1, 2)
    return s


def _maps(s):
    case, n = s["case"], s["lengths"].to(torch.int64)
    zero = n.new_zeros(1)
    cu = torch.cat([zero, n.cumsum(0)])
    row0 = cu[:-1] if case["packed"] else torch.arange(case["batch"], device=n.device) * s["stride"]
    kept = (n - case["lead"] - case["trail"]).clamp(min=0)
    ends = kept.cumsum(0)
    at = torch.arange(s["rows"], device=n.device)
    b = torch.searchsorted(ends, at, right=True)
    on, b = b < case["batch"], b.clamp(max=case["batch"] - 1)
    p = at - (ends - kept)[b]
    slots = torch.where(on, row0[b] + case["lead"] + p, -1)
    tok = torch.where(on, s["seq"][b] * SEQ_STRIDE + p, -1)
    per = ((n + TILE - 1) // TILE).clamp(min=1)
    ends = per.cumsum(0)
    at = torch.arange(s["rows"] // TILE + case["batch"] + 1, device=n.device)
    b = torch.searchsorted(ends, at, right=True)
    on, b = b < case["batch"], b.clamp(max=case["batch"] - 1)
    blocks = torch.where(on[:, None], torch.stack([b, (at - (ends - per)[b]) * TILE], 1), -1)
    counts = torch.stack([kept.sum(), per.sum(), kept.sum() * 0])
    return {"cu": cu.to(torch.int32), "slots": slots, "tok": tok, "blocks": blocks.to(torch.int32), "counts": counts}


def _padded(s):
    """How the rows [outer * rows] lie in a [batch, longest] frame: the row of each place, and which places are rows."""
    case, cu = s["case"], s["cu"].to(torch.int64)
    wide = max(1, case["longest"])
    p = torch.arange(wide, device=cu.device)
    row0 = cu[:-1] if case["packed"] else torch.arange(case["batch"], device=cu.device) * s["stride"]
    on = p[None] < (cu[1:] - cu[:-1])[:, None]
    return torch.where(on, row0[:, None] + p, 0), on


def _framed(x, at, on):
    """[outer, H, rows, D] -> fp32 [batch, H, longest, D], zero where no row is."""
    flat = x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])
    return (flat[at].float() * on[..., None, None]).transpose(1, 2)


def _unframed(y, s, at, on, like):
    """The frame's rows back in the layout of `like`, zero in rows of no sequence."""
    outer, _, rows, _ = like.shape
    flat = torch.zeros(outer * rows + 1, y.shape[1], y.shape[3], device=y.device, dtype=y.dtype)
    flat[torch.where(on, at, outer * rows)] = y.transpose(1, 2)
    return flat[:-1].reshape(outer, rows, y.shape[1], y.shape[3]).transpose(1, 2)


def _attention(s, grad):
    case, q, k, v = s["case"], s["q"], s["k"], s["v"]
    scale, group = case["dim"] ** -0.5, case["heads"] // case["kv_heads"]
    at, on = _padded(s)
    fq, fk, fv = _framed(q, at, on), _framed(k, at, on), _framed(v, at, on)
    b, h, n, d = fq.shape
    # the query heads of one key head lie one after the other: their rows share its keys
    fq = fq.reshape(b, case["kv_heads"], group * n, d)
    x = fq @ fk.transpose(2, 3) * scale
    x = x.masked_fill(~on[:, None, None, :], -math.inf)
    top = x.amax(3, keepdim=True).clamp(min=-1e30)
    x = torch.exp(x - top)
    z = x.sum(3, keepdim=True).clamp(min=1e-30)
    p = x / z
    lse = (top + torch.log(z)).reshape(b, h, n, 1) * on[:, None, :, None]
    o = p @ fv
    out = _unframed(o.reshape(b, h, n, d), s, at, on, q).to(q.dtype)
    lse = _unframed(lse, s, at, on, q)[..., 0]
    if not grad:
        return {"out": out, "lse": lse}
    do = _framed(s["dout"], at, on).reshape(b, case["kv_heads"], group * n, d)
    dv = p.transpose(2, 3) @ do
    ds = (do @ fv.transpose(2, 3) - (do * o).sum(3, keepdim=True)).mul_(p)
    dq, dk = ds @ fk * scale, ds.transpose(2, 3) @ fq * scale
    return {"out": out, "lse": lse, "dq": _unframed(dq.reshape(b, h, n, d), s, at, on, q).to(q.dtype),
            "dk": _unframed(dk, s, at, on, k).to(k.dtype), "dv": _unframed(dv, s, at, on, v).to(v.dtype)}


def _logprobs(s, grad):
    case, x = s["case"], s["logits"].float()
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    z = e.sum(1, keepdim=True)
    logz = torch.log(z)
    lse = top + logz
    entropy = (logz - (e * (x - top)).sum(1, keepdim=True) / z)[:, 0]
    given = x.gather(1, s["tokens"])
    logprob = (given - top) - logz
    if grad:
        p = e / z
        dx = -p * (s["g_logprob"].sum(1, keepdim=True) + s["g_entropy"][:, None] * ((x - top) - logz + entropy[:, None]))
        dx.scatter_add_(1, s["tokens"], s["g_logprob"])
        return {"logprob": logprob, "entropy": entropy, "dlogits": dx.to(s["logits"].dtype)}
    rank = 1 + torch.stack([(x > t[:, None]).sum(1) for t in given.unbind(1)], 1)
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["top"]]
    return {"logprob": logprob, "rank": rank.to(torch.int32), "entropy": entropy, "lse": lse[:, 0], "top_id": ids,
            "top_logprob": (x.gather(1, ids) - top) - logz}


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return _maps(s) if op == "maps" else _attention(s, op.endswith("grad")) if op.startswith("attention") else _logprobs(s, op.endswith("grad"))
    from proteus_b200 import kernels as K
    if op == "maps":
        return K.seq_maps(s["lengths"], s["rows"], stride=s["stride"], lead=s["case"]["lead"], trail=s["case"]["trail"], seq=s["seq"])._asdict()
    if op.startswith("attention"):
        plan = K.SeqPlan(s["cu"], s["blocks"], s["counts"], s["stride"])
        out, lse = K.attention(s["q"], s["k"], s["v"], plan)
        if op == "attention":
            return {"out": out, "lse": lse}
        dq, dk, dv = K.attention_grad(s["dout"], s["q"], s["k"], s["v"], out, lse, plan)
        return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    r = K.token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"])
    if op == "logprobs":
        return r._asdict()
    dx = K.token_logprobs_grad(s["logits"], s["tokens"], r.lse, r.entropy, s["g_logprob"], s["g_entropy"])
    return {"logprob": r.logprob, "entropy": r.entropy, "dlogits": dx}


def work(case):
    if case["op"] == "maps":
        n = _lengths(case)
        rows = sum(n) if case["packed"] else case["batch"] * max(1, case["longest"])
        cap = max(1, rows) // TILE + case["batch"] + 1
        return {"bytes": case["batch"] * (4 + 8) + 4 * (case["batch"] + 1) + 16 * rows + 8 * cap + 24, "flops": 0}
    size = 4 if case.get("dtype") == "fp32" else 2
    if case["op"].startswith("attention"):
        n, d = _lengths(case), case["dim"]
        q, kv, pairs = sum(n) * case["heads"] * d * size, sum(n) * case["kv_heads"] * d * size, sum(x * x for x in n) * case["heads"] * d
        lse = 4 * sum(n) * case["heads"]
        if case["op"] == "attention":
            return {"bytes": 2 * q + 2 * kv + lse, "flops": 4 * pairs}
        return {"bytes": 4 * q + 4 * kv + lse, "flops": 14 * pairs}
    n, v, j = case["rows"], case["vocab"], case["given"]
    if case["op"] == "logprobs":
        return {"bytes": n * v * size + n * (j * 16 + 8 + 12 * case["top"]), "flops": 5 * n * v}
    return {"bytes": 2 * n * v * size + n * (j * 16 + 8), "flops": 12 * n * v}


def exact(case, seed):
    if case["op"] == "maps":
        return None
    s = prepare(case, seed)
    if case["op"].startswith("logprobs"):
        # the definition: log softmax, and derivatives of sum g log p[token] + g_H H by the logits
        x, t = s["logits"].double(), s["tokens"]
        lse = torch.logsumexp(x, 1)
        logp = x - lse[:, None]
        h = -(logp.exp() * logp).sum(1)
        got = {"logprob": torch.gather(logp, 1, t), "entropy": h}
        if case["op"] == "logprobs":
            best = torch.topk(logp, case["top"], dim=1).values
            return got | {"rank": None, "lse": lse, "top_id": None, "top_logprob": best}
        p, g = logp.exp(), s["g_logprob"].double()
        del x
        dx = torch.zeros_like(p).scatter_add_(1, t, g) - p * g.sum(1)[:, None]
        dx -= s["g_entropy"].double()[:, None] * p * (logp + h[:, None])
        return got | {"dlogits": dx}
    # one sequence and one head after the other
    d, group = case["dim"], case["heads"] // case["kv_heads"]
    cu = s["cu"].tolist()
    zero = {"out": s["q"], "dq": s["q"], "dk": s["k"], "dv": s["v"]}
    got = {name: torch.zeros(x.shape, dtype=torch.float64, device=x.device) for name, x in zero.items()}
    got["lse"] = torch.zeros(s["q"].shape[:3], dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        n = cu[b + 1] - cu[b]
        o, r = (0, slice(cu[b], cu[b + 1])) if case["packed"] else (b, slice(0, n))
        if not n:
            continue
        for j in range(case["kv_heads"]):
            hs = slice(j * group, (j + 1) * group)
            q, k, v, do = s["q"][o, hs, r].double(), s["k"][o, j, r].double(), s["v"][o, j, r].double(), s["dout"][o, hs, r].double()
            x = torch.einsum("gid,jd->gij", q, k) / math.sqrt(d)
            p = torch.softmax(x, 2)
            out = torch.einsum("gij,jd->gid", p, v)
            got["out"][o, hs, r], got["lse"][o, hs, r] = out, torch.logsumexp(x, 2)
            if case["op"] == "attention":
                continue
            dp = torch.einsum("gid,jd->gij", do, v)
            ds = p * (dp - (p * dp).sum(2, keepdim=True)) / math.sqrt(d)
            got["dq"][o, hs, r] = torch.einsum("gij,jd->gid", ds, k)
            got["dk"][o, j, r] = torch.einsum("gij,gid->jd", ds, q)
            got["dv"][o, j, r] = torch.einsum("gij,gid->jd", p, do)
    return {name: got[name] for name in (("out", "lse") if case["op"] == "attention" else ("out", "lse", "dq", "dk", "dv"))}


