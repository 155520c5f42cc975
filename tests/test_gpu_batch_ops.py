"""The operators on a model's batches and answers against plain 64-bit forms: row maps, attention over
the valid rows with its gradient, log probabilities of given tokens with theirs.

Tolerances are worst-case sums of the roundings that each result goes through (u = 2^-24 for fp32;
h = half a step of the tensors' type, relative), evaluated on the test's own values."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _kn():
    from proteus_b200 import kernels
    return kernels


def _half(dt):
    return torch.finfo(dt).eps / 2


# ------------------------------------------------------------------------------------------- maps
def _maps_plain(lens, n_rows, stride, lead, trail, seq):
    cu, slots, tok, blocks = [0], [], [], []
    for b, n in enumerate(lens):
        row0 = b * stride if stride else cu[-1]
        for p in range(lead, n - trail):
            slots.append(row0 + p)
            tok.append((seq[b] if seq is not None else b) * 1024 + p - lead)
        blocks += [(b, p) for p in range(0, max(n, 1), 128)]
        cu.append(cu[-1] + n)
    counts = [len(slots), len(blocks), 0]
    cap = n_rows // 128 + len(lens) + 1
    assert len(blocks) <= cap and len(slots) <= n_rows
    pad = [-1] * (n_rows - len(slots))
    return cu, slots + pad, tok + pad, blocks + [(-1, -1)] * (cap - len(blocks)), counts


def _same_maps(m, want):
    for name, got, w in zip(m._fields, m, want):
        assert got.tolist() == [list(x) if isinstance(x, tuple) else x for x in w], name


@pytest.mark.parametrize("B,longest", [(1, 1), (1, 0), (1, 129), (3, 128), (7, 500), (1023, 9), (1024, 3), (1025, 3), (3000, 70)])
@pytest.mark.parametrize("packed,lead,trail", [(False, 1, 1), (True, 0, 0), (True, 1, 0), (False, 3, 200)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_maps(B, longest, packed, lead, trail, dtype):
    KN = _kn()
    g = torch.Generator().manual_seed(B + longest)
    lens = torch.randint(0, longest + 1, (B,), generator=g).tolist()
    lens[B // 2] = longest
    seq = torch.randint(0, 2 ** 21, (B,), generator=g)
    stride = 0 if packed else longest + 1
    n_rows = (sum(lens) + 5) if packed else B * stride
    for s in (seq, None):
        m = KN.seq_maps(torch.tensor(lens, dtype=dtype, device=DEV), n_rows, stride=stride, lead=lead, trail=trail,
                        seq=None if s is None else s.to(DEV))
        _same_maps(m, _maps_plain(lens, n_rows, stride, lead, trail, None if s is None else s.tolist()))


@pytest.mark.parametrize("B", [4, 2000])
def test_maps_of_lengths_that_do_not_fit(B):
    """Cut lengths are counted; packed sequences that together pass the rows are all taken as empty."""
    KN = _kn()
    lens = [3, -2, 900, 5] + [1] * (B - 4)
    m = KN.seq_maps(torch.tensor(lens, device=DEV), B * 8, stride=8)
    want = _maps_plain([3, 0, 8, 5] + [1] * (B - 4), B * 8, 8, 0, 0, None)
    want[4][2] = 2
    _same_maps(m, want)
    m = KN.seq_maps(torch.tensor([3, -2, 900, 5] + [1] * (B - 4), device=DEV), 901)
    want = _maps_plain([0] * B, 901, 0, 0, 0, None)
    want[4][2] = 2  # the negative one, and the sum
    _same_maps(m, want)


def test_maps_of_no_sequence_and_refusals():
    KN = _kn()
    m = KN.seq_maps(torch.zeros(0, dtype=torch.int32, device=DEV), 300)
    assert m.cu.tolist() == [0] and m.counts.tolist() == [0, 0, 0]
    assert (m.slots == -1).all() and (m.tok == -1).all() and (m.blocks == -1).all()
    n = torch.ones(4, dtype=torch.int32, device=DEV)
    for kw in ({"n_rows": 0}, {"n_rows": 31, "stride": 8}, {"n_rows": 8, "lead": -1}, {"n_rows": 8, "stride": -1}):
        with pytest.raises(ValueError):
            KN.seq_maps(n, **kw)
    with pytest.raises(TypeError):
        KN.seq_maps(n.float(), 8)
    with pytest.raises(TypeError):
        KN.seq_maps(n, 8, seq=n)
    with pytest.raises(ValueError):
        KN.seq_maps(n, 8, seq=torch.zeros(4, dtype=torch.int64))


def test_maps_are_a_batch_of_the_data_pipeline():
    """slots and tok of the padded batch's lengths are its valid rows and token ids."""
    from proteus_b200.data import SwissProt, synthetic_dataset
    from proteus_b200.esm import Vocab
    KN = _kn()
    ds = SwissProt(synthetic_dataset(12, seed=4))
    b = ds.make_batch([3, 0, 7, 11], Vocab().get_vocab())
    m = KN.seq_maps(b.attention_mask.to(DEV).sum(1), b.n_rows, stride=b.input_ids.shape[1], lead=1, trail=1,
                    seq=torch.tensor([3, 0, 7, 11], device=DEV))
    n = b.valid_rows.numel()
    assert int(m.counts[0]) == n and torch.equal(m.slots[:n].cpu(), b.valid_rows) and torch.equal(m.tok[:n].cpu(), b.tok)


# -------------------------------------------------------------------------------------- attention
def _batch(lens, packed, H, Hk, D, dtype, seed=0, poison=True, extra=0):
    """q, k, v, dout as a forward leaves them (rotary output contiguous by head, a projection's
    columns), NaN in every row of no sequence."""
    KN = _kn()
    g = torch.Generator(device=DEV).manual_seed(seed)
    B, wide = len(lens), max(max(lens), 1)
    outer, rows = (1, max(sum(lens) + extra, 1)) if packed else (B, wide + extra)
    mk = lambda h: torch.randn(outer, h, rows, D, generator=g, device=DEV)  # noqa: E731
    q, k, v, do = (1.5 * mk(H)).to(dtype), mk(Hk).to(dtype), mk(Hk).to(dtype), mk(H).to(dtype)
    v = v.transpose(1, 2).contiguous().transpose(1, 2)
    do = do.transpose(1, 2).contiguous().transpose(1, 2)
    m = KN.seq_maps(torch.tensor(lens, device=DEV), outer * rows, stride=0 if packed else rows)
    on = torch.zeros(outer, rows, dtype=torch.bool, device=DEV)
    where, c = [], 0
    for b, n in enumerate(lens):
        where.append((0, slice(c, c + n)) if packed else (b, slice(0, n)))
        on[where[-1]] = True
        c += n
    if poison:
        for t in (q, k, v, do):
            t.masked_fill_(~on[:, None, :, None], float("nan"))
    return q, k, v, do, m.plan(0 if packed else rows), where, on


def _plain(q, k, v, do, where, scale):
    """64-bit results and, for each, the largest error that the roundings may make."""
    H, Hk, D, dt = q.shape[1], k.shape[1], q.shape[3], q.dtype
    h = U if dt == torch.float32 else _half(dt)
    ref = {n: torch.zeros(t.shape, dtype=torch.float64, device=DEV) for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    ref["lse"] = torch.zeros(q.shape[:3], dtype=torch.float64, device=DEV)
    tol = {n: torch.zeros_like(t) for n, t in ref.items()}
    for o, r in where:
        if r.stop == r.start:
            continue
        for j in range(Hk):
            hs = slice(j * (H // Hk), (j + 1) * (H // Hk))
            Q, K, V, G = q[o, hs, r].double(), k[o, j, r].double(), v[o, j, r].double(), do[o, hs, r].double()
            S = Q @ K.T * scale
            # a score: D products summed, scaled, brought to base 2 and subtracted from the maximum
            es = U * ((D + 4) * (Q.abs() @ K.abs().T * abs(scale)) + 6 * S.abs().amax(-1, keepdim=True) + 8)
            n = S.shape[-1]
            lse = torch.logsumexp(S, -1)
            P = torch.exp(S - lse[..., None])
            out, A = P @ V, P @ V.abs()
            el = es.amax(-1) + U * (n + 8)  # of the log-sum-exp: its terms' and its sum's
            ep = es + el[..., None]         # relative, of a probability
            ref["out"][o, hs, r], ref["lse"][o, hs, r] = out, lse
            # fp16 below its normal range: half its spacing, of P, and of dS at the scale that brings the
            # largest |dout| to 2^-4 or more
            fp = 2.0 ** -25 if dt == torch.float16 else 0.0
            fs = fp * 16 * G.abs().max()
            eo = h * A + (ep * P + fp) @ V.abs() + U * n * A
            tol["out"][o, hs, r] = eo + h * out.abs()
            tol["lse"][o, hs, r] = el + U * lse.abs()
            dP = G @ V.T
            delta = (P * dP).sum(-1, keepdim=True)
            dS = P * (dP - delta)
            # dP: D products; delta from the rounded output; dS rounded once
            ed = (G.abs() * (eo + h * out.abs() + U * D * out.abs())).sum(-1, keepdim=True)
            eS = ep * dS.abs() + P * (U * D * (G.abs() @ V.abs().T) + ed) + (h + 3 * U) * dS.abs() + fs
            ref["dq"][o, hs, r] = dS @ K * scale
            tol["dq"][o, hs, r] = ((eS + U * n * dS.abs()) @ K.abs()) * abs(scale) + h * ref["dq"][o, hs, r].abs()
            N = n * (H // Hk)
            t = lambda x, y: (x.transpose(-1, -2) @ y).sum(0)  # noqa: E731
            ref["dk"][o, j, r] = t(dS, Q) * scale
            tol["dk"][o, j, r] = t(eS + U * N * dS.abs(), Q.abs()) * abs(scale) + h * ref["dk"][o, j, r].abs()
            ref["dv"][o, j, r] = t(P, G)
            tol["dv"][o, j, r] = t((ep + h + U * N) * P + fp, G.abs()) + h * ref["dv"][o, j, r].abs()
    tiny = torch.finfo(dt).tiny if dt != torch.float32 else 0.0
    for name in ("out", "dq", "dk", "dv"):
        tol[name] += tiny
    return ref, tol


def _check(got, ref, tol):
    for name, t in got.items():
        err = (t.double() - ref[name]).abs()
        assert torch.isfinite(t).all(), name
        worst = (err - tol[name]).max().item()
        assert worst <= 0, (name, worst, err.max().item())


LENS = [[1], [2], [37], [64], [65], [127, 128, 129], [1, 0, 300, 0], [257, 31, 1, 513], [0, 0, 5]]
LENS += [[15, 16, 17, 18], [3, 140, 7, 0, 16, 2, 70]]  # the gradient's short sequences, among longer ones


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype,D,H,Hk", [(torch.bfloat16, 64, 4, 4), (torch.float16, 64, 4, 1), (torch.bfloat16, 24, 6, 3),
                                          (torch.float16, 16, 2, 2), (torch.float32, 64, 2, 1), (torch.float32, 20, 3, 3),
                                          (torch.bfloat16, 40, 2, 1), (torch.bfloat16, 13, 2, 2)])
def test_attention_and_gradient(lens, packed, dtype, D, H, Hk):
    KN = _kn()
    q, k, v, do, plan, where, on = _batch(lens, packed, H, Hk, D, dtype, seed=len(lens) + D, extra=3)
    ref, tol = _plain(q, k, v, do, where, D ** -0.5)
    out, lse = KN.attention(q, k, v, plan)
    _check({"out": out, "lse": lse}, ref, tol)
    dq, dk, dv = KN.attention_grad(do, q, k, v, out, lse, plan)
    _check({"dq": dq, "dk": dk, "dv": dv}, ref, tol)
    off = ~on
    for t in (out, dq, dk, dv):
        assert (t.transpose(1, 2)[off] == 0).all()
    assert (lse.transpose(1, 2)[off] == 0).all()


@pytest.mark.parametrize("B,longest", [(7, 700), (33, 150), (1100, 4), (3, 4)])
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float16, 24), (torch.float32, 20), (torch.bfloat16, 13)])
def test_attention_padded_is_packed_with_zero_rows_between(B, longest, dtype, D):
    """A sequence's results do not depend on where its rows lie, and every row of no sequence comes out
    as zero, however unevenly they are spread (lengths of 0 to `longest`, the last one alone or not at all)."""
    KN = _kn()
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, longest + 1, (B,), generator=g).tolist()
    lens[0], lens[B // 2] = longest, 0
    got = {}
    for packed in (False, True):
        q, k, v, do, plan, where, on = _batch(lens, packed, 6, 2, D, dtype, extra=5)
        gen = torch.Generator(device=DEV).manual_seed(9)
        rows = [torch.randn(4, 6, sum(lens), D, generator=gen, device=DEV).to(dtype)[i][:h] for i, h in enumerate((6, 2, 2, 6))]
        for t, x in zip((q, k, v, do), rows):
            t.transpose(1, 2)[on] = x.transpose(0, 1)
        out, lse = KN.attention(q, k, v, plan)
        got[packed] = (out, lse[..., None], *KN.attention_grad(do, q, k, v, out, lse, plan)), on
    for a, b in zip(got[False][0], got[True][0]):
        assert torch.equal(a.transpose(1, 2)[got[False][1]], b.transpose(1, 2)[got[True][1]])
        for t, on in ((a, got[False][1]), (b, got[True][1])):
            assert (t.transpose(1, 2)[~on] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,H,Hk", [(8, 4, 2), (64, 2, 2), (13, 3, 1)])
@pytest.mark.parametrize("L", [2, 3, 4, 9, 16, 17])
def test_attention_gradient_over_few_keys(L, D, H, Hk, dtype):
    """Over few keys dP and delta nearly cancel, so that delta has to be better than the rounded output
    makes it. What may be left is the rounding of dS and that of the result, each off by at most half a step
    h of every element, uniformly within it: h / sqrt(3) of the norm each at most, and sqrt(2 / 3) h
    together, since they are independent. The limit is h; delta from the output passes it at 2, 3 and 4 keys
    (1.4 h, 1.2 h, 1.1 h in bf16)."""
    KN = _kn()
    q, k, v, do, plan, where, _ = _batch([L] * 150, True, H, Hk, D, dtype, seed=L)
    ref, _ = _plain(q, k, v, do, where, D ** -0.5)
    out, lse = KN.attention(q, k, v, plan)
    h = torch.finfo(dtype).eps / 2
    for name, t in zip(("dq", "dk", "dv"), KN.attention_grad(do, q, k, v, out, lse, plan)):
        err = (t.double() - ref[name]).norm() / ref[name].norm()
        assert err <= h, (name, (err / h).item())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_attention_scale_and_sharp_scores(dtype):
    """A given scale, and scores up to several hundred: one probability near 1, the others vanish."""
    KN = _kn()
    q, k, v, do, plan, where, _ = _batch([150, 70], True, 2, 2, 32, dtype, seed=3)
    for scale in (1.0, 8.0, -0.3):
        ref, tol = _plain(q, k, v, do, where, scale)
        out, lse = KN.attention(q, k, v, plan, scale)
        dq, dk, dv = KN.attention_grad(do, q, k, v, out, lse, plan, scale)
        _check({"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}, ref, tol)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_attention_scores_rising_along_the_keys(dtype):
    """Each 16 keys' scores stand 8 above the 16 before, from -200 to 190 over 800 keys: every reference that
    the exponents had is left behind by more than any of the types has room for."""
    KN = _kn()
    q, k, v, do, plan, where, _ = _batch([800, 40, 161], True, 2, 1, 16, dtype, seed=5)
    for o, r in where:
        n = r.stop - r.start
        q[o, :, r, 0] = 1.0
        k[o, :, r, 0] = (torch.arange(n, device=DEV).div(16, rounding_mode="floor") * 8 - n / 4).to(dtype)
    ref, tol = _plain(q, k, v, do, where, 1.0)
    # Weights below fp32's normal range are taken as zero, off by up to 2^-126 each. With |dP - delta| < 2^6,
    # |q| < 2^3, |k| < 2^8 and 1600 < 2^11 terms a sum is off by less than 2^-126 2^6 2^8 2^11 = 2^-101.
    for name in ("out", "dq", "dk", "dv"):
        tol[name] += 2.0 ** -101
    out, lse = KN.attention(q, k, v, plan, 1.0)
    dq, dk, dv = KN.attention_grad(do, q, k, v, out, lse, plan, 1.0)
    _check({"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}, ref, tol)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("first", [1, 31, 32, 33, 64, 96, 130])
def test_attention_first_scores_of_minus_infinity(first, dtype):
    """Keys whose scores are -inf weigh nothing: the result is that of the other keys alone."""
    KN = _kn()
    q, k, v, do, plan, where, _ = _batch([200], True, 2, 2, 24, dtype, seed=6)
    q[..., 0] = q[..., 0].abs() + 0.5
    kk, vv = k[:, :, first:].contiguous(), v[:, :, first:].contiguous()
    k[:, :, :first, 0] = float("-inf")
    out, lse = KN.attention(q, k, v, plan)
    s = q.double() @ kk.double().transpose(2, 3) * 24 ** -0.5
    want = torch.softmax(s, -1) @ vv.double()
    h = _half(dtype) if dtype != torch.float32 else U
    # of P and of the result h each; scores off by some 30 roundings of fp32 at 10 or so
    tol = 2 * h * (torch.softmax(s, -1) @ vv.double().abs()) + 2.0 ** -12 * h + 600 * U
    assert ((out.double() - want).abs() <= tol).all()
    assert (lse.double() - torch.logsumexp(s, -1)).abs().max() <= 600 * U


@pytest.mark.parametrize("size", [2.0 ** -12, 1.0, 2.0 ** 5, 2.0 ** 9])
def test_attention_gradient_of_small_and_large_fp16(size):
    """Incoming fp16 gradients far from 1: dS would leave fp16's range at its ends; one sequence of
    gradients 2^6 larger than the others' keeps its own range. (At 2^9 that sequence's own gradients pass
    65504, fp16's largest: infinite, and no concern of the others.)"""
    KN = _kn()
    q, k, v, do, plan, where, _ = _batch([300, 65, 140], True, 4, 2, 64, torch.float16, seed=11)
    do = do * size
    do[:, :, 300:365] *= 64
    ref, tol = _plain(q, k, v, do, where, 0.125)
    out, lse = KN.attention(q, k, v, plan)
    dq, dk, dv = KN.attention_grad(do, q, k, v, out, lse, plan)
    step = 2.0 ** -25  # half the spacing of fp16 below its normal range
    for name in ("dq", "dk", "dv"):
        tol[name] += step
    for o, r in where:
        if torch.isfinite(do[o, :, r]).all():
            _check({n: t[o, :, r] for n, t in (("dq", dq), ("dk", dk), ("dv", dv))}, {n: t[o, :, r] for n, t in ref.items()},
                   {n: t[o, :, r] for n, t in tol.items()})
        else:
            assert size == 2.0 ** 9 and r.start == 300


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_strides(dtype):
    """Columns of one projection (row stride 3 H D), rows taken in twos, a head axis in reverse order
    of memory, and a start off the 16-byte boundary give what contiguous tensors give."""
    KN = _kn()
    H, D, lens = 4, 64, [90, 140, 3]
    q, k, v, do, plan, _, _ = _batch(lens, True, H, H, D, dtype, seed=8, poison=False)
    n = q.shape[2]
    want = KN.attention(q, k, v, plan)
    wgrad = KN.attention_grad(do, q, k, v, *want, plan)

    def columns(i, x):
        w = torch.zeros(1, n, 3, H, D, dtype=dtype, device=DEV)
        w[:, :, i] = x.transpose(1, 2)
        return w[:, :, i].transpose(1, 2)

    def every_other(x):
        w = torch.full((1, H, 2 * n, D), float("nan"), dtype=dtype, device=DEV)
        w[:, :, ::2] = x
        return w[:, :, ::2]

    def shifted(x):
        w = torch.zeros(x.numel() + 1, dtype=dtype, device=DEV)
        w[1:] = x.contiguous().view(-1)
        return w[1:].view(x.shape)

    def wide(x):  # row stride no multiple of 16 bytes
        w = torch.zeros(1, H, n, D + 3, dtype=dtype, device=DEV)
        w[..., :D] = x
        return w[..., :D]

    for f in (lambda t: [columns(i, x) for i, x in enumerate(t)] , lambda t: [every_other(x) for x in t],
              lambda t: [shifted(x) for x in t], lambda t: [wide(x) for x in t],
              lambda t: [x.transpose(2, 3).contiguous().transpose(2, 3) for x in t]):
        a = f([q, k, v])
        out, lse = KN.attention(*a, plan)
        ref, tol = _plain(q, k, v, do, [(0, slice(0, 90)), (0, slice(90, 230)), (0, slice(230, 233))], D ** -0.5)
        _check({"out": out, "lse": lse}, ref, tol)
        dq, dk, dv = KN.attention_grad(f([do, do, do])[0], *a, out, lse, plan)
        _check({"dq": dq, "dk": dk, "dv": dv}, ref, tol)
    assert torch.equal(want[0], KN.attention(q, k, v, plan)[0])
    assert all(torch.equal(a, b) for a, b in zip(wgrad, KN.attention_grad(do, q, k, v, *want, plan)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_bad_sequence_stays_alone(dtype):
    """NaN and infinity in one packed sequence reach no other, forward or backward."""
    KN = _kn()
    q, k, v, do, plan, where, _ = _batch([100, 60, 200], True, 2, 1, 64, dtype, seed=5)
    out, lse = KN.attention(q, k, v, plan)
    grads = KN.attention_grad(do, q, k, v, out, lse, plan)
    bad = slice(100, 160)
    q2, k2, v2, do2 = (t.clone() for t in (q, k, v, do))
    q2[:, :, bad], k2[:, :, bad], v2[:, :, bad], do2[:, :, bad] = float("inf"), float("nan"), float("-inf"), float("nan")
    out2, lse2 = KN.attention(q2, k2, v2, plan)
    grads2 = KN.attention_grad(do2, q2, k2, v2, out2, lse2, plan)
    for x, y in zip((out, lse, *grads), (out2, lse2, *grads2)):
        for r in (slice(0, 100), slice(160, 360)):
            assert torch.equal(x[:, :, r], y[:, :, r])


def test_attention_autograd_and_differences():
    """backward() gives attention_grad's results, with a gradient that is a broadcast scalar too; along
    a direction they match the difference of the forward."""
    KN = _kn()
    q, k, v, do, plan, _, _ = _batch([33, 140], True, 4, 2, 32, torch.float32, seed=2)
    out, lse = KN.attention(q, k, v, plan)
    want = KN.attention_grad(do, q, k, v, out, lse, plan)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o2, l2 = KN.attention(*leaves, plan)
    assert not l2.requires_grad and torch.equal(o2, out)
    got = torch.autograd.grad(o2, leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    o2, _ = KN.attention(*leaves, plan)
    o2.sum().backward()
    ones = KN.attention_grad(torch.ones_like(out), q, k, v, out, lse, plan)
    assert all(torch.equal(a.grad, b) for a, b in zip(leaves, ones))
    # central difference, step e: error e^2/6 of the third derivative plus the sums' roundings over e
    g = torch.Generator(device=DEV).manual_seed(1)
    e = 2.0 ** -7
    for i in range(3):
        d = torch.randn(leaves[i].shape, generator=g, device=DEV)
        at = lambda s: [t + s * e * d if j == i else t for j, t in enumerate((q, k, v))]  # noqa: E731,B023
        diff = ((KN.attention(*at(1), plan)[0].double() - KN.attention(*at(-1), plan)[0].double()) * do.double()).sum() / (2 * e)
        dot = (want[i].double() * d.double()).sum()
        assert abs(diff - dot) <= 2e-3 * (want[i].double().norm() * d.double().norm()) ** 1, (i, diff.item(), dot.item())


def test_attention_refusals():
    KN = _kn()
    q, k, v, do, plan, _, _ = _batch([5, 9], False, 4, 2, 16, torch.bfloat16)
    out, lse = KN.attention(q, k, v, plan)
    with pytest.raises(ValueError):
        KN.attention(q, k[:, :, :5], v, plan)
    with pytest.raises(TypeError):
        KN.attention(q, k.float(), v.float(), plan)
    with pytest.raises(TypeError):
        KN.attention(q.double(), k.double(), v.double(), plan)
    with pytest.raises(ValueError):
        KN.attention(q[:, :3], k, v, plan)
    with pytest.raises(ValueError):
        KN.attention(q, k, v, plan._replace(stride=0))
    with pytest.raises(ValueError):
        KN.attention(q, k, v, plan._replace(blocks=plan.blocks[:1]))
    with pytest.raises(TypeError):
        KN.attention(q, k, v, plan._replace(cu=plan.cu.long()))
    with pytest.raises(ValueError):
        KN.attention(q, k, v, plan._replace(cu=plan.cu.cpu()))
    wide = torch.zeros(2, 4, 9, 65, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError):
        KN.attention(wide, wide, wide, plan)
    with pytest.raises(ValueError):
        KN.attention_grad(do[:, :, :5], q, k, v, out, lse, plan)
    with pytest.raises(TypeError):
        KN.attention_grad(do.float(), q, k, v, out, lse, plan)


# --------------------------------------------------------------------------------- log probabilities
def _scores(logits, tokens, top):
    """64-bit results and error bounds of the fp32 ones."""
    x = logits.double()
    t2 = tokens if tokens.dim() == 2 else tokens[:, None]
    V = x.shape[1]
    m = x.amax(1, keepdim=True)
    none = m == -math.inf
    d = x - m.masked_fill(none, 0)
    e = torch.exp(d)
    Z = e.sum(1, keepdim=True)
    logz = torch.log(Z)
    lse = (m + logz)[:, 0]
    dz = torch.where(e > 0, e * d, 0.0)
    ent = torch.where(none[:, 0], 0.0, (logz - dz.sum(1, keepdim=True) / Z)[:, 0])
    on = (t2 >= 0) & (t2 < V)
    xt = x.gather(1, t2.clamp(0, V - 1))
    lp = torch.where(on, torch.where(none, -math.inf, xt - m - logz), 0.0)
    rank = torch.where(on, 1 + (x[:, None, :] > xt[:, :, None]).sum(2), 0)
    # a term e^d: two roundings of its exponent and 2 units of the exponential; V terms in chains of
    # at most 8 a step, then a tree
    terms = V / 512 + 24
    ez = U * (terms + 4 + 3 * (e * d.abs().nan_to_num(0, 0, 0)).sum(1, keepdim=True) / Z)
    elz = ez + 2 * U * logz.abs() + U
    tol_lse = (elz + U * (m.abs() + lse[:, None].abs()))[:, 0]
    tol_lp = elz + U * (2 * (xt - m).abs().nan_to_num(0, 0, 0) + 2 * lp.abs().nan_to_num(0, 0, 0))
    tol_ent = (elz + 3 * ez * dz.abs().sum(1, keepdim=True) / Z + U * (terms + 4) * dz.abs().sum(1, keepdim=True) / Z)[:, 0] + 2 * U
    key = torch.where(torch.isnan(x), math.inf, x)
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :top]
    return lp, rank, ent, lse, ids, tol_lp, tol_ent, tol_lse


def _close(got, want, tol):
    same = (got.double() == want) | (torch.isnan(got) & torch.isnan(want))
    bad = ~(same | ((got.double() - want).abs() <= tol))
    assert not bad.any(), ((got.double() - want).abs()[bad].max().item(), int(bad.sum()))


SIZES = [(1, 1), (5, 2), (7, 33), (300, 33), (9, 64), (3, 65), (4, 255), (3, 257), (2, 1000), (3, 1025), (2, 4099), (1, 65537),
         (200, 9001), (2, 40000)]


@pytest.mark.parametrize("N,V", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("J,top", [(None, 0), (1, 5), (3, 32), (20, 1), (64, 0), (0, 20)])
def test_token_logprobs(N, V, dtype, J, top):
    KN = _kn()
    top = min(top, V)
    g = torch.Generator(device=DEV).manual_seed(N * 7 + V)
    logits = (torch.randn(N, V, generator=g, device=DEV) * 4).to(dtype)
    tokens = torch.randint(-1, V + 1, (N,) if J is None else (N, J), generator=g, device=DEV)
    r = KN.token_logprobs(logits, tokens, top=top)
    lp, rank, ent, lse, ids, tl, te, ts = _scores(logits, tokens, top)
    assert r.logprob.shape == tokens.shape and r.rank.shape == tokens.shape and r.top_id.shape == (N, top)
    _close(r.logprob.reshape(N, -1), lp, tl)
    assert torch.equal(r.rank.reshape(N, -1).long(), rank)
    _close(r.entropy, ent, te)
    _close(r.lse, lse, ts)
    assert torch.equal(r.top_id, ids)
    tlp, _, _, _, _, ttl, _, _ = _scores(logits, ids, 0)
    _close(r.top_logprob, tlp, ttl)


@pytest.mark.parametrize("V", [33, 300, 5000, 20000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_token_logprobs_of_masked_rows_and_ties(V, dtype):
    """-inf columns, a row of -inf, rows at the type's lowest value, all equal, NaN, +inf, signed zeros."""
    KN = _kn()
    g = torch.Generator(device=DEV).manual_seed(V)
    x = torch.randn(10, V, generator=g, device=DEV).to(dtype)
    low = torch.finfo(dtype).min
    x[0] = float("-inf")
    x[1] = low
    x[2] = float("-inf")
    x[2, V // 2] = 1.5
    x[3, : V - 3] = low
    x[4] = 2.0
    x[5, ::2] = float("-inf")
    x[6, 7] = float("nan")
    x[7, 9] = float("inf")
    x[8] = (torch.arange(V, device=DEV) % 3).to(dtype)
    x[9] = 0.0
    x[9, ::2] = -0.0
    tokens = torch.tensor([[0, V // 2, V - 1, 7, 9, -100, V]], device=DEV).expand(10, -1)
    top = min(20, V)
    r = KN.token_logprobs(x, tokens, top=top)
    lp, rank, ent, lse, ids, tl, te, ts = _scores(x, tokens, top)
    keep = torch.tensor([i for i in range(10) if i not in (6, 7)], device=DEV)
    _close(r.logprob[keep], lp[keep], tl[keep])
    _close(r.entropy[keep], ent[keep], te[keep])
    _close(r.lse[keep], lse[keep], ts[keep])
    assert torch.equal(r.rank[keep].long(), rank[keep])
    assert torch.equal(r.top_id, ids)
    for i in (6, 7):
        assert torch.isnan(r.lse[i]) and torch.isnan(r.entropy[i]) and torch.isnan(r.logprob[i, :3]).all()
        assert (r.logprob[i, 5:] == 0).all() and (r.rank[i, 5:] == 0).all()
    gl, gh = torch.ones(10, 7, device=DEV), torch.ones(10, device=DEV)
    dx = KN.token_logprobs_grad(x, tokens, r.lse, r.entropy, gl, gh)
    assert (dx[0] == 0).all() and torch.isfinite(dx[keep]).all()
    _grad_close(dx[keep], x[keep], tokens[keep], gl[keep], gh[keep])


def _grad_close(dx, logits, tokens, gl, gh):
    x = logits.double()
    N, V = x.shape
    t = tokens if tokens.dim() == 2 else tokens[:, None]
    none = (x.amax(1, keepdim=True) == -math.inf)
    logp = torch.where(none, -math.inf, x - torch.logsumexp(x, 1, keepdim=True))
    # a row at the lowest value: its log-sum-exp is lost in the value, its probabilities are not
    m = x.amax(1, keepdim=True).masked_fill(none, 0)
    logp = torch.where(none, logp, (x - m) - torch.log(torch.exp(x - m).sum(1, keepdim=True)))
    p = torch.exp(logp)
    plogp = torch.where(p > 0, p * logp, 0.0)
    H = -plogp.sum(1, keepdim=True)
    on = ((t >= 0) & (t < V)) & ~none
    one = torch.zeros_like(x)
    mag = torch.zeros_like(x)
    G = torch.zeros(N, 1, dtype=torch.float64, device=DEV)
    Ga = G.clone()
    if gl is not None and t.shape[1]:
        g = gl.reshape(N, -1).double() * on
        tc = t.clamp(0, V - 1)
        one.scatter_add_(1, tc, g)
        mag.scatter_add_(1, tc, g.abs())
        G, Ga = g.sum(1, keepdim=True), g.abs().sum(1, keepdim=True)
    h = (torch.zeros(N, device=DEV) if gh is None else gh).double()[:, None]
    want = one - p * G - h * (plogp + p * H)
    # log p is taken from the fp32 log-sum-exp: its error (a chain of V / 512 + 24 roundings, one of a
    # value up to 64) is relative in p; then the products' own roundings, and one to the type
    ep = U * (V / 512 + 40 + 64 + 4 * torch.where(p > 0, logp.abs(), 0.0).clamp(max=120))
    part = p * (Ga + h.abs() * (torch.where(p > 0, logp.abs(), 0.0) + H))
    tol = (ep + 8 * U) * part + p * h.abs() * ep + (t.shape[1] + 2) * U * (mag + p * Ga) + 2.0 ** -130
    if dx.dtype != torch.float32:
        tol = tol + _half(dx.dtype) * want.abs() + torch.finfo(dx.dtype).tiny
    bad = (dx.double() - want).abs() > tol
    assert not bad.any(), ((dx.double() - want).abs()[bad].max().item(), int(bad.sum()))


@pytest.mark.parametrize("N,V", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("J,entropy", [(None, False), (1, True), (20, True), (64, False), (0, True)])
def test_token_logprobs_grad(N, V, dtype, J, entropy):
    """Against the formula, tokens drawn with repeats (the same one several times in a row) and some
    outside the vocabulary."""
    KN = _kn()
    g = torch.Generator(device=DEV).manual_seed(N * 5 + V)
    logits = (torch.randn(N, V, generator=g, device=DEV) * 3).to(dtype)
    shape = (N,) if J is None else (N, J)
    tokens = torch.randint(-1, min(V + 1, 12), shape, generator=g, device=DEV)
    gl = torch.randn(shape, generator=g, device=DEV) if J != 0 else None
    gh = torch.randn(N, generator=g, device=DEV) if entropy else None
    r = KN.token_logprobs(logits, tokens)
    dx = KN.token_logprobs_grad(logits, tokens, r.lse, r.entropy, gl, gh)
    assert dx.dtype == dtype
    _grad_close(dx, logits, tokens, gl, gh)


@pytest.mark.parametrize("V", [33, 20000])
def test_token_logprobs_far_from_zero(V):
    """Logits around 5000: the row's maximum and log Z, not their sum, give the gradient."""
    KN = _kn()
    g = torch.Generator(device=DEV).manual_seed(V)
    logits = (torch.randn(4, V, generator=g, device=DEV) * 3).round() + 5000.0
    tokens = torch.randint(0, V, (4, 2), generator=g, device=DEV)
    gl, gh = torch.randn(4, 2, generator=g, device=DEV), torch.randn(4, generator=g, device=DEV)
    r = KN.token_logprobs(logits, tokens)
    _grad_close(KN.token_logprobs_grad(logits, tokens, r.lse, r.entropy, gl, gh), logits, tokens, gl, gh)


@pytest.mark.parametrize("V", [33, 2000])
def test_token_logprobs_strides_and_autograd(V):
    """Rows of a wider tensor, a column-major one, an expanded row; backward() and a difference."""
    KN = _kn()
    g = torch.Generator(device=DEV).manual_seed(V)
    base = torch.randn(6, V + 5, generator=g, device=DEV)
    tokens = torch.randint(0, V, (6, 2), generator=g, device=DEV)
    plain = base[:, 3:V + 3].contiguous()
    want = KN.token_logprobs(plain, tokens, top=4)
    for x in (base[:, 3:V + 3], plain.t().contiguous().t()):
        # 16-byte loads start at a boundary of memory: another start adds the same terms in another order, and
        # each order is within the bound of the 64-bit value
        got = KN.token_logprobs(x, tokens, top=4)
        lp, rank, ent, lse, ids, tl, te, ts = _scores(plain, tokens, 4)
        _close(got.logprob, lp, tl)
        _close(got.entropy, ent, te)
        _close(got.lse, lse, ts)
        assert torch.equal(got.rank, want.rank) and torch.equal(got.top_id, ids) and torch.equal(want.top_id, ids)
    e = plain[:1].expand(6, V)
    assert torch.equal(KN.token_logprobs(e, tokens).lse, want.lse[:1].expand(6))
    x = plain.clone().requires_grad_()
    r = KN.token_logprobs(x, tokens, top=4)
    gl, gh = torch.randn(6, 2, generator=g, device=DEV), torch.randn(6, generator=g, device=DEV)
    ((r.logprob * gl).sum() + (r.entropy * gh).sum()).backward()
    dx = KN.token_logprobs_grad(plain, tokens, want.lse, want.entropy, gl, gh)
    assert torch.equal(x.grad, dx) and not r.lse.requires_grad and not r.top_logprob.requires_grad
    only = torch.autograd.grad(KN.token_logprobs(x, tokens).entropy.sum(), x)[0]
    assert torch.equal(only, KN.token_logprobs_grad(plain, tokens, want.lse, want.entropy, None, torch.ones(6, device=DEV)))
    d, s = torch.randn(6, V, generator=g, device=DEV), 2.0 ** -7
    f = lambda y: (lambda q: (q.logprob.double() * gl).sum() + (q.entropy.double() * gh).sum())(KN.token_logprobs(y, tokens))  # noqa: E731
    diff = (f(plain + s * d) - f(plain - s * d)) / (2 * s)
    assert abs(diff - (dx.double() * d).sum()) <= 2e-3 * dx.double().norm() * d.double().norm()


def test_token_logprobs_empty_and_refusals():
    KN = _kn()
    x, t = torch.randn(4, 33, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    r = KN.token_logprobs(x[:0], t[:0], top=3)
    assert r.top_id.shape == (0, 3) and KN.token_logprobs_grad(x[:0], t[:0], r.lse, r.entropy).shape == (0, 33)
    for bad in (lambda: KN.token_logprobs(x, t, top=33), lambda: KN.token_logprobs(x, t, top=-1), lambda: KN.token_logprobs(x[0], t),
                lambda: KN.token_logprobs(x, t[:, None].expand(4, 65)), lambda: KN.token_logprobs(x[:, :0], t),
                lambda: KN.token_logprobs(x, t.cpu())):
        with pytest.raises(ValueError):
            bad()
    r = KN.token_logprobs(x, t)
    for bad in (lambda: KN.token_logprobs(x.double(), t), lambda: KN.token_logprobs(x, t.int()), lambda: KN.token_logprobs(x, t[:3]),
                lambda: KN.token_logprobs_grad(x, t, r.lse.double(), r.entropy),
                lambda: KN.token_logprobs_grad(x, t, r.lse, r.entropy, torch.ones(4, 1, device=DEV))):
        with pytest.raises(TypeError):
            bad()


def test_attention_offsets_past_32_bits():
    """A packed batch whose queries have more than 2^31 elements: its last sequences, with all their
    heads, come out as they do alone."""
    KN = _kn()
    H, Hk, D, tail = 34, 2, 64, [77, 16, 130]
    lens = [100] * 9990 + tail
    n = sum(lens)
    g = torch.Generator(device=DEV).manual_seed(0)
    mk = lambda h: torch.empty(1, h, n, D, dtype=torch.bfloat16, device=DEV).normal_(generator=g)  # noqa: E731
    q, k, v, do = mk(H), mk(Hk), mk(Hk), mk(H)
    assert q.numel() > 2 ** 31
    plan = KN.seq_maps(torch.tensor(lens, device=DEV), n).plan(0)
    out, lse = KN.attention(q, k, v, plan)
    grads = KN.attention_grad(do, q, k, v, out, lse, plan)
    m = sum(tail)
    cut = [x[:, :, -m:].contiguous() for x in (q, k, v, do)]
    few = KN.seq_maps(torch.tensor(tail, device=DEV), m).plan(0)
    o2, l2 = KN.attention(*cut[:3], few)
    want = (o2, l2, *KN.attention_grad(cut[3], *cut[:3], o2, l2, few))
    for a, b in zip((out, lse, *grads), want):
        assert torch.equal(a[:, :, -m:], b)


def test_token_logprobs_offsets_past_32_bits():
    """More than 2^31 logits: the last rows come out as they do alone."""
    KN = _kn()
    N, V, last = 31000, 70001, 500
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.empty(N, V, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    assert x.numel() > 2 ** 31
    tokens = torch.randint(0, V, (N, 2), generator=g, device=DEV)
    gl = torch.randn(N, 2, generator=g, device=DEV)
    r, w = KN.token_logprobs(x, tokens, top=3), KN.token_logprobs(x[-last:], tokens[-last:], top=3)
    for a, b in zip(r, w):
        assert torch.equal(a[-last:], b)
    dx = KN.token_logprobs_grad(x, tokens, r.lse, r.entropy, gl)
    dw = KN.token_logprobs_grad(x[-last:], tokens[-last:], w.lse, w.entropy, gl[-last:])
    assert torch.equal(dx[-last:], dw)


def test_two_streams_at_once():
    """Calls under way together share nothing: the results are those of calls one after the other."""
    KN = _kn()
    sets = [_batch([300, 5, 170], True, 4, 2, 64, dt, seed=s)[:5] for s, dt in ((1, torch.bfloat16), (2, torch.float16))]
    logits = [torch.randn(50, v, device=DEV) for v in (33, 20000)]
    tokens = torch.arange(50, device=DEV)

    def work(i):
        q, k, v, do, plan = sets[i]
        out, lse = KN.attention(q, k, v, plan)
        return [out, lse, *KN.attention_grad(do, q, k, v, out, lse, plan), *KN.token_logprobs(logits[i], tokens % 33, top=4)]

    want = [work(0), work(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(work(i))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_expanded_and_scaled_inputs(dtype):
    """Keys and values of one head expanded over the batch's key heads, a gradient that is one row
    expanded, and a scale of zero: the same as with the copies."""
    KN = _kn()
    q, k, v, do, plan, where, on = _batch([40, 129], True, 4, 1, 32, dtype, seed=8)
    ke, ve = k.expand(1, 2, -1, -1), v.expand(1, 2, -1, -1)
    de = do[:, :1, :1].expand_as(q)
    ref, tol = _plain(q, ke, ve, de, where, 32 ** -0.5)
    out, lse = KN.attention(q, ke, ve, plan)
    dq, dk, dv = KN.attention_grad(de, q, ke, ve, out, lse, plan)
    _check({"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}, ref, tol)
    ref, tol = _plain(q, k, v, do, where, 0.0)
    out, lse = KN.attention(q, k, v, plan, 0.0)
    dq, dk, dv = KN.attention_grad(do, q, k, v, out, lse, plan, 0.0)
    _check({"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}, ref, tol)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B", [1, 40])
def test_attention_of_empty_sequences_only(B, dtype, packed):
    """Nothing to attend to: zeros, from inputs that are NaN throughout."""
    KN = _kn()
    q, k, v, do, plan, _, on = _batch([0] * B, packed, 4, 2, 32, dtype, extra=7)
    assert not on.any() and q.isnan().all()
    out, lse = KN.attention(q, k, v, plan)
    for t in (out, lse, *KN.attention_grad(do, q, k, v, out, lse, plan)):
        assert (t == 0).all()

