"""Tensor-level wrappers over the C ABI, one per kernel, plus the reference's kernel-level functions
(`filter_candidates`, `sub_stats`, `gram_accumulate`, `grouped_merge`) with the same arguments,
results and error behaviour as haelyons/proteus atlas/filter_triton.py, atlas/stats_triton.py and
atlas/core.py:75-104 — backed only by the sm_100a library (no fallback).
"""
from __future__ import annotations

import struct
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import call, dtype_code, launch, ptr, require_cuda, stream_ptr

I64_MIN = torch.iinfo(torch.int64).min


def _i32(t):
    return t if t.dtype == torch.int32 else t.to(torch.int32)


def round_up(x: int, m: int) -> int:
    return (x + m - 1) // m * m


# ----------------------------------------------------------------------------- K1 filter
def filter_compact(H, rowmap32, thr_pos, thr_neg, out_val, out_row, out_col, count, cap):
    """atlas_filter_compact on preallocated buffers (count must be zero on entry)."""
    T, D = H.shape
    call("atlas_filter_compact", ptr(H), dtype_code(H.dtype), T, D, H.stride(0), ptr(rowmap32), ptr(thr_pos),
         ptr(thr_neg), ptr(out_val), ptr(out_row), ptr(out_col), ptr(count), int(cap), stream_ptr(H.device))


def filter_candidates(H, rowmap, thr_pos, thr_neg, max_out, **_tile):
    """Drop-in for filter_triton.filter_candidates (filter_triton.py:65-86): returns
    (vals fp32 [max_out], rows int64, cols int64, count 0-d device tensor); count > max_out means
    overflow. Tile arguments of the Triton version are accepted and ignored."""
    require_cuda(H, "H")
    assert H.stride(1) == 1
    dev = H.device
    out_val = torch.empty(max_out, device=dev, dtype=torch.float32)
    out_row = torch.empty(max_out, device=dev, dtype=torch.int32)
    out_col = torch.empty(max_out, device=dev, dtype=torch.int32)
    counter = torch.zeros(1, device=dev, dtype=torch.int32)
    filter_compact(H, _i32(rowmap), thr_pos.contiguous().float(), thr_neg.contiguous().float(), out_val, out_row,
                   out_col, counter, max_out)
    return out_val, out_row.long(), out_col.long(), counter[0]


# ----------------------------------------------------------------------------- gathers / stats
def gather_transpose(H, rows32, XT, col0: int):
    T, D = H.shape
    call("atlas_gather_transpose", ptr(H), dtype_code(H.dtype), T, D, H.stride(0), ptr(rows32), rows32.numel(),
         ptr(XT), XT.stride(0), int(col0), stream_ptr(H.device))


def gather_rows(H, rows32, R):
    T, D = H.shape
    call("atlas_gather_rows", ptr(H), dtype_code(H.dtype), T, D, H.stride(0), ptr(rows32), rows32.numel(), ptr(R),
         stream_ptr(H.device))


def sub_stats_into(XT, col0, n, E0, E1, levels, sum_, sq, bins, masks, n_pad):
    """Accumulate subsample statistics of XT[:, col0:col0+n] into (sum_, sq, bins) and write masks."""
    import ctypes
    D = XT.shape[0]
    B = E0.shape[1]
    NL = len(levels)
    lev = (ctypes.c_int32 * max(NL, 1))(*levels) if NL else None
    call("atlas_sub_stats", ptr(XT), dtype_code(XT.dtype), XT.stride(0), int(col0), int(n), D, ptr(E0), ptr(E1), B,
         ctypes.cast(lev, ctypes.c_void_p) if lev is not None else None, NL, ptr(sum_), ptr(sq), ptr(bins),
         ptr(masks) if NL else None, int(n_pad), stream_ptr(XT.device))


def stats_enrich_supported(dtype, B: int, NL: int, A_pad: int) -> bool:
    return bool(_lib.load().atlas_stats_enrich_supported(dtype_code(dtype), B, NL, A_pad))


class StatsEnrichWorkspace:
    """Zero-filled device workspace of atlas_sub_stats_enrich (range partials of the column sums and
    per-column-tile tickets), grown on demand."""

    def __init__(self, device):
        self.device = device
        self.buf = None

    def get(self, D: int, n: int) -> torch.Tensor:
        need = int(_lib.load().atlas_stats_enrich_ws_bytes(D, n))
        if self.buf is None or self.buf.numel() < need:
            self.buf = torch.zeros(need, dtype=torch.uint8, device=self.device)
        return self.buf


def sub_stats_enrich_into(XT, col0, n, E0, E1, levels, sum_, sq, bins, annT, enr, A, ws: StatsEnrichWorkspace):
    """Fused atlas_sub_stats_enrich over XT[:, col0:col0+n]: moments and bin masses of the columns
    and the enrichment contingencies enr [2*NL*D, A] += masks . annT^T, masks never materialised."""
    import ctypes
    D = XT.shape[0]
    B = E0.shape[1]
    NL = len(levels)
    lev = (ctypes.c_int32 * NL)(*levels)
    w = ws.get(D, n)
    call("atlas_sub_stats_enrich", ptr(XT), dtype_code(XT.dtype), XT.stride(0), int(col0), int(n), D, ptr(E0), ptr(E1),
         B, ctypes.cast(lev, ctypes.c_void_p), NL, ptr(sum_), ptr(sq), ptr(bins), ptr(annT), annT.shape[0],
         annT.shape[1], ptr(enr), int(A), ptr(w), w.numel(), stream_ptr(XT.device))


def sub_stats(X, E0, E1, levels, **_tile):
    """Drop-in for stats_triton.sub_stats (stats_triton.py:77-117): X [n, D] (unit column stride);
    returns (sum fp64 [D], sumsq fp64 [D], counts int32 [2, D, B], masks int8 [2, NL, D, n8])."""
    require_cuda(X, "X")
    assert X.stride(1) == 1
    n, D = X.shape
    B = E0.shape[1]
    NL = len(levels)
    n8 = round_up(n, 8)
    dev = X.device
    XT = torch.empty(D, max(n8, 8), device=dev, dtype=X.dtype)
    if n:
        gather_transpose(X, torch.arange(n, device=dev, dtype=torch.int32), XT, 0)
    s = torch.zeros(D, device=dev, dtype=torch.float64)
    sq = torch.zeros(D, device=dev, dtype=torch.float64)
    bins = torch.zeros(2, D, B, device=dev, dtype=torch.int64)
    masks = torch.zeros(2, max(NL, 1), D, max(n8, 8), device=dev, dtype=torch.int8)
    if n:
        sub_stats_into(XT, 0, n, E0.contiguous().float(), E1.contiguous().float(), list(levels), s, sq, bins, masks,
                       masks.shape[-1])
    return s, sq, bins.to(torch.int32), masks[:, :NL, :, :n8]


def count_gemm_i8(masks2d, annT, out, A: int):
    """out[M, A] (int64) += masks2d[M, n_pad] @ annT[A_pad, n_pad]^T, exact."""
    M, n_pad = masks2d.shape
    call("atlas_count_gemm_i8", ptr(masks2d), M, n_pad, ptr(annT), annT.shape[0], ptr(out), int(A),
         stream_ptr(masks2d.device))


def gram_upper(XT, n: int, C):
    """C[D, D] += XT[:, :n] XT[:, :n]^T on the upper 128-block triangle."""
    D = XT.shape[0]
    call("atlas_gram_upper", ptr(XT), dtype_code(XT.dtype), XT.stride(0), int(n), D, ptr(C), stream_ptr(XT.device))


def gram_accumulate(X, C, **_tile):
    """Drop-in for stats_triton.gram_accumulate (stats_triton.py:148-169): C [D, D] fp32 contiguous
    += X^T X on the upper block triangle (blocks of 128), in place; returns C."""
    require_cuda(X, "X")
    assert X.stride(1) == 1 and C.is_contiguous() and C.dtype == torch.float32
    n, D = X.shape
    if n == 0:
        return C
    n8 = round_up(n, 8)
    XT = torch.empty(D, n8, device=X.device, dtype=X.dtype)
    gather_transpose(X, torch.arange(n, device=X.device, dtype=torch.int32), XT, 0)
    gram_upper(XT, n, C)
    return C


# ----------------------------------------------------------------------------- merges
class MergeWorkspace:
    """Device scratch of atlas_grouped_merge, grown on demand and reused."""

    def __init__(self, device):
        self.device = torch.device(device)
        self.G = self.n = -1
        self.i32 = None
        self.bytes = None

    def get(self, G: int, n_max: int):
        lib = _lib.load()
        need_i = lib.atlas_merge_ws_i32(G, n_max)
        need_b = lib.atlas_merge_ws_bytes(n_max)
        if self.i32 is None or self.i32.numel() < need_i:
            self.i32 = torch.empty(int(need_i * 1.25) + 64, device=self.device, dtype=torch.int32)
        if self.bytes is None or self.bytes.numel() < need_b:
            self.bytes = torch.empty(int(need_b * 1.25) + 256, device=self.device, dtype=torch.uint8)
        return self.i32, self.bytes


_WS: dict = {}


def grouped_merge_records(state_sc, state_tok, state_val, K, g, sc, tok, val, n_dev, n_max, ws: MergeWorkspace = None):
    G = state_sc.shape[0]
    if ws is None:
        ws = _WS.setdefault(state_sc.device, MergeWorkspace(state_sc.device))
    wi, wb = ws.get(G, n_max)
    call("atlas_grouped_merge", ptr(state_sc), ptr(state_tok), ptr(state_val), G, int(K), ptr(g), ptr(sc), ptr(tok),
         ptr(val), ptr(n_dev), int(n_max), ptr(wi), ptr(wb), stream_ptr(state_sc.device))


def grouped_merge(state_score, state_pay, g, score, pay, K, pay_fill=None):
    """Drop-in for core.grouped_merge (core.py:75-104) for int64 scores with payloads
    (int64, fp32): merges candidates into the per-group top-K in place. Returns the number of
    candidates (the reference returns the number of touched groups, which needs a host sync)."""
    require_cuda(state_score, "state_score")
    assert state_score.dtype == torch.int64 and len(state_pay) == 2
    n = g.numel()
    if n == 0:
        return 0
    dev = state_score.device
    n_dev = torch.tensor([n], device=dev, dtype=torch.int32)
    grouped_merge_records(state_score, state_pay[0], state_pay[1], K, _i32(g).contiguous(), score.contiguous(),
                          pay[0].to(torch.int64).contiguous(), pay[1].to(torch.float32).contiguous(), n_dev, n)
    return n


def merge_rows(sc, tok, val, osc, otok, oval):
    G, K = sc.shape
    call("atlas_merge_rows", ptr(sc), ptr(tok), ptr(val), ptr(osc), ptr(otok), ptr(oval), G, K, stream_ptr(sc.device))


# ----------------------------------------------------------------------------- a model's batches and answers
def _same_device(first, **others):
    for name, t in others.items():
        if t.device != first.device:
            raise ValueError(f"{name} is on {t.device}, the first argument on {first.device}")


def _refuse_tangents(**tensors):
    """Forward-mode derivatives: a dual tensor has no requires_grad, and its result would come without a tangent. Called
    where a dual level is open (_current_level, 0.06 us to look at; unpack_dual takes 0.8 us a tensor)."""
    for name, t in tensors.items():
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name} carries a forward-mode tangent: only reverse-mode gradients are supported")


class SeqPlan(NamedTuple):
    """Which rows of a batch's tensors belong to which sequence, as attention reads it: `cu` int32
    [B + 1] prefix sums of the lengths, `blocks` int32 [n, 2] and `counts` int64 [3] of seq_maps, and
    `stride`, the rows of each sequence in a padded batch (0: packed end to end). Attention passes over
    entries of another table that name no sequence of the batch or a first position that is not a multiple
    of 128, and leaves the rows of an entry that is missing as they were."""
    cu: torch.Tensor
    blocks: torch.Tensor
    counts: torch.Tensor
    stride: int


class SeqMaps(NamedTuple):
    """Result of seq_maps (see there)."""
    cu: torch.Tensor
    slots: torch.Tensor
    tok: torch.Tensor
    blocks: torch.Tensor
    counts: torch.Tensor

    def plan(self, stride: int) -> SeqPlan:
        return SeqPlan(self.cu, self.blocks, self.counts, int(stride))


def seq_maps(lengths, n_rows: int, *, stride: int = 0, lead: int = 0, trail: int = 0, seq=None) -> SeqMaps:
    """The row maps of a batch, built on the device from its sequences' lengths without a host read:
    `lengths` int32 or int64 [B] counts every row of a sequence, special tokens included; the batch's
    tensors have `n_rows` rows, sequence b at row b*stride (padded, stride > 0) or right behind the one
    before it (packed, stride 0). `lead` and `trail` positions at a sequence's start and end (<cls>,
    <eos>) get no slot. Returns SeqMaps:

      cu     int32 [B + 1]                    prefix sums of the lengths
      slots  int64 [n_rows]                   rows of the kept positions, in order (a batch's valid rows)
      tok    int64 [n_rows]                   their token ids: pack_tok(seq[b], position - lead); seq None: b
      blocks int32 [n_rows // 128 + B + 1, 2] (sequence, first position) of every 128 positions
      counts int64 [3]                        kept positions, blocks, lengths that did not fit

    slots, tok and blocks are -1 behind their last entry. A length outside [0, stride] (packed:
    [0, n_rows]) is cut and counted in counts[2]; packed sequences that together do not fit are all
    taken as empty, which counts once more."""
    require_cuda(lengths, "lengths")
    dt, dev = lengths.dtype, lengths.device
    if lengths.dim() != 1 or dt not in (torch.int32, torch.int64):
        raise TypeError(f"lengths must be int32 or int64 [B], got {dt} {list(lengths.shape)}")
    B = lengths.shape[0]
    if n_rows < 1 or stride < 0 or lead < 0 or trail < 0 or stride * B > n_rows:
        raise ValueError(f"{B} sequences of stride {stride} (lead {lead}, trail {trail}) do not fit {n_rows} rows")
    if seq is not None:
        if seq.device != dev:
            _same_device(lengths, seq=seq)
        if seq.shape != lengths.shape or seq.dtype != torch.int64:
            raise TypeError(f"seq must be int64 [{B}], got {seq.dtype} {list(seq.shape)}")
        seq = seq.contiguous()
    lengths = lengths.contiguous()
    cap = n_rows // 128 + B + 1
    if B == 0:
        none = torch.full((n_rows,), -1, dtype=torch.int64, device=dev)
        return SeqMaps(torch.zeros(1, dtype=torch.int32, device=dev), none, none.clone(),
                       torch.full((cap, 2), -1, dtype=torch.int32, device=dev), torch.zeros(3, dtype=torch.int64, device=dev))
    # new_empty without a dtype is the cheapest allocation: 1.3 us of the host's instead of 2.3
    cu = torch.empty(B + 1, dtype=torch.int32, device=dev)
    slots = torch.empty(n_rows, dtype=torch.int64, device=dev)
    blocks, tok, counts = cu.new_empty((cap, 2)), slots.new_empty(n_rows), slots.new_empty(3)
    need = _lib.load().atlas_seq_maps_ws_bytes(B)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    launch(dev, "atlas_seq_maps", lengths.data_ptr(), int(dt == torch.int64), B, n_rows, stride, lead, trail, ptr(seq),
           cu.data_ptr(), slots.data_ptr(), tok.data_ptr(), blocks.data_ptr(), counts.data_ptr(), ptr(ws), need)
    return SeqMaps(cu, slots, tok, blocks, counts)


def _rows_like(t, heads: int):
    """An uninitialised [outer, heads, rows, D] tensor whose memory is [outer, rows, heads, D], the
    layout the next projection reads."""
    o, _, n, d = t.shape
    return t.new_empty_strided((o, heads, n, d), (n * heads * d, d, heads * d, 1))


def _unit(t):
    return t if t.stride(-1) == 1 else t.contiguous()


def _strides(*ts):
    """The (outer, head, row) strides of the tensors as the host array the C ABI takes."""
    return struct.pack(f"{3 * len(ts)}q", *[x for t in ts for x in t.stride()[:3]])


def _check_attention(q, k, v, plan):
    """Shapes (outer, H, rows, D), key heads and batch of an attention call, or an error that names what is wrong."""
    require_cuda(q, "q")
    cu, blocks, counts, stride = plan
    dev = q.device
    if not (k.device == dev and v.device == dev and cu.device == dev and blocks.device == dev and counts.device == dev):
        _same_device(q, k=k, v=v, cu=cu, blocks=blocks, counts=counts)
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4 or ks != v.shape or qs[0] != ks[0] or qs[2:] != ks[2:]:
        raise ValueError(f"q [outer, H, rows, D], k and v [outer, Hk, rows, D]: got {list(qs)}, {list(ks)}, {list(v.shape)}")
    if not q.dtype == k.dtype == v.dtype:
        raise TypeError(f"q, k and v must have one dtype, got {q.dtype}, {k.dtype}, {v.dtype}")
    (o, h, n, d), hk, B, bs = qs, ks[1], cu.shape[0] - 1, blocks.shape
    if not 1 <= d <= 64:
        raise ValueError(f"head dimension {d}: 1 to 64 are supported")
    if hk < 1 or h % hk:
        raise ValueError(f"{h} query heads over {hk} key heads: not a multiple")
    if B < 0 or cu.dtype != torch.int32 or blocks.dtype != torch.int32 or counts.dtype != torch.int64 or len(bs) != 2 or \
            bs[1] != 2 or counts.shape != (3,):
        raise TypeError("plan: cu int32 [B + 1], blocks int32 [n, 2], counts int64 [3] (seq_maps)")
    if stride == 0 and o != 1:
        raise ValueError(f"a packed batch has one outer index, got {o}")
    if stride and (o != B or n != stride):
        raise ValueError(f"a padded batch of {B} sequences of stride {stride} against q {list(qs)}")
    if bs[0] < o * n // 128 + B + 1:
        raise ValueError(f"plan of {bs[0]} blocks: too few for {o * n} rows")
    return o, h, n, d, hk, B


def _attention_forward(q, k, v, plan, scale):
    o, h, n, d, hk, B = _check_attention(q, k, v, plan)
    dev = q.device
    out, lse = _rows_like(q, h), q.new_empty((o, h, n), dtype=torch.float32)
    if B == 0 or out.numel() == 0:
        return out.zero_(), lse.zero_()
    q, k, v = _unit(q), _unit(k), _unit(v)
    cu, blocks, counts = plan.cu.contiguous(), plan.blocks.contiguous(), plan.counts.contiguous()
    launch(dev, "atlas_attention", q.data_ptr(), k.data_ptr(), v.data_ptr(), dtype_code(q.dtype), _strides(q, k, v, out), o, n, h, hk,
           d, cu.data_ptr(), blocks.data_ptr(), counts.data_ptr(), B, blocks.shape[0], int(plan.stride == 0), scale, out.data_ptr(),
           lse.data_ptr())
    return out, lse


def attention_grad(dout, q, k, v, out, lse, plan: SeqPlan, scale: float | None = None):
    """(dq, dk, dv) of attention(q, k, v, plan, scale) for the gradient `dout` of its output: the
    probabilities are computed again from `lse`, the keys' gradients summed over the query heads that
    share them. No atomics on them: the same call gives the same bits. Rows of no sequence come out as zero."""
    if forward_ad._current_level >= 0:
        _refuse_tangents(dout=dout, q=q, k=k, v=v, out=out, lse=lse)
    o, h, n, d, hk, B = _check_attention(q, k, v, plan)
    dev = q.device
    if not (dout.device == dev and out.device == dev and lse.device == dev):
        _same_device(q, dout=dout, out=out, lse=lse)
    if dout.shape != q.shape or out.shape != q.shape or lse.shape != q.shape[:3]:
        raise ValueError(f"dout and out must be {list(q.shape)}, lse {list(q.shape[:3])}")
    if dout.dtype != q.dtype or out.dtype != q.dtype or lse.dtype != torch.float32:
        raise TypeError(f"dout and out must be {q.dtype}, lse float32")
    scale = d ** -0.5 if scale is None else float(scale)
    dq, dk, dv = _rows_like(q, h), _rows_like(k, hk), _rows_like(v, hk)
    if B == 0 or dq.numel() == 0:
        return dq.zero_(), dk.zero_(), dv.zero_()
    ws = torch.empty(int(_lib.load().atlas_attention_grad_ws_bytes(o, n, h, hk, B)), dtype=torch.uint8, device=dev)
    dout, q, k, v, out, lse = _unit(dout), _unit(q), _unit(k), _unit(v), _unit(out), lse.contiguous()
    cu, blocks, counts = plan.cu.contiguous(), plan.blocks.contiguous(), plan.counts.contiguous()
    launch(dev, "atlas_attention_grad", dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
           dtype_code(q.dtype), _strides(dout, q, k, v, out, dq, dk, dv), o, n, h, hk, d, cu.data_ptr(), blocks.data_ptr(),
           counts.data_ptr(), B, blocks.shape[0], int(plan.stride == 0), scale, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
           ws.data_ptr(), ws.shape[0])
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu, blocks, counts, stride, scale):
        plan = SeqPlan(cu, blocks, counts, stride)
        out, lse = _attention_forward(q, k, v, plan, scale)
        ctx.save_for_backward(q, k, v, out, lse, cu, blocks, counts)
        ctx.stride, ctx.scale = stride, scale
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _dlse):
        q, k, v, out, lse, cu, blocks, counts = ctx.saved_tensors
        return *attention_grad(dout, q, k, v, out, lse, SeqPlan(cu, blocks, counts, ctx.stride), ctx.scale), *[None] * 5


def attention(q, k, v, plan: SeqPlan, scale: float | None = None):
    """Attention over the valid rows of a batch: every row of a sequence attends to every row of the
    same sequence. q [outer, H, rows, D] and k, v [outer, Hk, rows, D] (bf16, fp16 or fp32, any strides,
    D <= 64, query head h reads key head h // (H // Hk)); a padded batch has outer = B and rows =
    plan.stride, a packed one outer = 1. scale: D ** -0.5 if not given. Returns out (q's shape, memory
    [outer, rows, H, D]) and the log-sum-exp of the scores, fp32 [outer, H, rows]; both zero in rows of
    no sequence, whose inputs are never read (they may hold NaN). Differentiable in q, k and v (not
    through the log-sum-exp), once. A query whose scores are all -inf has log-sum-exp -inf and an output of
    NaN. A backward pass that goes into a CUDA graph calls attention_grad: autograd's own must not be captured
    while an eager graph of the same leaves is alive. Tensors with a forward-mode tangent are refused."""
    if forward_ad._current_level >= 0:
        _refuse_tangents(q=q, k=k, v=v)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _Attention.apply(q, k, v, plan.cu, plan.blocks, plan.counts, plan.stride, scale)
    return _attention_forward(q, k, v, plan, scale)


class TokenLogprobs(NamedTuple):
    """Result of token_logprobs (see there)."""
    logprob: torch.Tensor
    rank: torch.Tensor
    entropy: torch.Tensor
    lse: torch.Tensor
    top_id: torch.Tensor
    top_logprob: torch.Tensor


def _check_logits(logits, tokens):
    """N, V and the tokens of a row, or an error that names what is wrong."""
    require_cuda(logits, "logits")
    if tokens.device != logits.device:
        _same_device(logits, tokens=tokens)
    shape, given = logits.shape, tokens.shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError(f"logits must be [N, V] with V >= 1, got {list(shape)}")
    if tokens.dtype != torch.int64 or not 1 <= len(given) <= 2 or given[0] != shape[0]:
        raise TypeError(f"tokens must be int64 [N] or [N, J], got {tokens.dtype} {list(given)}")
    J = given[1] if len(given) == 2 else 1
    if J > 64:
        raise ValueError(f"{J} tokens a row: at most 64")
    return *shape, J


def _plain_rows(t, N, V):
    """t [N, V] with unit column stride and rows that do not overlap (an expanded row is copied out), and its
    row stride (of a single row, whatever that says, the row's length)."""
    s0, s1 = t.stride()
    if (s1 == 1 or V == 1) and (N <= 1 or s0 >= V):
        return t, max(s0, V)
    return t.contiguous(), V


def _token_logprobs_forward(logits, tokens, top):
    N, V, J = _check_logits(logits, tokens)
    dt, dev = dtype_code(logits.dtype), logits.device
    if not 0 <= top <= min(32, V):
        raise ValueError(f"top must be in [0, min(32, V)], got {top} for V = {V}")
    (logits, ld), tokens = _plain_rows(logits, N, V), tokens.contiguous()
    # new_empty without a dtype is the cheapest allocation: 1.3 us of the host's instead of 2.3
    shape = tokens.shape
    rank, top_id = torch.empty(shape, dtype=torch.int32, device=dev), tokens.new_empty((N, top))
    logprob = torch.empty(shape, dtype=torch.float32, device=dev)
    entropy, lse, top_logprob = logprob.new_empty(N), logprob.new_empty(N), logprob.new_empty((N, top))
    if N:
        launch(dev, "atlas_token_logprobs", logits.data_ptr(), dt, N, V, ld, tokens.data_ptr(), J, top, logprob.data_ptr(),
               rank.data_ptr(), entropy.data_ptr(), lse.data_ptr(), top_id.data_ptr(), top_logprob.data_ptr())
    return TokenLogprobs(logprob, rank, entropy, lse, top_id, top_logprob)


def _row_vector(logits, name, t, shape):
    if t.device != logits.device:
        _same_device(logits, **{name: t})
    if t.dtype != torch.float32 or t.shape != shape:
        raise TypeError(f"{name} must be float32 {list(shape)}, got {t.dtype} {list(t.shape)}")
    return t.contiguous()


def token_logprobs_grad(logits, tokens, lse, entropy, g_logprob=None, g_entropy=None):
    """Gradient by the logits, [N, V] in their dtype, of sum(g_logprob * logprob) + sum(g_entropy *
    entropy), from token_logprobs' lse and entropy. Either gradient may be None. A token given twice
    in a row counts twice; one outside [0, V) not at all."""
    if forward_ad._current_level >= 0:
        _refuse_tangents(logits=logits, lse=lse, entropy=entropy, g_logprob=g_logprob, g_entropy=g_entropy)
    N, V, J = _check_logits(logits, tokens)
    dt, dev = dtype_code(logits.dtype), logits.device
    lse, entropy = _row_vector(logits, "lse", lse, (N,)), _row_vector(logits, "entropy", entropy, (N,))
    if g_logprob is not None:
        g_logprob = _row_vector(logits, "g_logprob", g_logprob, tokens.shape)
    if g_entropy is not None:
        g_entropy = _row_vector(logits, "g_entropy", g_entropy, (N,))
    (logits, ld), tokens = _plain_rows(logits, N, V), tokens.contiguous()
    dx = logits.new_empty((N, V))
    if N:
        launch(dev, "atlas_token_logprobs_grad", logits.data_ptr(), dt, N, V, ld, tokens.data_ptr(), J, lse.data_ptr(),
               entropy.data_ptr(), ptr(g_logprob), ptr(g_entropy), dx.data_ptr(), V)
    return dx


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top):
        r = _token_logprobs_forward(logits, tokens, top)
        ctx.save_for_backward(logits, tokens, r.lse, r.entropy)
        ctx.mark_non_differentiable(r.rank, r.lse, r.top_id, r.top_logprob)
        ctx.set_materialize_grads(False)
        return tuple(r)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logprob, _rank, g_entropy, *_rest):
        return token_logprobs_grad(*ctx.saved_tensors, g_logprob, g_entropy), None, None


def token_logprobs(logits, tokens, top: int = 0) -> TokenLogprobs:
    """What a model answers at each row of `logits` [N, V] (bf16, fp16 or fp32; any row stride): for
    `tokens` int64 [N] or [N, J] (J <= 64) their log probability (fp32) and rank (int32, 1 + how many
    logits are larger), the row's entropy and log-sum-exp (fp32 [N]), and the `top` (<= 32) most likely
    tokens (top_id int64, top_logprob fp32 [N, top]; ties to the lowest id). A token outside [0, V)
    means none: log probability 0, rank 0. A row of -inf only has log probabilities -inf and entropy 0.
    logprob and entropy are differentiable in the logits, once; a backward pass that goes into a CUDA graph calls
    token_logprobs_grad, as with attention. Logits with a forward-mode tangent are refused."""
    if forward_ad._current_level >= 0:
        _refuse_tangents(logits=logits)
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobs.apply(logits, tokens, top))
    return _token_logprobs_forward(logits, tokens, top)
