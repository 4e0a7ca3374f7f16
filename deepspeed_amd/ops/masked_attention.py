"""Attention over packed rows (csrc/masked_attention.hip), forward and backward:
several documents beside one another in a row, prefixes that see themselves both
ways, scores capped by a tanh, a bias that falls with the distance. bf16, heads of 64,
96 and 128, grouped key heads; the single-token form over the paged pool is
``paged_attention.paged_decode_attention``."""

import math
from dataclasses import dataclass
from typing import Optional

import torch

from ._loader import get_ext
from .linear import untransformed


@dataclass
class PackedRows:
    """What the rows of a packed batch see, made once a batch by ``packed_rows`` and
    used by every layer. ``spans`` int32 [4, B, S]: the first key that a query sees and
    the one behind the last, the first query that sees a key and the one behind the
    last."""

    spans: torch.Tensor
    causal: bool


def _torch_spans(ids, prefix, causal):
    B, S = ids.shape
    at = torch.arange(S, device=ids.device).expand(B, S)
    begins = torch.ones_like(ids, dtype=torch.bool)
    begins[:, 1:] = ids[:, 1:] != ids[:, :-1]
    first = torch.where(begins, at, 0).cummax(1).values
    later = torch.where(begins, at, S).flip(1).cummin(1).values.flip(1)
    end = torch.full_like(at, S)
    end[:, :-1] = later[:, 1:]
    inside = first
    if prefix is not None:
        known = (ids >= 0) & (ids < prefix.shape[1])
        n = prefix.long().gather(1, torch.where(known, ids, 0).long()) \
            if prefix.shape[1] else torch.zeros_like(at)
        inside = first + torch.where(known, n, 0).clamp(min=0).minimum(end - first)
    if causal:
        spans = [first, torch.maximum(at + 1, inside),
                 torch.where(at >= inside, at, first), end]
    else:
        spans = [first, end, first, end]
    return torch.stack([torch.where(ids < 0, at, s) for s in spans]).int()


def packed_rows(document_ids: torch.Tensor,
                prefix_lens: Optional[torch.Tensor] = None,
                causal: bool = True) -> PackedRows:
    """``document_ids`` [B, S] int32 or int64: a document is a run of one id, and its
    tokens see that document alone; rows of a negative id (padding) see nothing and
    are seen by none. ``prefix_lens`` [B, N] (causal only): the first ``prefix_lens[b,
    d]`` tokens of the documents of id d are seen by all of their document; ids from N
    on have no prefix."""
    if document_ids.dim() != 2 or document_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError("packed_rows: document_ids is int32 or int64 [B, S], got "
                         f"{document_ids.dtype} {tuple(document_ids.shape)}")
    if prefix_lens is not None:
        if not causal:
            raise ValueError("packed_rows: without causal there is no prefix")
        if prefix_lens.dim() != 2 or prefix_lens.dtype not in (
                torch.int32, torch.int64) or \
                prefix_lens.shape[0] != document_ids.shape[0]:
            raise ValueError("packed_rows: prefix_lens is int32 or int64 [B, N]")
        if prefix_lens.device != document_ids.device:
            raise ValueError("packed_rows: tensors on different devices")
    if document_ids.is_cuda and get_ext() is not None and untransformed():
        prefix = prefix_lens
        if prefix is not None:
            if prefix.dtype is torch.int64:       # no length wraps to another
                prefix = prefix.clamp(0, document_ids.shape[1]).int()
            prefix = prefix.contiguous()
        spans = get_ext().packed_spans(document_ids.contiguous(), prefix, causal)
    else:
        spans = _torch_spans(document_ids, prefix_lens, causal)
    return PackedRows(spans, causal)


def _formulas(q, k, v, far, seen, scale, softcap, slopes):
    """q [B, Sq, H, D], k and v [B, Sk, Hkv, D] of one type, far [Sq, Sk] the distances,
    ``seen`` [B or 1, 1, Sq, Sk] or None (all)."""
    G = q.shape[2] // k.shape[2]
    q, k, v = (x.transpose(1, 2) for x in (q, k, v))
    k, v = (x.repeat_interleave(G, 1) for x in (k, v))
    t = (q @ k.transpose(2, 3).contiguous()) * scale
    if softcap:
        t = torch.tanh(t / softcap) * softcap
    if slopes is not None:
        t = t - slopes.to(t.dtype).view(-1, 1, 1) * far
    if seen is None:
        return (torch.softmax(t, -1) @ v).transpose(1, 2)
    t = t.masked_fill(~seen, -math.inf)
    top = t.amax(-1, keepdim=True).detach()
    some = seen.any(-1, keepdim=True)
    p = torch.exp(t - torch.where(some, top, 0.0))
    p = torch.where(seen, p, 0.0)
    p = p / torch.where(some, p.sum(-1, keepdim=True), 1.0)
    return (p @ v).transpose(1, 2)


def _torch_attention(q, k, v, spans, causal, scale, softcap, slopes):
    """The formulas in fp32 (fp64 for fp64), on whole score matrices. What is hidden is
    in no sum, as in the kernels: rows of no use count as 0, and if others are not finite
    each query goes through its own keys alone. Not so where there are no values to look
    at, under a transform, and not for gradients that come in so to rows of use."""
    B, S, _, _ = q.shape
    kind, wide = q.dtype, torch.float64 if q.dtype is torch.float64 else torch.float32
    q, k, v = (x.to(wide) for x in (q, k, v))
    at = torch.arange(S, device=q.device)
    far = (at[:, None] - at).abs()
    how = scale, softcap, slopes
    if S == 0 or spans is None and not causal:
        return _formulas(q, k, v, far, None, *how).to(kind)
    if spans is not None:
        lo, hi, klo, khi = spans[..., None]
        seen = ((at >= lo) & (at < hi))[:, None]
        used = (lo < hi)[..., None]
        q = torch.where(used, q, 0.0)
        k, v = (torch.where((klo < khi)[..., None], x, 0.0) for x in (k, v))
    else:
        seen = (at <= at[:, None])[None, None]
        used = torch.ones_like(at, dtype=torch.bool)[:, None, None]
    if torch.compiler.is_compiling() or not untransformed() or q.is_meta or \
            all(bool(torch.isfinite(x).all()) for x in (q, k, v)):
        o = _formulas(q, k, v, far, seen, *how)
    else:
        ends = torch.stack([0 * at, at + 1], -1).expand(B, S, 2) if spans is None \
            else spans[:2].permute(1, 2, 0).clamp(0, S)
        rows = [_formulas(q[b:b + 1, i:i + 1], k[b:b + 1, lo:hi], v[b:b + 1, lo:hi],
                          far[i:i + 1, lo:hi], None, *how)
                if lo < hi else torch.zeros_like(q[b:b + 1, i:i + 1])
                for b, row in enumerate(ends.tolist()) for i, (lo, hi) in enumerate(row)]
        o = torch.cat(rows, 1).view(q.shape)
    return torch.where(used, o, 0.0).to(kind)


def _checked_slopes(alibi_slopes, q, what):
    if alibi_slopes is None:
        return None
    if alibi_slopes.requires_grad:
        raise ValueError(f"{what}: alibi_slopes have no gradient")
    if alibi_slopes.shape != (q.shape[-2],) or \
            not alibi_slopes.dtype.is_floating_point:
        raise ValueError(f"{what}: alibi_slopes is one number a query head, got "
                         f"{alibi_slopes.dtype} {tuple(alibi_slopes.shape)}")
    if alibi_slopes.device != q.device:
        raise ValueError(f"{what}: tensors on different devices")
    return alibi_slopes.float().contiguous()


def _checked_cap(softcap, what):
    softcap = float(softcap or 0.0)
    if softcap != 0.0 and not 1e-30 < softcap < 1e30:
        raise ValueError(f"{what}: softcap is 0 (none) or positive, got {softcap}")
    return softcap


def masked_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                     rows: Optional[PackedRows] = None, causal: bool = True,
                     scale: Optional[float] = None, softcap: float = 0.0,
                     alibi_slopes: Optional[torch.Tensor] = None) -> torch.Tensor:
    """q [B, S, H, D], k and v [B, S, Hkv, D] -> [B, S, H, D], differentiable in q, k
    and v (once). Scores ``scale q k`` (default 1 / sqrt(D)), with ``softcap`` c
    then c tanh(score / c), with ``alibi_slopes`` [H] less slope times the distance of
    query and key, softmax over the keys that a query sees: those of ``rows``, or
    without them by ``causal`` all up to its own or all there are. A query that sees
    none gives 0 and has no gradient. On a GPU bf16 and heads of 64, 96 or 128; scores and
    a row's log of their sum are fp32 there, so that gradients lose digits with scores
    past 1e5 and results with such past 1e9, unless a cap holds them."""
    ext = get_ext()
    if q.is_cuda and ext is not None and untransformed():
        spans, causal = (None, causal) if rows is None else (rows.spans, rows.causal)
        return ext.masked_attention(q, k, v, spans, alibi_slopes, causal, scale,
                                    softcap or 0.0)
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or \
            q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3] or \
            0 in (q.shape[2], k.shape[2]) or q.shape[2] % k.shape[2]:
        raise ValueError("masked_attention: q is [B, S, H, D], k and v are [B, S, Hkv, "
                         "D] with H a multiple of Hkv, got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if not q.dtype == k.dtype == v.dtype:
        raise ValueError("masked_attention: q, k and v of one type")
    if rows is not None and (rows.spans.shape[1:] != q.shape[:2]
                             or rows.spans.device != q.device):
        raise ValueError("masked_attention: rows of another batch or device: "
                         f"{tuple(rows.spans.shape)} for q {tuple(q.shape)}")
    softcap = _checked_cap(softcap, "masked_attention")
    slopes = _checked_slopes(alibi_slopes, q, "masked_attention")
    spans, causal = (rows.spans, rows.causal) if rows is not None else (None, causal)
    scale = scale if scale is not None else 1.0 / math.sqrt(q.shape[3])
    return _torch_attention(q, k, v, spans, causal, scale, softcap, slopes)
