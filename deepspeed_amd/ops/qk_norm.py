"""RMS norms of the queries' and keys' heads with the position rotation behind them
(csrc/qk_norm.hip), forward and backward: one launch between a layer's joint
projection and its attention."""

from typing import Optional, Tuple

import torch

from ._loader import get_ext
from .linear import untransformed

LAYOUTS = ("half", "interleaved")


def _torch_heads(x, weight, cos, sin, positions, eps, layout, one_plus):
    """The formulas in fp32 (fp64 for fp64)."""
    wide = torch.float64 if x.dtype is torch.float64 else torch.float32
    B, S, _, D = x.shape
    n = 2 * cos.shape[1]
    at = torch.arange(S, device=x.device).expand(B, S) if positions is None \
        else positions.reshape(B, S).long()
    there = (at >= 0) & (at < cos.shape[0])
    c, s = (torch.where(there[..., None], t[torch.where(there, at, 0)], float("nan"))
            .to(wide)[:, :, None] for t in (cos, sin))
    xf = x.to(wide)
    y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * \
        (weight.to(wide) + (1.0 if one_plus else 0.0))
    # a row without a position is none: also where nothing turns
    y = y * torch.where(there, 1.0, float("nan")).to(wide)[..., None, None]
    if layout == "half":
        a, b = y[..., :n // 2], y[..., n // 2:n]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = y[..., 0:n:2], y[..., 1:n:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([turned, y[..., n:]], -1).to(x.dtype)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor,
                 k_weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                 positions: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 layout: str = "half", one_plus: bool = False
                 ) -> Tuple[torch.Tensor, torch.Tensor]:
    """q [B, S, H, D] and k [B, S, Hk, D] (slices of a joint projection as they are) ->
    new tensors: each head divided by its root mean square, times ``q_weight`` or
    ``k_weight`` [D] (``one_plus``: 1 + weight), then turned by its token's angles.
    cos, sin: fp32 [positions, n] (``rope_tables(2 n, ..)``), which turn the first 2 n
    coordinates, i with i + n (layout "half") or neighbours ("interleaved").
    ``positions`` int32 [B, S], by default a token's place in its row; tokens whose
    position is not in the tables become NaN. Differentiable (once) in q, k and the
    weights. bf16, fp16 or fp32, even D up to 512, all in fp32 and rounded once."""
    if layout not in LAYOUTS:
        raise ValueError(f"qk_norm_rope: layout is one of {LAYOUTS}, got {layout!r}")
    ext = get_ext()
    if q.is_cuda and ext is not None and untransformed():
        return ext.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps,
                                layout == "half", one_plus)
    D = q.shape[-1] if q.dim() else 0
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or \
            k.shape[3] != D or D % 2 or not 2 <= D <= 512 or \
            0 in (q.shape[2], k.shape[2]):
        raise ValueError("qk_norm_rope: q is [B, S, H, D], k [B, S, Hk, D], D even and "
                         f"up to 512, got {tuple(q.shape)} and {tuple(k.shape)}")
    if q_weight.shape != (D,) or k_weight.shape != (D,):
        raise ValueError("qk_norm_rope: weights are [D]")
    if not q.dtype == k.dtype == q_weight.dtype == k_weight.dtype or q.dtype not in (
            torch.bfloat16, torch.float16, torch.float32, torch.float64):
        raise ValueError("qk_norm_rope: heads and weights of one type, got "
                         f"{q.dtype}, {k.dtype}, {q_weight.dtype}, {k_weight.dtype}")
    if cos.shape != sin.shape or cos.dim() != 2 or not 2 <= 2 * cos.shape[1] <= D or \
            cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
        raise ValueError("qk_norm_rope: cos and sin are fp32 [positions, rotated / 2]")
    if positions is None:
        if q.shape[1] > cos.shape[0]:
            raise ValueError("qk_norm_rope: rows longer than the tables")
    elif positions.dtype is not torch.int32 or \
            positions.numel() != q.shape[0] * q.shape[1]:
        raise ValueError("qk_norm_rope: positions are int32, one a token")
    if any(t is not None and t.device != q.device
           for t in (k, q_weight, k_weight, cos, sin, positions)):
        raise ValueError("qk_norm_rope: tensors on different devices")
    if cos.requires_grad or sin.requires_grad:
        raise ValueError("qk_norm_rope: cos and sin have no gradient")
    how = cos, sin, positions, eps, layout, one_plus
    return _torch_heads(q, q_weight, *how), _torch_heads(k, k_weight, *how)
