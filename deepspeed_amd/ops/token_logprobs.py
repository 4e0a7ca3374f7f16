"""Log probabilities of given tokens, with the entropy of their distribution and its
best tokens (csrc/token_logprobs.hip): what a policy's loss is made of, and what a
server answers beside its tokens. The logits are read once and nothing of their size is
written but, backward, their gradient."""

from typing import NamedTuple

import torch

from ._loader import get_ext
from .linear import untransformed

# Best tokens that a call may ask for, and the vocabulary it may ask them of.
MOST, WIDEST = 32, 500_000


class TokenLogprobs(NamedTuple):
    """``logprobs`` and ``entropy`` fp32, one a token; ``top_logprobs`` fp32 and
    ``top_ids`` int64 [.., top], best first, of equal logits the lower id first."""

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor
    top_ids: torch.Tensor


def _torch_logprobs(logits, tokens, top, ignore_index):
    """The formulas in fp32 (fp64 for fp64)."""
    x = logits if logits.dtype is torch.float64 else logits.float()
    V = x.shape[-1]
    live = tokens != ignore_index
    known = (tokens >= 0) & (tokens < V)
    x = x.masked_fill(~live[..., None], 0.0)
    lp = torch.log_softmax(x, -1)
    # a logit of no share adds nothing, though its logarithm be past all numbers
    none = lp.exp() == 0
    some = lp.masked_fill(none, 0.0)
    share = torch.where(none, 0.0, some.exp() * some)
    entropy = torch.where(live, -share.sum(-1), 0.0)
    got = lp.gather(-1, torch.where(known, tokens, 0)[..., None])[..., 0]
    got = got * torch.where(known | ~live, 1.0, float("nan")).to(got.dtype)
    got = torch.where(live, got, 0.0)
    order = tokens.new_empty(*tokens.shape, 0)
    if top:
        # NaN above all, infinity among it, as numbers that are equal in order of their
        # ids: by values, then by which are none
        nan = x.detach() != x.detach()
        order = torch.sort(x.detach().masked_fill(nan, 0.0), dim=-1, descending=True,
                           stable=True).indices
        first = torch.sort(nan.gather(-1, order).to(torch.int8), dim=-1,
                           descending=True, stable=True).indices
        order = order.gather(-1, first)[..., :top]
    best = lp.detach().gather(-1, order)
    return TokenLogprobs(got, entropy,
                         torch.where(live[..., None], best, float("-inf")),
                         torch.where(live[..., None], order, -1))


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """``logits`` [.., V] bf16, fp16 or fp32 and ``tokens`` [..] (integers) -> the log
    probability of each token under the softmax of its logits, the entropy of that
    softmax in nats, and its ``top`` (up to 32) best tokens with theirs. Differentiable
    (once) in the logits through ``logprobs`` and ``entropy``. Tokens of
    ``ignore_index`` give 0 and 0, no gradient, and ids of -1; a token that is not in
    the vocabulary gives NaN, and a NaN logit counts above all others."""
    ext = get_ext()
    if logits.is_cuda and ext is not None and untransformed():
        return TokenLogprobs(*ext.token_logprobs(logits, tokens, top, ignore_index))
    if logits.dim() < 1 or logits.shape[:-1] != tokens.shape or logits.shape[-1] < 1:
        raise ValueError("token_logprobs: logits [.., V] and tokens [..], got "
                         f"{tuple(logits.shape)} and {tuple(tokens.shape)}")
    if tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"token_logprobs: integer tokens, got {tokens.dtype}")
    if logits.dtype not in (torch.bfloat16, torch.float16, torch.float32,
                            torch.float64):
        raise ValueError(f"token_logprobs: floating logits, got {logits.dtype}")
    V = logits.shape[-1]
    if not 0 <= top <= min(MOST, V) or (top and V > WIDEST):
        raise ValueError(f"token_logprobs: up to {MOST} best of {WIDEST} tokens at "
                         f"most, got {top} of {V}")
    if logits.device != tokens.device:
        raise ValueError("token_logprobs: tensors on different devices")
    return _torch_logprobs(logits, tokens.long(), top, ignore_index)
