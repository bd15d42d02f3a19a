"""Log probabilities of given tokens with the entropy and the most likely alternatives, and their gradient: what a server answers beside a token, and what
training on preferences or rewards takes of its logits.  One pass over the logits forward, one backward, nothing of their size in between."""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib as L

TOP_MAX = 32


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor      # float32 [...]
    entropy: torch.Tensor      # float32 [...], in nats
    top_logprob: torch.Tensor  # float32 [..., top], descending
    top_id: torch.Tensor       # int64 [..., top], -1 where there is none


def _gradient(ctx, g_logprob, g_entropy, g_top, _):
    dx = L.host().token_logprobs_grad(*ctx.saved_tensors, g_logprob, g_entropy, g_top)
    return dx if dx.shape == ctx.shape else dx.view(ctx.shape), None, None


_gradient_once = torch.autograd.function.once_differentiable(_gradient)


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top):
        logprob, entropy, top_logprob, top_id, rows, tokens, stats = L.host().token_logprobs(logits, tokens, top, True)
        ctx.save_for_backward(rows, tokens, stats, entropy, top_id)
        ctx.shape = logits.shape
        ctx.mark_non_differentiable(top_id)
        ctx.set_materialize_grads(False)
        return logprob, entropy, top_logprob, top_id

    @staticmethod
    def backward(ctx, *grads):
        # what marks the gradient as one that has none of its own takes as long as the rest of this call; only a pass that builds a graph needs it
        return (_gradient_once if torch.is_grad_enabled() else _gradient)(ctx, *grads)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """Of logits [..., V] (float32, bf16 or f16) and tokens [...] (int64): the log probability of each token, the entropy of each row's
    distribution in nats, and the `top` (0 to 32) most likely alternatives as log probabilities in descending order with their indices, of equal
    ones the lowest first.  Everything is summed in float32.

    A negative token stands for none: its log probability is 0 and has no gradient (labels of -100); one from V on gives NaN and no gradient.  Logits
    of -inf are masked: they have no probability and are never an alternative (index -1 and -inf where fewer than `top` are left); a row of nothing
    else has a log probability of -inf and an entropy of 0, and no gradient.  A row that holds a NaN or +inf gives NaN; a NaN is never an alternative.

    Differentiable (once, in reverse mode; logits with a tangent are refused) in the logits through the log probabilities, the entropy and the alternatives' log probabilities.  As for any operator, a backward
    pass is captured into a CUDA graph only while no eager autograd graph of the same leaves is alive."""
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobs.apply(logits, tokens, top))
    return TokenLogprobs(*L.host().token_logprobs(logits, tokens, top, False))
