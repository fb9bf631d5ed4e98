"""Log probabilities of given tokens under rows of logits, with entropy and top alternatives, and
their gradient: what a decoder answers with, and what a cross-entropy or policy-gradient loss
trains on (the reference's loss is torch's cross entropy, chat/nanochat/gpt.py:167-170).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import ops


class TokenLogprobs(NamedTuple):
    logp: torch.Tensor      # [...] float32: log p(token)
    entropy: torch.Tensor   # [...] float32: -sum p log p, in nats
    top_ids: torch.Tensor   # [..., n_top] int64: most probable entries, ties to the lower index
    top_logp: torch.Tensor  # [..., n_top] float32


class TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature, n_top, ignore_index):
        logp, entropy, lse, top_ids, top_logp = ops.token_logprobs_fwd(logits, tokens, temperature, n_top, ignore_index)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, tokens.contiguous(), lse, entropy)
        ctx.temperature, ctx.ignore_index = temperature, ignore_index
        ctx.mark_non_differentiable(top_ids, top_logp)
        return logp, entropy, top_ids, top_logp

    @staticmethod
    def backward(ctx, g_logp, g_entropy, _ids, _top):
        # (the guard against a second differentiation only where a graph of this one is made)
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, g_logp, g_entropy)


def _backward(ctx, g_logp, g_entropy):
    logits, tokens, lse, entropy = ctx.saved_tensors
    if g_logp is None and g_entropy is None:
        return None, None, None, None, None
    return ops.token_logprobs_bwd_unchecked(logits, tokens, lse, entropy, g_logp, g_entropy, ctx.temperature,
                                            ctx.ignore_index), None, None, None, None


_backward_once = torch.autograd.function.once_differentiable(_backward)


def token_logprobs(logits, tokens, temperature=1.0, n_top=0, ignore_index=-100) -> TokenLogprobs:
    """logits [..., V] (fp32 or bf16), tokens int64 [...] -> TokenLogprobs of softmax(logits / temperature).

    n_top <= min(32, V) alternatives per row in the order (logit descending, index ascending).
    logp and entropy are differentiable in logits; the alternatives are not.  Entries of
    -infinity (a mask) have probability 0; a row whose token is ignore_index gives 0, ids of -1
    and no gradient; the mean of -logp over the other rows is the cross entropy.  Another token
    outside the vocabulary makes its row's logp NaN, and the gradient too where that logp is used."""
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*TokenLogprobsFn.apply(logits, tokens, temperature, n_top, ignore_index))
    logp, entropy, _, top_ids, top_logp = ops.token_logprobs_fwd(logits, tokens, temperature, n_top, ignore_index,
                                                                 keep_lse=False)
    return TokenLogprobs(logp, entropy, top_ids, top_logp)
