"""Residual RMS norm with its gradient (the norm in front of every attention and MLP block;
the reference takes it from torch, chat/nanochat/gpt.py:62-64).

    h = x + residual,   y = h * rsqrt(mean(h^2) + eps) * weight

h is held in x's dtype (the residual stream), everything else in fp32 up to y's one rounding.
"""
from __future__ import annotations

import torch

from . import ops


class AddRMSNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, h, rstd = ops.rms_norm_fwd(x, residual, weight, eps, return_rstd=True)
        ctx.set_materialize_grads(False)
        ctx.has_residual = residual is not None
        ctx.save_for_backward(h, rstd, weight)
        return (y, h) if ctx.has_residual else y

    @staticmethod
    def backward(ctx, dy, dh=None):
        # (the guard against a second differentiation only where a graph of this one is made)
        return _backward_once(ctx, dy, dh) if torch.is_grad_enabled() else _backward(ctx, dy, dh)


def _backward(ctx, dy, dh):
    h, rstd, weight = ctx.saved_tensors
    dw = None
    if dy is None:  # only h was used
        dx = dh
    else:
        dx, dw = ops.rms_norm_bwd_unchecked(dy, dh, h.contiguous(), rstd, weight, ctx.needs_input_grad[2])
    return dx, dx if ctx.has_residual else None, dw, None


_backward_once = torch.autograd.function.once_differentiable(_backward)


def add_rms_norm(x, residual=None, weight=None, eps=1e-5):
    """(y, h) for x, residual [..., K] (fp32 or bf16) and weight [K] (fp32, bf16 or None: ones).

    Without a residual h is x.  Differentiable in x, residual and weight."""
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)
                                    or (weight is not None and weight.requires_grad)):
        if residual is None:
            return AddRMSNormFn.apply(x, None, weight, eps), x
        return AddRMSNormFn.apply(x, residual, weight, eps)
    return ops.rms_norm_fwd(x, residual, weight, eps)
