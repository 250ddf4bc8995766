"""Gradients of the feature operators that have one: ``torch.autograd`` nodes over the forward
and backward entry points. They are used only where an input asks for a gradient."""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from mlx_lattice_b200 import _ext


def wanted(*tensors) -> bool:
    """Whether a call on these (optional) tensors has to record a gradient."""
    return torch.is_grad_enabled() and any(
        isinstance(t, torch.Tensor) and t.requires_grad for t in tensors)


class RowNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, feats, weight, bias, eps, rms):
        out, mean, rstd = _ext.row_norm_forward(feats, weight, bias, eps, rms)
        ctx.rms = rms
        ctx.save_for_backward(feats, weight, mean, rstd)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        feats, weight, mean, rstd = ctx.saved_tensors
        grads = _ext.row_norm_backward(
            grad, feats, weight, mean, rstd, ctx.rms, ctx.needs_input_grad[1], ctx.needs_input_grad[2])
        return (*grads, None, None)


class Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, feats, residual, p, seed, offset):
        ctx.p, ctx.offset = p, offset
        # a device seed is saved as a tensor, so that changing it before the backward pass,
        # which draws the mask again, is noticed
        ctx.seed = None if isinstance(seed, torch.Tensor) else seed
        ctx.save_for_backward(seed if ctx.seed is None else None)
        return _ext.dropout(feats, p, seed, offset, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        seed = ctx.saved_tensors[0] if ctx.seed is None else ctx.seed
        grad_feats = _ext.dropout(grad, ctx.p, seed, ctx.offset) if ctx.needs_input_grad[0] else None
        return grad_feats, grad if ctx.needs_input_grad[1] else None, None, None, None


class GatedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, feats, gate, initial_state, offsets, reverse, want_state):
        out, final, carries = _ext.recurrence_forward(
            feats, gate, offsets, initial_state, reverse, want_state=want_state, want_carries=True)
        ctx.reverse = reverse
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(feats, gate, initial_state, offsets, carries)
        return out, final

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, grad_final):
        feats, gate, initial_state, offsets, carries = ctx.saved_tensors
        if grad is None:
            grad = torch.zeros_like(feats)
        grads = _ext.recurrence_backward(
            grad, grad_final, feats, gate, offsets, initial_state, ctx.reverse, carries,
            want_initial=ctx.needs_input_grad[2])
        return (*grads, None, None, None)
