"""Differentiable operators of a training step, on hand-written kernels of ``liblbm_hip.so``.

Every block of the tracker joins its residual as ``norm(x + dropout(f(x)))`` (reference: lbm/models/lbm/transformer.py:272-338,
msdeformattn.py:185) with p = 0.1 in training.  These are that join, and its two parts, with their gradients, for rows of any
length in float32, float16 or bfloat16:

    layer_norm(x, weight, bias)                                    the last dimension normalised
    dropout(x, p, seed, offset)                                    x / (1 - p) where kept, else 0
    dropout_add_layer_norm(x, residual, weight, bias, p, seed, offset)   layer_norm(residual + dropout(x)), one pass each way

Random numbers are arguments, not state: the mask is a function of ``(seed, offset, element)`` alone (Philox4x32-10; the formula is
in include/lbm_hip.h), is never stored, and is the same for every type, shape of the same elements and run.  Give each call of
a step its own ``offset`` and each step its own ``seed``.  ``seed`` may be an int64 GPU tensor of one element: a captured graph reads it
when it is replayed, so advancing it in place draws new masks; between a forward pass and its backward pass it must not change
(outside of a graph autograd checks that).

There is no CPU path, and no automatic type conversion under ``torch.autocast``: x and residual are taken in the types they have.
The gradients of the two normalisations are not differentiable themselves (refused); dropout's are.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import hip

Seed = Union[int, torch.Tensor]


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, p, seed, offset):
        y, mean, rstd = hip.norm_forward(x, weight, bias, eps, residual, p, seed, offset, want_stats=True)
        on_device = isinstance(seed, torch.Tensor)
        ctx.save_for_backward(x, residual, weight, bias, mean, rstd, seed if on_device else None)
        ctx.eps, ctx.p, ctx.seed, ctx.offset = eps, p, None if on_device else seed, offset
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():      # create_graph: a result without a graph would drop the second derivatives in silence
            raise hip.HipError("the gradients of layer_norm and dropout_add_layer_norm are not differentiable (create_graph=True)")
        x, residual, weight, bias, mean, rstd, seed = ctx.saved_tensors
        dx, dres, dw, db = hip.norm_backward(dy, x, mean, rstd, weight, bias, ctx.eps, residual, ctx.p, ctx.seed if seed is None else seed,
                                             ctx.offset, want=ctx.needs_input_grad[:4])
        return dx, dres, dw, db, None, None, None, None


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, offset):
        on_device = isinstance(seed, torch.Tensor)
        ctx.save_for_backward(seed if on_device else None)
        ctx.p, ctx.seed, ctx.offset = p, None if on_device else seed, offset
        return hip.dropout(x, p, seed, offset)

    @staticmethod
    def backward(ctx, dy):
        seed, = ctx.saved_tensors
        return dropout(dy, ctx.p, ctx.seed if seed is None else seed, ctx.offset), None, None, None


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension, in x's type; statistics in fp32.

    x (..., D): rows of the last dimension at one stride are read where they lie (a slice of a merged projection), any other
    layout is copied first.  weight / bias (D,): x's type or float32, both the same; either may be None.  The result is dense.
    Squared deviations beyond fp32's range (3.4e38) are outside the domain."""
    if _wants_grad(x, weight, bias):
        return _Norm.apply(x, None, weight, bias, eps, 0.0, 0, 0)
    return hip.norm_forward(x, weight, bias, eps)


def dropout(x: torch.Tensor, p: float, seed: Seed, offset: int = 0) -> torch.Tensor:
    """``x / (1 - p)`` where the mask of (seed, offset) keeps an element, 0 elsewhere -- whatever the dropped value was, NaN included.

    p is taken to the nearest multiple of 2^-32 (0: a plain copy; 1: all zeros).  The result is dense, in x's type."""
    if _wants_grad(x):
        return _Dropout.apply(x, p, seed, offset)
    return hip.dropout(x, p, seed, offset)


def dropout_add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                           p: float = 0.0, seed: Seed = 0, offset: int = 0, eps: float = 1e-5) -> torch.Tensor:
    """``layer_norm(residual + dropout(x, p, seed, offset), weight, bias, eps)`` with the sum kept in fp32, in the residual's type.

    x and residual have the same shape (..., D); the residual has x's type or float32 (half-precision products beside an fp32
    residual stream).  Nothing is stored for the backward pass but the inputs and two fp32 numbers a row."""
    if _wants_grad(x, residual, weight, bias):
        return _Norm.apply(x, residual, weight, bias, eps, p, seed, offset)
    return hip.norm_forward(x, weight, bias, eps, residual, p, seed, offset)
