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
The host path -- checks, outputs, autograd nodes -- is C++ (csrc/torch_ops.cpp): in a step of the tracker's sizes it is what these calls cost.
The gradients of the two normalisations are not differentiable themselves (refused); dropout's are.  ``torch.func`` transforms (``vmap``, ``grad``),
batched gradients and sparse tensors are refused; ``torch.compile`` runs the operators as they are, outside of its graphs.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import hip

Seed = Union[int, torch.Tensor]


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension, in x's type; statistics in fp32.

    x (..., D): rows of the last dimension at one stride are read where they lie (a slice of a merged projection), any other
    layout is copied first.  weight / bias (D,): x's type or float32, both the same; either may be None.  The result is dense.
    A row whose sum or sum of squared deviations is beyond fp32's range (3.4e38) gives NaN."""
    return hip.ops().norm(x, None, weight, bias, eps, 0.0, 0, None, 0)


def dropout(x: torch.Tensor, p: float, seed: Seed, offset: int = 0) -> torch.Tensor:
    """``x / (1 - p)`` where the mask of (seed, offset) keeps an element, 0 elsewhere -- whatever the dropped value was, NaN included.

    p is taken to the nearest multiple of 2^-32 (0: a plain copy; 1: all zeros).  The result is dense, in x's type; an x that is not dense
    (a slice's rows included) is copied first."""
    return hip.ops().dropout(x, *hip._drop_args(p, seed, offset))


def dropout_add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                           p: float = 0.0, seed: Seed = 0, offset: int = 0, eps: float = 1e-5) -> torch.Tensor:
    """``layer_norm(residual + dropout(x, p, seed, offset), weight, bias, eps)`` with the sum kept in fp32, in the residual's type.

    x and residual have the same shape (..., D); the residual has x's type or float32 (half-precision products beside an fp32
    residual stream).  Nothing is stored for the backward pass but the inputs and two fp32 numbers a row."""
    return hip.ops().norm(x, residual, weight, bias, eps, *hip._drop_args(p, seed, offset))
