"""The head and its loss in one: softmax cross entropy of a linear projection onto a vocabulary, without
the logits in memory, with its gradients.

The reference ends its model with an `nn.Linear` and trains it with `nn.CrossEntropyLoss`
(models/vit.py:62, main_train_tinyvit_mnist.py:62-76); with a vocabulary instead of ten classes the
[tokens, vocab] logits, their softmax and its gradient are the largest tensors of a step.  Here the
forward pass keeps one fp32 number per token, and the backward pass computes the logits again, a piece of the
vocabulary at a time.

Operands are bf16 (accumulation, softmax and losses fp32).  Under bf16 autocast fp32 tensors are taken too and
rounded to bf16, as F.linear does there; their gradients come back in fp32, straight from the fp32
accumulators."""
from __future__ import annotations

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from backend import ops as _ops


def _operand(t, name):
    if t.dtype == torch.bfloat16:
        return t
    if t.dtype == torch.float32 and torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") == torch.bfloat16:
        return t.to(torch.bfloat16)
    raise ValueError(f"linear_cross_entropy: {name} is {t.dtype}; it takes bfloat16 (float32 too under bfloat16 autocast)")


def _forward(hidden, weight, bias, target, ignore_index, reduction):
    h, w, t = _operand(hidden, "hidden"), _operand(weight, "weight"), target
    if hidden.ndim != 2:
        h, t = h.reshape(-1, hidden.shape[-1]), target.reshape(-1)
    loss, lse, _ = _ops.linear_cross_entropy_forward(h, w, bias, t, ignore_index, reduction)
    return h, w, t, loss.view(target.shape) if reduction == "none" else loss, lse


class _LinearCrossEntropyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, bias, target, ignore_index, reduction):
        ctx.dtypes = hidden.dtype, weight.dtype, None if bias is None else bias.dtype
        ctx.shape, ctx.args = hidden.shape, (ignore_index, reduction)
        h, w, t, loss, lse = _forward(hidden, weight, bias, target, ignore_index, reduction)
        ctx.save_for_backward(h, w, bias, t, lse)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        h, w, bias, t, lse = ctx.saved_tensors
        want = [dt if need else None for dt, need in zip(ctx.dtypes, ctx.needs_input_grad)]
        dh, dw, db = _ops.linear_cross_entropy_backward(grad.reshape(-1), h, w, bias, t, lse, *ctx.args, *want)
        return None if dh is None else dh.view(ctx.shape), dw, db, None, None, None     # (a head frozen in training: only dh)


def linear_cross_entropy(hidden, weight, target, bias=None, ignore_index=-100, reduction="mean"):
    """F.cross_entropy(F.linear(hidden, weight, bias), target) in fp32, without the logits.

    hidden [..., D], weight [V, D] (D a multiple of 8), bias [V] (float32 or bfloat16), target [...] int64.
    reduction "mean" (over the tokens whose target is not ignore_index), "sum" or "none"; the result is fp32.
    A target outside the vocabulary makes its loss NaN and is reported by backend.ops.check_status()."""
    if hidden.ndim < 1 or weight.ndim != 2 or target.shape != hidden.shape[:-1]:
        raise ValueError("linear_cross_entropy takes hidden [..., D], weight [V, D] and target [...], got "
                         f"{tuple(hidden.shape)}, {tuple(weight.shape)} and {tuple(target.shape)}")
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        return _LinearCrossEntropyFn.apply(hidden, weight, bias, target, int(ignore_index), reduction)
    return _forward(hidden, weight, bias, target, int(ignore_index), reduction)[3]


class LinearCrossEntropy(nn.Module):
    """`nn.CrossEntropyLoss` that takes the head's input and weights in place of its logits:
    loss(hidden, head.weight, target, head.bias)."""

    def __init__(self, ignore_index=-100, reduction="mean"):
        super().__init__()
        if reduction not in ("mean", "sum", "none"):
            raise ValueError(f"unknown reduction {reduction!r}")
        self.ignore_index, self.reduction = ignore_index, reduction

    def forward(self, hidden, weight, target, bias=None):
        return linear_cross_entropy(hidden, weight, target, bias, self.ignore_index, self.reduction)

    def extra_repr(self):
        return f"ignore_index={self.ignore_index}, reduction={self.reduction!r}"
