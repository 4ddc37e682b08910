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

from torch import nn

from backend import ops as _ops
from backend._ext import ext as _ext


def linear_cross_entropy(hidden, weight, target, bias=None, ignore_index=-100, reduction="mean"):
    """F.cross_entropy(F.linear(hidden, weight, bias), target) in fp32, without the logits.

    hidden [..., D], weight [V, D] (D a multiple of 8), bias [V] (float32 or bfloat16), target [...] int64.
    reduction "mean" (over the tokens whose target is not ignore_index), "sum" or "none"; the result is fp32.
    A target outside the vocabulary makes its loss NaN and is reported by backend.ops.check_status()."""
    return _ext().xent_call(hidden, weight, bias, target, ignore_index, _ops._reduction(reduction), _ops._status_ptr(hidden))


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
