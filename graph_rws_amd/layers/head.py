"""Classifier over many classes fused with its loss (csrc/head.hip).

``linear_cross_entropy`` is ``F.cross_entropy(F.linear(hidden[rows], weight,
bias), labels)`` and ``linear_distill`` the divergence of the same logits
from a teacher's top logits (``core.top_logits`` makes the lists).  The
logits [n, classes] are never kept: the forward reduces them in the
product's epilogue, the backward makes them again piece by piece of the
classes.

``LinearHead`` holds a classifier's weight and bias and makes these calls;
``helper.train_epoch_head`` trains one on top of a graph model.

Under autocast hidden, weight and bias are taken in the autocast dtype, as
``F.linear`` takes them.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import Function

from ..core import ops as _ops

_REDUCTIONS = ("mean", "none")


class _FirstOnly(Function):
    """The gradients, tied to the parameters they belong to (the first of the
    arguments): differentiating them again is an error and not a zero."""

    @staticmethod
    def forward(ctx, params, *grads):
        ctx.set_materialize_grads(False)
        return tuple(g.view_as(g) if g is not None else None for g in grads[params:])

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("linear_cross_entropy / linear_distill have no second derivative")


class _Head(Function):
    @staticmethod
    def forward(ctx, hidden, weight, bias, rows, labels, teacher_index, teacher_logits, temperature, per_row):
        call = _ops.HeadCall(hidden, weight, bias, rows, labels, teacher_index, teacher_logits, temperature)
        loss, counts, saved = _ops.head_fwd(call, per_row)
        if any(ctx.needs_input_grad[:3]):
            ctx.save_for_backward(hidden, weight, bias, rows, labels, teacher_index, teacher_logits, counts, saved)
            ctx.temperature = temperature
        ctx.mark_non_differentiable(counts)
        return loss, counts

    @staticmethod
    def backward(ctx, dloss, _dcounts):
        hidden, weight, bias, rows, labels, index, logits, counts, saved = ctx.saved_tensors
        call = _ops.HeadCall(hidden, weight, bias, rows, labels, index, logits, ctx.temperature)
        grads = _ops.head_bwd(call, saved, counts, dloss, ctx.needs_input_grad[:3])
        if torch.is_grad_enabled():  # create_graph=True
            grads = _FirstOnly.apply(4, hidden, weight, bias, dloss, *grads)
        return (*grads, None, None, None, None, None, None)


def _apply(hidden, weight, bias, rows, labels, index, logits, temperature, reduction):
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {_REDUCTIONS} (got {reduction!r})")
    if hidden.is_cuda and torch.is_autocast_enabled("cuda"):
        dt = torch.get_autocast_dtype("cuda")
        hidden, weight = hidden.to(dt), weight.to(dt)
        bias = bias.to(dt) if bias is not None else None
    _ops.check_head(hidden, weight, bias, rows, labels, index, logits, temperature)
    return _Head.apply(hidden, weight, bias, rows, labels, index, logits, float(temperature), reduction == "none")


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
                         bias: Optional[torch.Tensor] = None, rows: Optional[torch.Tensor] = None,
                         reduction: str = "mean"):
    """(loss, counts) of softmax cross entropy of hidden[rows] @ weight.T +
    bias against labels.

    hidden [N, D], weight [V, D], bias [V] (one dtype of f32, f16, bf16),
    labels int64 [n] (-100: the row does not count), rows int64 [n] (None =
    the first n rows; distinct ones where hidden needs a gradient, which is
    NaN at a row listed twice: gather such rows first).  reduction "mean": the f32 mean over counted
    rows, NaN when none counts or a label or row id is out of range; "none":
    f32 [n], 0 for rows that do not count.  counts: int64 [3] on the device,
    {rows whose label is the first largest logit, counted rows, bad input}.
    """
    return _apply(hidden, weight, bias, rows, labels, None, None, 1.0, reduction)


def linear_distill(hidden: torch.Tensor, weight: torch.Tensor, teacher_index: torch.Tensor,
                   teacher_logits: torch.Tensor, bias: Optional[torch.Tensor] = None,
                   rows: Optional[torch.Tensor] = None, temperature: float = 1.0, reduction: str = "mean"):
    """(loss, counts) of T^2 KL(softmax(teacher / T) || softmax(z / T)) with
    z = hidden[rows] @ weight.T + bias and the teacher's softmax over its
    listed classes.

    teacher_index int32 or int64 [n, k] (-1: no entry), teacher_logits
    [n, k] (-inf: no entry); a row without entries does not count.  The other
    arguments and reduction as in linear_cross_entropy.  counts: int64 [2] on
    the device, {counted rows, bad input}.  No gradient reaches the teacher.
    """
    if teacher_index is None or teacher_logits is None:
        raise ValueError("linear_distill: teacher_index and teacher_logits are required")
    loss, counts = _apply(hidden, weight, bias, rows, None, teacher_index, teacher_logits, temperature, reduction)
    return loss, counts[1:]


class LinearHead(torch.nn.Module):
    """Classifier over many classes on top of a model's hidden rows: weight
    [classes, width] and bias, as torch.nn.Linear has them."""

    def __init__(self, width: int, classes: int, bias: bool = True):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.empty(classes, width))
        self.bias = torch.nn.Parameter(torch.empty(classes)) if bias else None
        self.reset_parameters()

    def reset_parameters(self):
        torch.nn.init.normal_(self.weight, std=self.weight.shape[1] ** -0.5)
        if self.bias is not None:
            torch.nn.init.zeros_(self.bias)

    def forward(self, hidden: torch.Tensor) -> torch.Tensor:
        """The logits themselves, [rows, classes]."""
        return torch.nn.functional.linear(hidden, self.weight, self.bias)

    def loss(self, hidden, labels, rows=None, reduction: str = "mean"):
        """linear_cross_entropy of this classifier."""
        return linear_cross_entropy(hidden, self.weight, labels, self.bias, rows, reduction)

    def distill(self, hidden, teacher_index, teacher_logits, rows=None, temperature: float = 1.0,
                reduction: str = "mean"):
        """linear_distill of this classifier (the student)."""
        return linear_distill(hidden, self.weight, teacher_index, teacher_logits, self.bias, rows, temperature,
                              reduction)

    @torch.no_grad()
    def top(self, hidden, k: int, rows_at_once: int = 8192):
        """(values, classes int32) [rows, k]: this classifier's top logits (the
        teacher's lists), `rows_at_once` rows of logits in memory at a time."""
        parts = [_ops.top_logits(self(hidden[i:i + rows_at_once]), k)
                 for i in range(0, max(1, hidden.shape[0]), rows_at_once)]
        return torch.cat([v for v, _ in parts]), torch.cat([c for _, c in parts])
