"""Log probabilities of given classes, entropy and alternatives, with
gradients: what training by rewards, on pseudo labels or towards sure answers
takes of a classifier, and what scoring with one reports.

``log_probs`` reads logits in memory (csrc/logp.hip).  ``linear_log_probs``
makes those of a classifier, log_probs(F.linear(hidden[rows], weight, bias),
index), without keeping them (csrc/head.hip): its forward reduces them in the
product's epilogue, its backward makes them again piece by piece of the
classes.  Under autocast hidden, weight and bias are taken in the autocast
dtype, as ``F.linear`` takes them.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd import Function

from ..core import ops as _ops


class LogProbs(NamedTuple):
    """logp f32, shaped as the given classes; entropy f32 [n] (natural
    logarithms); with top > 0 the largest logits' log probabilities f32 and
    classes int32 [n, top], largest first (None without).  logp and entropy
    carry gradients."""
    logp: torch.Tensor
    entropy: torch.Tensor
    top_logp: Optional[torch.Tensor] = None
    top_index: Optional[torch.Tensor] = None


class _Once(Function):
    """Gradients tied to the tensors they belong to (the first `owners`):
    differentiating them again is an error and not a zero."""

    @staticmethod
    def forward(ctx, owners, *tensors):
        ctx.set_materialize_grads(False)
        return tuple(g.view_as(g) if g is not None else None for g in tensors[owners:])

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("log_probs / linear_log_probs have no second derivative")


class _LogProbs(Function):
    @staticmethod
    def forward(ctx, logits, index, temperature, top):
        ctx.set_materialize_grads(False)
        x, index = _ops._unit_columns(logits), index.contiguous()
        need = ctx.needs_input_grad[0]
        logp, entropy, saved, top_logp, top_index = _ops.log_probs_fwd(x, index, temperature, top, need)
        if need:
            # the argument and not a copy of it, which has no history of its own
            ctx.save_for_backward(logits, index, saved, entropy)
            ctx.temperature = temperature
        if top:
            ctx.mark_non_differentiable(top_logp, top_index)
        return logp, entropy, top_logp, top_index

    @staticmethod
    def backward(ctx, dlogp, dentropy, _dtop, _dindex):
        if dlogp is None and dentropy is None:
            return None, None, None, None
        logits, index, saved, entropy = ctx.saved_tensors
        grad = _ops.log_probs_bwd(_ops._unit_columns(logits.detach()), index, ctx.temperature, saved, entropy, dlogp,
                                  dentropy)
        if torch.is_grad_enabled():  # create_graph=True
            owners = [logits] + [d for d in (dlogp, dentropy) if d is not None]
            grad, = _Once.apply(len(owners), *owners, grad)
        return grad, None, None, None


def log_probs(logits: torch.Tensor, index: torch.Tensor, temperature: float = 1.0, top: int = 0) -> LogProbs:
    """LogProbs of softmax(logits / temperature), logits [n, classes].

    index int32 or int64 [n] or [n, k] (k <= 1024): the classes whose log
    probabilities are returned, in its shape; a negative one asks for nothing
    (log probability 0, no gradient), one past the last class is an error
    (NaN, no gradient).  A class of logit -inf, or further below the row's
    largest one than float32 holds, has log probability -inf and adds nothing
    to the entropy; a row of nothing but -inf is NaN, its gradient zeros; a
    row with NaN or +inf is NaN, and so is its gradient.  top <= min(classes,
    1024).  No host sync; no second derivative."""
    _ops.check_log_probs(logits, index, temperature, top)
    return LogProbs(*_LogProbs.apply(logits, index, float(temperature), int(top)))


class _LinearLogProbs(Function):
    @staticmethod
    def forward(ctx, hidden, weight, bias, rows, index, temperature, top):
        ctx.set_materialize_grads(False)
        call = _ops.given_call(hidden, weight, index, bias, rows, temperature)
        logp, entropy, saved, top_logp, top_index = _ops.head_log_probs_fwd(call, index.shape, top)
        if any(ctx.needs_input_grad[:3]):
            ctx.save_for_backward(hidden, weight, bias, rows, index, logp, entropy, saved)
            ctx.temperature = temperature
        if top:
            ctx.mark_non_differentiable(top_logp, top_index)
        return logp, entropy, top_logp, top_index

    @staticmethod
    def backward(ctx, dlogp, dentropy, _dtop, _dindex):
        if dlogp is None and dentropy is None:
            return (None,) * 7
        hidden, weight, bias, rows, index, logp, entropy, saved = ctx.saved_tensors
        call = _ops.given_call(hidden, weight, index, bias, rows, ctx.temperature)
        grads = _ops.head_log_probs_bwd(call, saved, logp, entropy, dlogp, dentropy, ctx.needs_input_grad[:3])
        if torch.is_grad_enabled():  # create_graph=True
            owners = [t for t in (hidden, weight, bias, dlogp, dentropy) if t is not None]
            grads = _Once.apply(len(owners), *owners, *grads)
        return (*grads, None, None, None, None)


def linear_log_probs(hidden: torch.Tensor, weight: torch.Tensor, index: torch.Tensor,
                     bias: Optional[torch.Tensor] = None, rows: Optional[torch.Tensor] = None,
                     temperature: float = 1.0, top: int = 0) -> LogProbs:
    """LogProbs of softmax((hidden[rows] @ weight.T + bias) / temperature).

    hidden [N, D], weight [V, D], bias [V] (one dtype of f32, f16, bf16), rows
    int64 [n] (None = the first n rows; distinct ones where hidden needs a
    gradient, which is NaN at a row listed twice: gather such rows first).
    index int32 or int64 [n] or [n, k] (k <= 1024), the given classes, and
    what is not a number as in log_probs; a row id out of range is an error
    (NaN in its row, no gradient).  top > 0 (for scoring) keeps the logits of
    up to 1 GiB, or 256 rows, at a time.  No host sync; no second derivative."""
    if hidden.is_cuda and torch.is_autocast_enabled("cuda"):
        dt = torch.get_autocast_dtype("cuda")
        hidden, weight = hidden.to(dt), weight.to(dt)
        bias = bias.to(dt) if bias is not None else None
    _ops.check_linear_log_probs(hidden, weight, index, bias, rows, temperature, top)
    return LogProbs(*_LinearLogProbs.apply(hidden, weight, bias, rows, index, float(temperature), int(top)))
