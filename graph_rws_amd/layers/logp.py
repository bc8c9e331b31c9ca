"""Log probabilities of given classes, entropy and alternatives, with
gradients: what training by rewards, on pseudo labels or towards sure answers
takes of a classifier, and what scoring with one reports.

``log_probs`` reads logits in memory (csrc/logp.hip).
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
            ctx.save_for_backward(x, index, saved, entropy)
            ctx.temperature = temperature
        if top:
            ctx.mark_non_differentiable(top_logp, top_index)
        return logp, entropy, top_logp, top_index

    @staticmethod
    def backward(ctx, dlogp, dentropy, _dtop, _dindex):
        if dlogp is None and dentropy is None:
            return None, None, None, None
        x, index, saved, entropy = ctx.saved_tensors
        grad = _ops.log_probs_bwd(x, index, ctx.temperature, saved, entropy, dlogp, dentropy)
        if torch.is_grad_enabled():  # create_graph=True
            owners = [x] + [d for d in (dlogp, dentropy) if d is not None]
            grad, = _Once.apply(len(owners), *owners, grad)
        return grad, None, None, None


def log_probs(logits: torch.Tensor, index: torch.Tensor, temperature: float = 1.0, top: int = 0) -> LogProbs:
    """LogProbs of softmax(logits / temperature), logits [n, classes].

    index int32 or int64 [n] or [n, k] (k <= 1024): the classes whose log
    probabilities are returned, in its shape; a negative one asks for nothing
    (log probability 0, no gradient), one past the last class is an error
    (NaN, no gradient).  A class of logit -inf has log probability -inf and
    adds nothing to the entropy; a row of nothing but -inf is NaN, its
    gradient zeros.  top <= min(classes, 1024).  No host sync; no second
    derivative."""
    _ops.check_log_probs(logits, index, temperature, top)
    return LogProbs(*_LogProbs.apply(logits, index, float(temperature), int(top)))
