"""The block operators of ``ops`` for programs that train through torch.autograd.

Thin ``torch.autograd.Function``s over the plain functions: the forward keeps what the backward pass needs (for the
recurrence one fp32 state in 32 frames, for dropout nothing but ``rng``), the gradients come from the same kernels as
``ops.*_backward``.  Gradients of gradients are refused.  So is a backward pass under HIP graph capture: gradients that
autograd accumulates into leaves which an eager graph still holds end the process there; capture the plain functions,
whose buffers are the caller's.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops


def _eager():
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("autograd backward under graph capture: capture the ops.*_backward functions instead")


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, groups, eps, act, act_first, lengths):
        y, stats = ops.group_norm_act(x, gamma, beta, groups, eps, act, act_first, lengths)
        ctx.save_for_backward(x, gamma, beta, stats, lengths)
        ctx.how = groups, act, act_first
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _eager()
        x, gamma, beta, stats, lengths = ctx.saved_tensors
        return (*ops.group_norm_act_backward(_dense(dy), x, gamma, beta, stats, *ctx.how, lengths), None, None, None, None, None)


class _GatedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, h0, lengths, reverse, recording):
        h, last, saved = ops.gated_recurrence(x, gate, h0, lengths, reverse, save=recording and any(ctx.needs_input_grad))
        ctx.save_for_backward(x, gate, saved, lengths)
        ctx.reverse = reverse
        return h, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dlast):
        _eager()
        x, gate, saved, lengths = ctx.saved_tensors
        dx, dgate, dh0 = ops.gated_recurrence_backward(_dense(dh), x, gate, saved, dlast.contiguous(), lengths, ctx.reverse)
        return dx, dgate, dh0 if ctx.needs_input_grad[2] else None, None, None, None


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, rng, site, residual):
        ctx.save_for_backward(rng)              # a step that is advanced before the backward pass is noticed there
        ctx.how = p, site, x.dtype
        return ops.dropout(x, p, rng, site, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _eager()
        (rng,), (p, site, dtype) = ctx.saved_tensors, ctx.how
        dx = ops.dropout_backward(_dense(dy), p, rng, site, dtype) if ctx.needs_input_grad[0] else None
        return dx, None, None, None, dy if ctx.needs_input_grad[4] else None


def _dense(t):
    """Autograd hands over gradients of any strides; the kernels want contiguous channels."""
    return t if t.stride(-1) == 1 else t.contiguous()


def group_norm_act(x, gamma, beta, groups, eps=1e-5, act=_lib.ACT_NONE, act_first=False, lengths=None):
    """ops.group_norm_act's y, with gradients of x, gamma and beta."""
    return _GroupNormAct.apply(x, gamma, beta, groups, eps, act, act_first, lengths)


def gated_recurrence(x, gate, h0=None, lengths=None, reverse=False):
    """ops.gated_recurrence's (h, last), with gradients of x, gate and h0."""
    # within apply the gradient mode is always off, and needs_input_grad does not know of it
    return _GatedRecurrence.apply(x, gate, h0, lengths, reverse, torch.is_grad_enabled())


def dropout(x, p, rng, site=0, residual=None):
    """ops.dropout, with gradients of x and residual.  Advance rng's step after the backward pass."""
    return _Dropout.apply(x, p, rng, site, residual)
