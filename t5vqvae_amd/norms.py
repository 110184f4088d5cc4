"""Dropout whose mask is never stored, layer / RMS norm, and the sum of a residual stream with a sublayer's output followed
by the norm: what stands in front of the quantizer in an encoder (python_transformers/modeling_t5.py:191-207, :864-865),
each ONE kernel forward and one (plus a small reduction for the parameters' gradients) backward.

    y        = dropout(x, p, residual)                       residual + dropout(x)
    out      = norm(hidden, weight, bias, p=p)                dropout(norm(hidden) * weight + bias)
    out, sum = add_norm(hidden, branch, weight, bias, ...)    sum = hidden + dropout(branch); out as above from sum

fp32, bf16 and fp16 tensors of any shape [..., D] on a ROCm device; an fp32 residual stream may meet a bf16 or fp16 branch
(autocast).  Arithmetic and statistics are fp32, outputs are rounded once.

Random numbers: by default a call moves torch's generator of the device on (``torch.manual_seed``, ``torch.cuda.get_rng_state``
and activation checkpointing work as with torch's own dropout; a captured graph draws anew on every replay).  A ``ticket`` --
an int64 tensor {seed, offset} on the device -- fixes the mask instead: the same ticket gives the same mask, and tickets whose
offsets are 8 apart share no numbers.  Bits of an element depend on its row and column only, not on the tensor's type, so
``add_norm`` drops exactly what ``dropout`` of the same ticket does.  p is rounded to a multiple of 2^-16 and the scale is that
of the rounded p (include/t5vq.h); dropped values are 0 even where they were infinite or NaN.
"""
from __future__ import annotations

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib, ops


def _rows(t, name, like=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    ops.require_device(t, name)
    if t.dim() == 0:
        raise RuntimeError(f"{name} must have at least one dimension")
    if like is not None and t.shape != like.shape:
        raise RuntimeError(f"{name} must have shape {tuple(like.shape)}, got {tuple(t.shape)}")
    if t.shape[-1] == 0:
        raise RuntimeError(f"{name} has rows of length 0")
    return t.reshape(-1, t.shape[-1]).contiguous()


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, ticket):
        y, drawn = ops.dropout_add(x, p, residual, ticket)
        ctx.save_for_backward(ticket if ticket is not None else drawn)
        ctx.p, ctx.dtype = p, x.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        (ticket,) = ctx.saved_tensors
        gx = None
        if ctx.needs_input_grad[0]:
            gx = ops.dropout_backward(g.contiguous(), ctx.p, ticket, ctx.dtype)
        return gx, (g if ctx.needs_input_grad[1] else None), None, None


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, branch, weight, bias, ticket, kind, eps, branch_p, p, out_dtype, row_norms, token_image):
        out, total, stats, xx, drawn = ops.norm_forward(
            hidden, weight, bias, kind=kind, eps=eps, branch=branch, branch_p=branch_p, p=p, ticket=ticket,
            out_dtype=out_dtype, want_row_norms=row_norms, token_image=token_image)
        ctx.save_for_backward(hidden if total is None else total, weight, stats, ticket if ticket is not None else drawn)
        ctx.kind, ctx.branch_p, ctx.p = kind, branch_p, p
        ctx.branch_dtype = None if branch is None else branch.dtype
        ctx.set_materialize_grads(False)
        if xx is not None:
            ctx.mark_non_differentiable(xx)
        return out, total, xx

    @staticmethod
    @once_differentiable
    def backward(ctx, g_out, g_sum, _):
        h, weight, stats, ticket = ctx.saved_tensors
        need_hidden, need_branch, need_weight, need_bias = ctx.needs_input_grad[:4]
        rest = (None,) * 8
        g_sum = None if g_sum is None else g_sum.contiguous()
        if g_out is None:                                       # nothing came back through the norm: the sum's gradient only
            gb = None
            if need_branch and g_sum is not None:
                gb = ops.dropout_backward(g_sum, ctx.branch_p, ticket, ctx.branch_dtype)
            return (g_sum if need_hidden else None, gb, None, None) + rest
        # without a dropout of the branch its gradient is the stream's, unless it is of another type
        same = ctx.branch_dtype == h.dtype and ops.dropout_keep_count(ctx.branch_p) == 65536
        gh, gb, gw, gbias = ops.norm_backward(
            g_out.contiguous(), g_sum, h, weight, stats, kind=ctx.kind, branch_p=ctx.branch_p, p=ctx.p, ticket=ticket,
            branch_dtype=ctx.branch_dtype if need_branch and not same else None, want_weight=need_weight, want_bias=need_bias)
        if need_branch and same:
            gb = gh
        return (gh if need_hidden else None, gb, gw, gbias) + rest


def _norm_call(hidden, branch, weight, bias, kind, eps, branch_p, p, ticket, out_dtype, row_norms=False, token_image=None):
    """(out, sum | None, xx | None) of [N, D] rows, with a gradient where one is wanted."""
    if _wants_grad(hidden, branch, weight, bias):
        return _Norm.apply(hidden, branch, weight, bias, ticket, kind, eps, branch_p, p, out_dtype, row_norms, token_image)
    out, total, _, xx, _ = ops.norm_forward(hidden, weight, bias, kind=kind, eps=eps, branch=branch, branch_p=branch_p, p=p,
                                            ticket=ticket, out_dtype=out_dtype, want_stats=False, want_row_norms=row_norms,
                                            token_image=token_image)
    return out, total, xx


def dropout(x, p: float = 0.1, residual=None, *, training: bool = True, ticket=None):
    """``residual + dropout(x)`` (or ``dropout(x)``), of residual's type; ``training=False`` drops nothing."""
    p = float(p) if training else 0.0
    rows = _rows(x, "x")
    if residual is None and ops.dropout_keep_count(p) == 65536:
        return x
    res = None if residual is None else _rows(residual, "residual", x)
    y = (_DropoutAdd.apply(rows, res, p, ticket) if _wants_grad(rows, res)
         else ops.dropout_add(rows, p, res, ticket)[0])
    return y.view(x.shape)


def norm(hidden, weight, bias=None, *, kind: str = "layer", eps: float = 1e-6, p: float = 0.0, training: bool = True,
         ticket=None, out_dtype=None):
    """``dropout(norm(hidden) * weight + bias)``; ``kind``: "layer" (mean and variance) or "rms" (T5LayerNorm).
    ``out_dtype``: hidden's (default) or float32."""
    rows = _rows(hidden, "hidden")
    out, _, _ = _norm_call(rows, None, weight, bias, kind, float(eps), 0.0, float(p) if training else 0.0, ticket, out_dtype)
    return out.view(hidden.shape)


def add_norm(hidden, branch, weight, bias=None, *, kind: str = "layer", eps: float = 1e-6, branch_p: float = 0.0,
             p: float = 0.0, training: bool = True, ticket=None, out_dtype=None):
    """``(out, sum)``: sum = hidden + dropout(branch; branch_p) in hidden's type -- the residual stream that the next
    sublayer continues -- and out = dropout(norm(sum) * weight + bias; p)."""
    rows, add = _rows(hidden, "hidden"), _rows(branch, "branch", hidden)
    if not training:
        branch_p = p = 0.0
    out, total, _ = _norm_call(rows, add, weight, bias, kind, float(eps), float(branch_p), float(p), ticket, out_dtype)
    return out.view(hidden.shape), total.view(hidden.shape)


class Dropout(nn.Module):
    """``nn.Dropout`` without a stored mask, with the residual sum behind it on request."""

    def __init__(self, p: float = 0.1):
        super().__init__()
        _lib.load_all()
        ops.dropout_keep_count(p)                                # refuses p outside [0, 1]
        self.p = float(p)

    def forward(self, x, residual=None, ticket=None):
        return dropout(x, self.p, residual, training=self.training, ticket=ticket)

    def extra_repr(self):
        return f"p={self.p}"


class Norm(nn.Module):
    """``nn.LayerNorm`` (kind="layer") / T5LayerNorm (kind="rms") with the dropout behind it; called with a ``branch`` it
    adds that (with its own dropout) to ``hidden`` first and returns ``(out, sum)``.  Same state_dict keys: weight (, bias)."""

    def __init__(self, hidden_size: int, kind: str = "layer", eps: float = 1e-6, bias=None, dropout_rate: float = 0.0,
                 branch_dropout_rate: float = 0.0):
        super().__init__()
        _lib.load_all()
        ops._norm_kind(kind)
        for p in (dropout_rate, branch_dropout_rate):
            ops.dropout_keep_count(p)
        self.kind, self.eps = kind, float(eps)
        self.dropout_rate, self.branch_dropout_rate = float(dropout_rate), float(branch_dropout_rate)
        self.weight = nn.Parameter(torch.ones(hidden_size))
        self.bias = nn.Parameter(torch.zeros(hidden_size)) if (kind == "layer" if bias is None else bias) else None

    def forward(self, hidden, branch=None, ticket=None, out_dtype=None):
        if branch is None:
            return norm(hidden, self.weight, self.bias, kind=self.kind, eps=self.eps, p=self.dropout_rate,
                        training=self.training, ticket=ticket, out_dtype=out_dtype)
        return add_norm(hidden, branch, self.weight, self.bias, kind=self.kind, eps=self.eps,
                        branch_p=self.branch_dropout_rate, p=self.dropout_rate, training=self.training, ticket=ticket,
                        out_dtype=out_dtype)

    def extra_repr(self):
        return (f"{self.weight.numel()}, kind={self.kind!r}, eps={self.eps}, dropout_rate={self.dropout_rate}, "
                f"branch_dropout_rate={self.branch_dropout_rate}")
