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

from . import _lib, ops


_dropout = _norm = None          # torch.ops.t5vq's overloads, looked up once: these calls are short


def _bind():
    global _dropout, _norm
    t5vq = _lib.load_torch_ops()
    _dropout, _norm = t5vq.dropout.default, t5vq.norm.default


def _not_a_tensor(name):
    return TypeError(f"{name} must be a tensor")


def dropout(x, p: float = 0.1, residual=None, *, training: bool = True, ticket=None):
    """``residual + dropout(x)`` (or ``dropout(x)``), of residual's type; ``training=False`` drops nothing."""
    if not isinstance(x, torch.Tensor):
        raise _not_a_tensor("x")
    if not training:
        p = 0.0
    if residual is None and ops.dropout_keep_count(p) == 65536:
        return x
    if _dropout is None:
        _bind()
    return _dropout(x, residual, p, ticket)


def norm(hidden, weight, bias=None, *, kind: str = "layer", eps: float = 1e-6, p: float = 0.0, training: bool = True,
         ticket=None, out_dtype=None):
    """``dropout(norm(hidden) * weight + bias)``; ``kind``: "layer" (mean and variance) or "rms" (T5LayerNorm).
    ``out_dtype``: hidden's (default) or float32."""
    if not isinstance(hidden, torch.Tensor):
        raise _not_a_tensor("hidden")
    if kind not in ops.NORM_KINDS:
        ops._norm_kind(kind)
    if _norm is None:
        _bind()
    return _norm(hidden, None, weight, bias, ops.NORM_KINDS[kind], eps, 0.0, p if training else 0.0, ticket, out_dtype)[0]


def add_norm(hidden, branch, weight, bias=None, *, kind: str = "layer", eps: float = 1e-6, branch_p: float = 0.0,
             p: float = 0.0, training: bool = True, ticket=None, out_dtype=None):
    """``(out, sum)``: sum = hidden + dropout(branch; branch_p) in hidden's type -- the residual stream that the next
    sublayer continues -- and out = dropout(norm(sum) * weight + bias; p)."""
    if not (isinstance(hidden, torch.Tensor) and isinstance(branch, torch.Tensor)):
        raise _not_a_tensor("hidden and branch")
    if not training:
        branch_p = p = 0.0
    if kind not in ops.NORM_KINDS:
        ops._norm_kind(kind)
    if _norm is None:
        _bind()
    out, total = _norm(hidden, branch, weight, bias, ops.NORM_KINDS[kind], eps, branch_p, p, ticket, out_dtype)
    return out, total


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
