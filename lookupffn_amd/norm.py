"""Layer norm over the last dimension, forward and backward, on hand-written kernels (csrc/layer_norm_rows.hip) in float32, float16 and bfloat16; the reference has
torch's (PL/lookup.py:84, PL/layer.py:23, src/roberta/tasks/mlm.py:33-112).  GPU only."""
from __future__ import annotations

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .cross_attention import _DTYPES, _host, _recorded, _refuse_foreign_leaves, _require


class LayerNorm(Function):
    """``layer_norm`` behind its checks, on rows: keeps its input and every row's mean and 1 / sigma."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        out, stats = ops.layer_norm(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, bias, stats)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, weight, bias, stats = ctx.saved_tensors
        wanted = ctx.needs_input_grad[0], weight is not None and ctx.needs_input_grad[1], bias is not None and ctx.needs_input_grad[2]
        grads = list(ops.layer_norm_rows_bwd(x, weight, bias, stats, g, *wanted))
        return (*(grads.pop(0) if w else None for w in wanted), None)


def layer_norm(x, weight=None, bias=None, *, eps=1e-5):
    """Layer norm over the last dimension:

        out = (x - mean(x)) / sqrt(mean((x - mean(x))^2) + eps) * weight + bias

    x: [..., columns] float32, float16 or bfloat16, with any strides (a copy is made where it is not rows of one stride), fewer than 2^24 rows of at most 2^24 columns.  weight, bias: [columns],
    both float32 or of x's type, each or None.  Sums in float32, one rounding.

    -> [..., columns] of x's type.  Gradients: x, weight and bias, sums over the rows in a fixed order, the same bits on every call; none of theirs, and none in forward mode (an error);
    captured in graphs as ``cross_attention`` is."""
    host = _host()
    if host:
        out = host.layer_norm(x, weight, bias, eps)
        if out is not None:
            return out
    _lib.require_gpu(x, weight, bias)
    _refuse_foreign_leaves(x, weight, bias)
    _require(x.dim() >= 1 and x.dtype in _DTYPES, f"x: [..., columns] float32, float16 or bfloat16, got {tuple(x.shape)} {x.dtype}")
    columns = x.shape[-1]
    _require(1 <= columns <= ops.LAYER_NORM_MAX_COLUMNS, f"x: {columns} columns")
    for name, t in (("weight", weight), ("bias", bias)):
        _require(t is None or t.shape == (columns,) and t.dtype in (torch.float32, x.dtype), f"{name}: [{columns}] float32 or {x.dtype}, got "
                 f"{None if t is None else (tuple(t.shape), t.dtype)}")
    _require(weight is None or bias is None or weight.dtype == bias.dtype, "weight and bias: of one type")
    eps = float(eps)
    _require(eps >= 0, f"eps: {eps}")
    rows = x.reshape(-1, columns)
    _require(rows.shape[0] <= ops.LAYER_NORM_MAX_ROWS, f"x: {rows.shape[0]} rows")
    args = rows, weight, bias, eps
    return (LayerNorm.apply(*args) if _recorded(x, weight, bias) else ops.layer_norm(*args, False)[0]).view(x.shape)
