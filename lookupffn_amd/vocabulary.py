"""Both ends of a language model's vocabulary: the rows of an embedding table, and the softmax cross entropy of a projection back to it.  Forward and
backward on hand-written kernels (csrc/embedding.hip, csrc/linear_cross_entropy.hip) in float32, float16 and bfloat16; the reference has torch's
(src/roberta/models/postnorm.py:6-28, src/roberta/tasks/mlm.py:33-112).  GPU only."""
from __future__ import annotations

import math

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .cross_attention import _DTYPES, _host, _recorded, _refuse_foreign_leaves, _require


class Embedding(Function):
    """``embedding`` behind its checks, on a list of tokens: keeps their numbers."""

    @staticmethod
    def forward(ctx, ids, weight, scale, padding):
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale, ctx.padding = weight.shape[0], scale, padding
        return ops.embedding(ids, weight, scale, padding)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        return None, ops.embedding_bwd(ctx.saved_tensors[0], g, ctx.rows, ctx.scale, ctx.padding), None, None


def embedding(ids, weight, *, scale=1.0, padding_idx=None):
    """Rows of a table by token number, times a scale:

        out[..., :] = scale * weight[ids[...], :]

    ids: int32 or int64, any shape; one outside the table gives zeros and no gradient.  weight: [rows, columns] float32, float16 or bfloat16, with any strides (a copy is made where
    columns do not lie together); columns at most 2^20.  Products in float32, one rounding.  padding_idx: a row that gets no gradient, counted from the end where negative.

    -> [..., columns] of weight's type.  Gradient: weight, the whole table, from the tokens sorted by their numbers: sums in float32 in a fixed order, one rounding, the same bits on
    every call; none of its own, and none in forward mode (an error); captured in graphs as ``cross_attention`` is."""
    host = _host()
    if host:
        out = host.embedding(ids, weight, scale, padding_idx)
        if out is not None:
            return out
    _lib.require_gpu(ids, weight)
    _refuse_foreign_leaves(weight)
    _require(ids.dtype in (torch.int32, torch.int64), f"ids: int32 or int64, got {ids.dtype}")
    _require(weight.dim() == 2 and weight.dtype in _DTYPES, f"weight: [rows, columns] float32, float16 or bfloat16, got {tuple(weight.shape)} {weight.dtype}")
    rows, columns = weight.shape
    _require(rows <= ops.EMBEDDING_MAX_ROWS and 1 <= columns <= ops.EMBEDDING_MAX_COLUMNS, f"weight: {tuple(weight.shape)}")
    _require(ids.numel() < 1 << 31, f"ids: {ids.numel()} tokens")
    _require(padding_idx is None or -rows <= padding_idx < rows, f"padding_idx: {padding_idx} of {rows} rows")
    scale = float(scale)
    _require(math.isfinite(scale), f"scale: {scale}")
    args = ids.reshape(-1), weight, scale, -1 if padding_idx is None else int(padding_idx) % rows
    out = Embedding.apply(*args) if _recorded(weight) else ops.embedding(*args)
    return out.view(*ids.shape, columns)


class LinearCrossEntropy(Function):
    """``linear_cross_entropy`` behind its checks, on rows of tokens: keeps where the labelled tokens are and two numbers of each for the backward."""

    @staticmethod
    def forward(ctx, hidden, weight, bias, labels, ignore_index, reduction):
        loss, kept = ops.linear_cross_entropy(hidden, weight, bias, labels, ignore_index, reduction, True)
        ctx.save_for_backward(hidden, weight, bias, labels, kept)
        ctx.ignore_index, ctx.reduction = ignore_index, reduction
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        hidden, weight, bias, labels, kept = ctx.saved_tensors
        wanted = ctx.needs_input_grad[0], ctx.needs_input_grad[1], bias is not None and ctx.needs_input_grad[2]
        grads = list(ops.linear_cross_entropy_bwd(hidden, weight, bias, labels, ctx.ignore_index, ctx.reduction, kept, g, *wanted))
        return (*(grads.pop(0) if w else None for w in wanted), None, None, None)


def linear_cross_entropy(hidden, weight, bias, labels, *, ignore_index=-100, reduction="mean"):
    """Softmax cross entropy of the logits hidden W^T + bias, which are not in memory as a whole:

        loss_n = log sum_v exp l_nv - l_n,label(n),  l_nv = hidden[n] . weight[v] + bias[v]

    hidden: [..., columns], weight: [vocabulary, columns] of its type, columns a multiple of 8 (at most 65536; vocabulary at most 2^22, tokens at most 2^24,
    2^32 numbers of hidden), with any strides (a copy is made where columns do not lie together or rows not at multiples of 16 bytes); bias: [vocabulary],
    float32 or of that type, or None; labels: [...] int32 or int64. A token whose label is ignore_index, or no number of the vocabulary, has no part in
    anything, whatever its row holds, and costs nothing: its loss and gradient are zeros. reduction: "mean" over the tokens that have a label (0 of none),
    "sum", or "none" (the shape of labels).

    float32: products of two half-precision terms a number, sums in float32, errors of the size of float32 products'; in the backward a number of hidden or
    weight is held to 2^-22 of the largest of its row, and a gradient of the logits to 2^-38 of the largest token's.  Where that would cost others their bits
    (labelled rows of hidden, or rows of weight, more than 2^16 apart, logits that may be 2^18, tokens' gradients more than 2^8 apart; zeros aside) its
    products are of the floats as they are, at a quarter of the speed.
    16 bits: sums in float32; in the backward the gradients of the logits are rounded to the type (half: held to 2^-38 of the largest token's), a float32
    bias's gradient is the sum of those.
    Memory, beside 16 to 20 bytes a token: both directions lay hidden's rows out once more, in whole 128 columns, and float32 weights (not in the forward of few tokens).  The
    forward has 8 bytes a token, labelled or not, for every 256 entries of the vocabulary (1.6 KB of 50265).  The backward has up to 1 GB for the logits' gradients, or, if that is more, 4.2 KB a
    token (float32 8.4), up to 256 MB, or 4 bytes a number of hidden, for sums of hidden's gradient, and up to 512 MB for weight's, where that is small and the tokens are many.  Of up to 64 tokens the
    logits are kept for it where they are no more bytes than weight.
    -> float32.  Gradients: hidden, weight and bias, the same bits on every call; none of theirs, and none in forward mode (an error); captured in graphs as ``cross_attention`` is."""
    host = _host()
    if host:
        out = host.linear_cross_entropy(hidden, weight, bias, labels, ignore_index, reduction)
        if out is not None:
            return out
    _lib.require_gpu(hidden, weight, bias, labels)
    _refuse_foreign_leaves(hidden, weight, bias)
    _require(hidden.dim() >= 1 and hidden.dtype in _DTYPES, f"hidden: [..., columns] float32, float16 or bfloat16, got {tuple(hidden.shape)} {hidden.dtype}")
    columns = hidden.shape[-1]
    _require(columns % 8 == 0 and 8 <= columns <= ops.LOSS_MAX_COLUMNS, f"hidden: {columns} columns")
    _require(weight.dim() == 2 and weight.shape[1] == columns and 1 <= weight.shape[0] <= ops.LOSS_MAX_VOCABULARY and weight.dtype == hidden.dtype,
             f"weight: [vocabulary, {columns}] {hidden.dtype}, got {tuple(weight.shape)} {weight.dtype}")
    _require(bias is None or bias.shape == weight.shape[:1] and bias.dtype in (torch.float32, hidden.dtype),
             f"bias: [{weight.shape[0]}] float32 or {hidden.dtype}, got {None if bias is None else (tuple(bias.shape), bias.dtype)}")
    _require(labels.shape == hidden.shape[:-1] and labels.dtype in (torch.int32, torch.int64),
             f"labels: {tuple(hidden.shape[:-1])} int32 or int64, got {tuple(labels.shape)} {labels.dtype}")
    _require(labels.numel() <= ops.LOSS_MAX_TOKENS and hidden.numel() <= ops.LOSS_MAX_NUMBERS, f"hidden: {tuple(hidden.shape)}")
    _require(reduction in ops.REDUCTIONS, f"reduction: {reduction!r}")
    _require(isinstance(ignore_index, int) and -1 << 63 <= ignore_index < 1 << 63, f"ignore_index: {ignore_index!r}")
    args = hidden.reshape(-1, columns), weight, bias, labels.reshape(-1), ignore_index, ops.REDUCTIONS.index(reduction)
    out = LinearCrossEntropy.apply(*args) if _recorded(hidden, weight, bias) else ops.linear_cross_entropy(*args, False)[0]
    return out.view(labels.shape) if reduction == "none" else out
