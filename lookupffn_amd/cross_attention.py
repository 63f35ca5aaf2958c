"""Attention of queries to the states of an encoder, of another length, and the norms of queries and keys for each head with the rotation
to their positions that come before it.  Forward and backward on hand-written kernels (csrc/cross_attention*.hip, csrc/qk_norm_rotary.hip) in
float32, float16 and bfloat16; nothing in the reference.  Arrays are [batch, tokens, heads, columns], as ``ops.attention`` has them and a product
leaves them; keys may have fewer heads than queries.  GPU only."""
from __future__ import annotations

import math

import torch
from torch.autograd import Function, forward_ad
from torch.autograd.function import once_differentiable
from torch.compiler import is_compiling

from . import _lib, ops

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _require(ok, what):
    if not ok:
        raise ValueError(what)


def _check_heads(name, t, like=None):
    _require(t.dim() == 4, f"{name}: [batch, tokens, heads, columns], got {tuple(t.shape)}")
    _require(t.dtype in _DTYPES, f"{name}: float32, float16 or bfloat16, got {t.dtype}")
    if like is not None:
        _require(t.dtype == like.dtype, f"{name}: {t.dtype}, queries are {like.dtype}")
        _require(t.shape[0] == like.shape[0] and t.shape[3] == like.shape[3], f"{name}: {tuple(t.shape)}, queries are {tuple(like.shape)}")


def _host():
    """The host path (csrc/host_attention.h), which answers None where it is not for a call; False where there is none."""
    if is_compiling():
        return False
    host = _lib.loaded_host
    return _lib.host() if host is None else host


def _recorded(*tensors):
    """Whether a call is the autograd function's: a gradient is recorded, or an input has a tangent of forward mode, which the function refuses and the operator
    behind it would drop."""
    tensors = [t for t in tensors if t is not None]
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        return True
    return not is_compiling() and forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _refuse_foreign_leaves(*tensors):
    """As the host path (csrc/host_attention.h) in front of its nodes: no forward is captured while a graph from before the capture holds one of its leaves, for
    the captured backward would end the process.  Without the host library nothing tells whether one does, and no forward with gradients is captured."""
    if is_compiling() or not torch.is_grad_enabled():
        return
    module = _lib.host_module()
    if module is not None:
        module.refuse_foreign_leaves(*tensors)
        return
    leaves = [t for t in tensors if t is not None and t.requires_grad and t.is_leaf and t.is_cuda]
    if leaves:
        with torch.cuda.device(leaves[0].device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("lookupffn_amd: a forward with gradients is captured only with the host library (_host.so), which looks whether a graph from "
                                   "before the capture still holds its leaves")


def rotary_table(positions, columns, base=10000.0, device=None):
    """Cosines and sines for ``qk_norm_rotary``: [positions, columns] float32, of angles p * base^(-2 i / columns) taken in 64 bits, the cosines of
    columns / 2 angles and then the sines.  columns: a multiple of 16, how many of a head are rotated."""
    _require(positions >= 1 and columns >= 16 and columns % 16 == 0, f"rotary_table: {positions} positions of {columns} columns")
    half = columns // 2
    angle = (torch.arange(positions, dtype=torch.float64, device=device)[:, None]
             * float(base) ** (-torch.arange(half, dtype=torch.float64, device=device) / half))
    return torch.cat((angle.cos(), angle.sin()), dim=1).float()


class QkNormRotary(Function):
    """``qk_norm_rotary`` behind its checks: saves what it is given; the norms are formed again in the backward."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, table, q_positions, k_positions, eps, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, table, q_positions, k_positions)
        ctx.eps, ctx.interleaved = eps, interleaved
        out = ops.qk_norm_rotary(q, k, q_weight, k_weight, table, q_positions, k_positions, eps, interleaved)
        return out[0], (out[1] if k is not None else None)

    @staticmethod
    @once_differentiable
    def backward(ctx, g_q, g_k):
        q, k, q_weight, k_weight, table, q_positions, k_positions = ctx.saved_tensors
        want = [q_weight is not None and ctx.needs_input_grad[2], k_weight is not None and ctx.needs_input_grad[3]]
        g_q = torch.zeros(q.shape, dtype=q.dtype, device=q.device) if g_q is None else g_q
        if k is not None:
            g_k = torch.zeros(k.shape, dtype=k.dtype, device=k.device) if g_k is None else g_k
        grads = list(ops.qk_norm_rotary_bwd(q, k, q_weight, k_weight, table, q_positions, k_positions, ctx.eps, ctx.interleaved, g_q, g_k, *want))
        grad_q, grad_k = grads.pop(0), None if k is None else grads.pop(0)
        grad_qw = grads.pop(0) if want[0] else None
        return grad_q, grad_k, grad_qw, (grads.pop(0) if want[1] else None), None, None, None, None, None


def _positions(name, p, t):
    if p is None or t is None:
        return None
    _require(p.dtype in (torch.int32, torch.int64), f"{name}: int32 or int64, got {p.dtype}")
    _require(p.shape == (t.shape[1],) or p.shape == t.shape[:2], f"{name}: {tuple(p.shape)} for {tuple(t.shape)}")
    return p


def _weight(name, w, t):
    if w is None or t is None:
        return None
    _require(w.shape == (t.shape[3],) and w.dtype in (torch.float32, t.dtype), f"{name}: [{t.shape[3]}] float32 or {t.dtype}, got {tuple(w.shape)} {w.dtype}")
    return w.float()


def qk_norm_rotary(q, k=None, q_weight=None, k_weight=None, *, table=None, q_positions=None, k_positions=None, eps=1e-6, interleaved=False):
    """Root-mean-square norms of queries and keys over the columns of each head, times a weight, and the rotation of their first columns
    to their positions, in one pass over both:

        y = x / sqrt(mean(x^2) + eps) * weight;  (a, b) -> (a cos - b sin, b cos + a sin)

    q: [B, L, heads, columns], k: [B, keys, key heads, columns] of the same type or None (single tokens against keys that are kept; their weight
    and positions are then left alone), with any strides (a copy is made where the columns do not lie together or not at multiples of 16 bytes).
    columns: a multiple of 8, at most 256.
    weights: [columns], float32 or of q's type, or None.  table: ``rotary_table`` or any [positions, rotated columns] float32 of cosines and then sines, or
    None for no rotation.  positions: int32 or int64, [L] or [B, L], or None for 0, 1, 2 ...; one outside the table takes its nearest row.  Pairs are columns
    (i, i + rotated / 2), with ``interleaved`` (2 i, 2 i + 1).  Norms and rotation in float32, one rounding.

    -> (q, k) in new contiguous arrays, k None where it was.  Gradients: q, k and both weights; sums in a fixed order; captured in graphs as ``cross_attention`` is."""
    host = _host()
    if host:
        out = host.qk_norm_rotary(q, k, q_weight, k_weight, table, q_positions, k_positions, eps, interleaved)
        if out is not None:
            return out
    _lib.require_gpu(q, k, q_weight, k_weight, table, q_positions, k_positions)
    _refuse_foreign_leaves(q, k, q_weight, k_weight if k is not None else None)
    _check_heads("q", q)
    columns = q.shape[3]
    _require(columns % 8 == 0 and 8 <= columns <= ops.QK_NORM_MAX_COLUMNS, f"q: heads of {columns} columns")
    if k is not None:
        _check_heads("k", k, q)
    _require(eps >= 0, f"eps: {eps}")
    q_weight, k_weight = _weight("q_weight", q_weight, q), _weight("k_weight", k_weight, k)
    if table is not None:
        _require(table.dim() == 2 and table.dtype == torch.float32 and table.shape[0] >= 1 and not table.requires_grad,
                 f"table: [positions, columns] float32 without gradient, got {tuple(table.shape)} {table.dtype}")
        _require(table.shape[1] % 16 == 0 and 16 <= table.shape[1] <= columns, f"table: {table.shape[1]} of {columns} columns")
    q_positions, k_positions = _positions("q_positions", q_positions, q), _positions("k_positions", k_positions, k)
    if q_positions is not None and k_positions is not None and q_positions.dtype != k_positions.dtype:
        q_positions, k_positions = q_positions.long(), k_positions.long()
    args = (q, k, q_weight, k_weight, table, q_positions, k_positions, float(eps),
            bool(interleaved))
    if _recorded(*args[:4]):
        return QkNormRotary.apply(*args)
    out = ops.qk_norm_rotary(*args)
    return out[0], (out[1] if k is not None else None)


class CrossAttentionFunction(Function):
    """``cross_attention`` behind its checks: keeps the result for the backward, with a number a row and what the result's rounding took."""

    @staticmethod
    def forward(ctx, q, k, v, key_mask, scale):
        out, kept = ops.cross_attention(q, k, v, key_mask, scale, True)
        ctx.save_for_backward(q, k, v, key_mask, out, kept)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        q, k, v, key_mask, out, kept = ctx.saved_tensors
        of_queries, of_keys = ctx.needs_input_grad[0], ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        grads = list(ops.cross_attention_bwd(q, k, v, key_mask, ctx.scale, out, kept, g, of_queries, of_keys))
        return ((grads.pop(0) if of_queries else None), *(grads if of_keys else (None, None)), None, None)


def cross_attention(q, k, v, key_mask=None, *, scale=None):
    """out[b, i, h] = sum_j p_j v[b, j, h'],  p = softmax_j(scale q[b, i, h] . k[b, j, h']) over the keys that take part.

    q: [B, L, heads, columns], k, v: [B, keys, key heads, columns], of one type, with any strides (as for ``qk_norm_rotary``); heads a multiple of
    key heads, neighbouring query heads share one.  columns: a multiple of 8, at most 128.  key_mask: [B, keys] bool, True where a key takes part, or
    None; whatever keys and values that take no part hold.  A query without keys gets zeros (and gives none a gradient).
    scale: positive, 1 / sqrt(columns) if None.  One query a sequence is the step of a decoder over kept keys and values.

    float32: products of two half-precision or three bfloat16 terms a number, sums in float32, errors of the size of float32 products' (results 2e-7 to 4e-7 of their norm with up
    to 700 keys, 1.1e-6 with 8192, 2.3e-6 with 32768; gradients 3e-7 to 6.3e-7 with up to 700 rows and keys, 2.5e-6 with 32768 keys,
    3.5e-6 with scores up to 40); with two terms (large
    calls, and the backward) a number of k or v (backward: also q and the gradient) 2^14 times smaller than the longest row of its batch and head begins to lose
    bits.  16 bits: softmax weights (backward: the scores' gradients, too) rounded to the type, sums in float32, one rounding of the result; a half-precision gradient row 2^16 times smaller than
    the longest of its batch and head begins to lose bits.  Infinities and NaN of keys that take part may make any result of their head NaN.
    -> [B, L, heads, columns].  Gradients: q, k and v, the same bits on every call; none of theirs, and none in forward mode (an error).  A step with its backward can be captured in a
    graph, but not while an earlier graph holds its leaves (RuntimeError)."""
    host = _host()
    if host:
        out = host.cross_attention(q, k, v, key_mask, scale)
        if out is not None:
            return out
    _lib.require_gpu(q, k, v, key_mask)
    _refuse_foreign_leaves(q, k, v)
    _check_heads("q", q)
    _check_heads("k", k, q)
    _check_heads("v", v, q)
    columns, heads, key_heads = q.shape[3], q.shape[2], k.shape[2]
    _require(v.shape == k.shape, f"v: {tuple(v.shape)}, k is {tuple(k.shape)}")
    _require(columns % 8 == 0 and 8 <= columns <= ops.CROSS_ATTENTION_MAX_COLUMNS, f"q: heads of {columns} columns")
    _require(key_heads >= 1 and heads % key_heads == 0, f"{heads} heads for {key_heads} key heads")
    if key_mask is not None:
        _require(key_mask.dtype == torch.bool and key_mask.shape == k.shape[:2],
                 f"key_mask: {tuple(k.shape[:2])} bool, got {tuple(key_mask.shape)} {key_mask.dtype}")
    scale = columns ** -0.5 if scale is None else float(scale)
    _require(0 < scale < math.inf, f"scale: {scale}")
    if _recorded(q, k, v):
        return CrossAttentionFunction.apply(q, k, v, key_mask, scale)
    return ops.cross_attention(q, k, v, key_mask, scale, False)[0]
