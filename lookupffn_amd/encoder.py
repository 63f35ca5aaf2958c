"""The caller of the hot path: the reference's pre-norm encoder with LookupFFN in
place of the feed-forward block (PL/layer.py, PL/encoder.py, and the embeddings
of src/roberta/models/postnorm.py:6-28), with the same module and parameter
names so that a reference state_dict loads unchanged.  ``LookupFFN`` and, without
gradients, the attention's products and softmax run on the gfx950 kernels of this
package; embeddings, LayerNorms and the attention in training are plain PyTorch-ROCm.
``CrossAttention`` reads the encoder's states from another sequence, with and without gradients.  ``LookupForMaskedLM`` is
the model with what it is pre-trained by: the embeddings' gradient, the head's layer norm and the loss over the vocabulary
run on this package's kernels too.

``config`` carries the attributes the reference reads: hidden_size,
num_attention_heads, attention_head_size, attention_probs_dropout_prob,
hidden_dropout_prob, layer_norm_eps, num_hidden_layers, vocab_size,
max_position_embeddings, type_vocab_size, pad_token_id, plus LookupFFN's
(ffn_num_table, ffn_table_size, projection_type, block_size) and optionally
checkpoint_attention.
"""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.utils.checkpoint import checkpoint

from . import ops
from .cross_attention import cross_attention, qk_norm_rotary, rotary_table
from .lookup import LookupFFN
from .norm import layer_norm
from .vocabulary import embedding, linear_cross_entropy

_GLOBAL_HOOKS = torch.nn.modules.module
_FORWARDS = {kind: kind.forward for kind in (nn.Linear, nn.LayerNorm, nn.Dropout, nn.Embedding)}       # (and Attention, below)


def _plain(module, kind):
    """module is a `kind` itself, the class as it was written, and nothing watches its calls: what it computes may be computed
    without calling it."""
    return (type(module) is kind and "forward" not in module.__dict__ and kind.forward is _FORWARDS[kind]
            and not (module._forward_hooks or module._forward_pre_hooks or module._backward_hooks or module._backward_pre_hooks))


def _nobody_watches():
    """No tracer, transform, mode or hook on every module has to see the operators one by one."""
    return not (torch.compiler.is_compiling() or torch.jit.is_tracing() or torch.jit.is_scripting() or torch.is_autocast_enabled("cuda")
                or torch._C._are_functorch_transforms_active() or torch._C._len_torch_dispatch_stack()
                or torch._C._len_torch_function_stack() or torch.autograd.forward_ad._current_level >= 0
                or _GLOBAL_HOOKS._global_forward_hooks or _GLOBAL_HOOKS._global_forward_pre_hooks
                or _GLOBAL_HOOKS._global_backward_hooks or _GLOBAL_HOOKS._global_backward_pre_hooks)


def _kernel_operand(t, shape, device):
    return (type(t) in (torch.Tensor, nn.Parameter) and t.dtype == torch.float32 and t.device == device and t.shape == shape
            and t.is_contiguous() and t.data_ptr() % 16 == 0)


class RobertaEmbeddings(nn.Module):
    """word + token-type + position embeddings, LayerNorm, dropout
    (src/roberta/models/postnorm.py:6-28); positions are offset by pad_token_id + 1.

    kernels: the tables are read, and their gradients summed, by this package's ``embedding`` (the same numbers forward; gradients that cannot be
    differentiated again) wherever a table is the nn.Embedding it was built with, of float32, float16 or bfloat16.  There a word, type or position outside its table (a
    sequence longer than max_position_embeddings) has a row of zeros and no gradient, where nn.Embedding fails."""

    kernels = False                      # (of a module that was pickled without)

    def __init__(self, config, kernels=False):
        super().__init__()
        self.kernels = kernels
        self.pad_token_id = config.pad_token_id
        self.word_embeddings = nn.Embedding(config.vocab_size, config.hidden_size)
        self.position_embeddings = nn.Embedding(config.max_position_embeddings + 2, config.hidden_size)
        self.token_type_embeddings = nn.Embedding(config.type_vocab_size, config.hidden_size)
        self.LayerNorm = nn.LayerNorm(config.hidden_size, eps=config.layer_norm_eps)
        self.dropout = nn.Dropout(config.hidden_dropout_prob)

    def _rows(self, table, ids):
        if (self.kernels and _plain(table, nn.Embedding) and table.weight.is_cuda and ops.row_format(table.weight.dtype) is not None
                and table.max_norm is None and not table.sparse and not table.scale_grad_by_freq):
            return embedding(ids, table.weight, padding_idx=table.padding_idx)
        return table(ids)

    def forward(self, input_ids, token_type_ids, position_ids):
        x = (self._rows(self.word_embeddings, input_ids)
             + self._rows(self.token_type_embeddings, token_type_ids)
             + self._rows(self.position_embeddings, position_ids + (self.pad_token_id + 1)))
        return self.dropout(self.LayerNorm(x))


class Attention(nn.Module):
    """Pre-norm multi-head self-attention (PL/layer.py:11-64): LayerNorm, q/k/v
    projections, softmax(q k^T / sqrt(d) - 1000 * (1 - mask)) v in float32, output
    projection.  ``fused=True`` evaluates the same expression with
    scaled_dot_product_attention; ``fused=False`` is the reference's literal
    sequence of matmuls."""

    def __init__(self, config, fused=True):
        super().__init__()
        self.num_attention_heads = config.num_attention_heads
        self.attention_head_size = config.attention_head_size
        self.all_head_size = self.num_attention_heads * self.attention_head_size
        self.dropout = nn.Dropout(config.attention_probs_dropout_prob)
        self.checkpoint_attention = bool(getattr(config, "checkpoint_attention", False))
        self.fused = fused

        self.LayerNorm = nn.LayerNorm(config.hidden_size, eps=config.layer_norm_eps)
        self.query = nn.Linear(config.hidden_size, config.hidden_size)
        self.key = nn.Linear(config.hidden_size, config.hidden_size)
        self.value = nn.Linear(config.hidden_size, config.hidden_size)
        self.dense = nn.Linear(config.hidden_size, config.hidden_size)

    def transpose_for_scores(self, x):
        return x.view(*x.shape[:-1], self.num_attention_heads, self.attention_head_size).permute(0, 2, 1, 3)

    def attention(self, query_layer, key_layer, value_layer, attention_mask):
        bias = -1000.0 * (1.0 - attention_mask[:, None, None, :].float())
        q, k, v = query_layer.float(), key_layer.float(), value_layer.float()
        if self.fused:
            ctx = F.scaled_dot_product_attention(q, k, v, attn_mask=bias,
                                                 dropout_p=self.dropout.p if self.training else 0.0)
        else:
            scale = self.attention_head_size ** 0.25
            probs = torch.softmax(torch.matmul(q / scale, (k / scale).transpose(-1, -2)) + bias, dim=-1)
            ctx = torch.matmul(self.dropout(probs), v)
        return ctx.to(value_layer.dtype)

    def _kernels_apply(self, x, mask):
        """The products and the softmax go to this package's kernels (csrc/linear.hip, csrc/attention.hip): fp32 on the GPU in eval() without
        gradients, heads of 64 columns, and every part of the module the one it was built with.  A module in train() keeps the
        library's with and without gradients: a checkpointed pass runs both, and the LookupFFN behind turns a rounding into another
        table row.  Against the library's fp32
        products and attention the encoder layer takes, 32 x 512 tokens of 768, 624 us instead of 1279, 4 x 128 tokens 86 instead of
        164, 16 tokens 86 instead of 166, and its attention half is half as far from 64 bits (5e-7 against 9e-7)."""
        linears = (self.query, self.key, self.value, self.dense)
        if not (x.is_cuda and x.dim() == 3 and x.dtype == torch.float32 and x.numel() > 0 and type(x) in (torch.Tensor, nn.Parameter)
                and self.fused and not self.training and type(self) is Attention
                and not any(name in self.__dict__ or getattr(Attention, name) is not method for name, method in _OWN_METHODS)):
            return False
        hidden = x.shape[2]
        return (self.attention_head_size == 64 and self.all_head_size == hidden and x.shape[1] <= ops.ATTENTION_MAX_KEYS
                and type(mask) is torch.Tensor and mask.shape == x.shape[:2] and mask.device == x.device
                and all(_plain(m, nn.Linear) and _kernel_operand(m.weight, (hidden, hidden), x.device)
                        and (m.bias is None or _kernel_operand(m.bias, (hidden,), x.device)) for m in linears)
                and not (torch.is_grad_enabled()
                         and (x.requires_grad or mask.requires_grad or any(p.requires_grad for p in self.parameters())))
                and _nobody_watches())

    def _norm_applies(self, x):
        """The LayerNorm is the one the module was built with and there are rows enough that its kernel splits them, and the weights,
        once for all tiles."""
        norm, shape = self.LayerNorm, x.shape[2:]
        return (x.shape[0] * x.shape[1] >= ops.LINEAR_NORM_MIN_ROWS and shape[0] <= ops.LINEAR_NORM_MAX_COLUMNS
                and _plain(norm, nn.LayerNorm) and norm.normalized_shape == tuple(shape) and _kernel_operand(x, x.shape, x.device)
                and all(p is None or _kernel_operand(p, shape, x.device) for p in (norm.weight, norm.bias)))

    def _forward_kernels(self, hidden_states, attention_mask, residual=None):
        B, L, hidden = hidden_states.shape
        q, k, v, dense, norm = self.query, self.key, self.value, self.dense, self.LayerNorm
        weights, biases = (q.weight, k.weight, v.weight), (q.bias, k.bias, v.bias)
        if self._norm_applies(hidden_states):
            qkv = ops.linear_norm(hidden_states.view(B * L, hidden), norm.weight, norm.bias, float(norm.eps), weights, biases)
        else:
            h = norm(hidden_states)
            if not _kernel_operand(h, hidden_states.shape, hidden_states.device):        # another LayerNorm may return anything
                out = self._attend(h, attention_mask)
                return out if residual is None else out + residual
            qkv = ops.linear(h.view(B * L, hidden), weights, biases, None)
        qkv = qkv.view(3, B, L, self.num_attention_heads, 64)
        ctx = ops.attention(qkv[0], qkv[1], qkv[2], attention_mask.float().contiguous())
        if residual is not None:
            residual = residual.contiguous().view(B * L, hidden)
        return ops.linear(ctx.view(B * L, hidden), (dense.weight,), (dense.bias,), residual).view(B, L, hidden)

    def _attend(self, h, attention_mask):
        q = self.transpose_for_scores(self.query(h))
        k = self.transpose_for_scores(self.key(h))
        v = self.transpose_for_scores(self.value(h))
        if self.checkpoint_attention:
            ctx = checkpoint(self.attention, q, k, v, attention_mask, use_reentrant=False)
        else:
            ctx = self.attention(q, k, v, attention_mask)
        ctx = ctx.permute(0, 2, 1, 3).contiguous()
        return self.dense(ctx.view(*ctx.shape[:-2], self.all_head_size))

    def forward(self, hidden_states, attention_mask):
        if self._kernels_apply(hidden_states, attention_mask):
            return self._forward_kernels(hidden_states, attention_mask)
        return self._attend(self.LayerNorm(hidden_states), attention_mask)


# What the kernels stand in for: a class or a module with another one has it called.
_FORWARDS[Attention] = Attention.forward
_OWN_METHODS = tuple((name, getattr(Attention, name)) for name in ("attention", "transpose_for_scores", "_attend"))


class CrossAttention(nn.Module):
    """Pre-norm attention of a sequence to the states of an encoder, of another length (nothing in the reference, whose encoder has no reader): LayerNorm of
    the hidden states, queries from them, keys and values from the states, norms of queries and keys for each head, with ``rotary_columns`` the rotation to
    their positions, softmax over the states that take part, output projection.  Forward and backward on this package's kernels
    (``qk_norm_rotary``, ``cross_attention``) in float32 and, under autocast, 16 bits.

    ``config`` as for ``Attention``, optionally num_key_value_heads (fewer than query heads), encoder_hidden_size (of the states) and rotary_columns
    (0: no rotation; positions up to max_position_embeddings).  The weights of the softmax have no dropout: attention_probs_dropout_prob is not read."""

    def __init__(self, config):
        super().__init__()
        self.num_attention_heads = config.num_attention_heads
        self.num_key_value_heads = getattr(config, "num_key_value_heads", None) or config.num_attention_heads
        self.attention_head_size = config.attention_head_size
        self.qk_norm_eps = config.layer_norm_eps
        all_heads, key_heads = self.num_attention_heads * self.attention_head_size, self.num_key_value_heads * self.attention_head_size
        states = getattr(config, "encoder_hidden_size", None) or config.hidden_size

        self.LayerNorm = nn.LayerNorm(config.hidden_size, eps=config.layer_norm_eps)
        self.query = nn.Linear(config.hidden_size, all_heads)
        self.key = nn.Linear(states, key_heads)
        self.value = nn.Linear(states, key_heads)
        self.dense = nn.Linear(all_heads, config.hidden_size)
        self.query_norm = nn.Parameter(torch.ones(self.attention_head_size))
        self.key_norm = nn.Parameter(torch.ones(self.attention_head_size))
        columns = getattr(config, "rotary_columns", 0)
        self.register_buffer("rotary", rotary_table(config.max_position_embeddings, columns) if columns else None, persistent=False)

    def _apply(self, fn, recurse=True):
        # the rotation goes where the module goes, in float32: 16 bits would turn far positions by other angles; a module that gets its memory only now has none to bring
        table = self.rotary
        super()._apply(fn, recurse)
        if table is not None and table.is_meta and not self.rotary.is_meta:
            self.rotary = rotary_table(*table.shape, device=self.rotary.device)
        elif table is not None and self.rotary.dtype != table.dtype:
            self.rotary = table.to(self.rotary.device)
        return self

    def _heads(self, x, heads):
        return x.view(*x.shape[:-1], heads, self.attention_head_size)

    def _states(self, encoder_hidden_states):
        return (self._heads(self.key(encoder_hidden_states), self.num_key_value_heads),
                self._heads(self.value(encoder_hidden_states), self.num_key_value_heads))

    def states(self, encoder_hidden_states, positions=None):
        """Keys (normed and rotated) and values [B, states, key heads, head size] of an encoder's states [B, states, hidden], for calls that read
        the same states again, such as a decoder's next tokens."""
        keys, values = self._states(encoder_hidden_states)
        return qk_norm_rotary(keys, None, self.key_norm, table=self.rotary, q_positions=positions, eps=self.qk_norm_eps)[0], values

    def forward(self, hidden_states, encoder_hidden_states=None, encoder_attention_mask=None, *, states=None, positions=None,
                encoder_positions=None):
        """hidden_states [B, L, hidden]; either encoder_hidden_states [B, states, hidden] or what ``states`` returned for them; the mask [B, states], True or
        above 0 where a state takes part; positions of the tokens and the states (with rotary_columns), 0, 1, 2 ... if None."""
        if (states is None) == (encoder_hidden_states is None):
            raise ValueError("either encoder_hidden_states or states")
        queries = self._heads(self.query(self.LayerNorm(hidden_states)), self.num_attention_heads)
        norm = dict(table=self.rotary, q_positions=positions, eps=self.qk_norm_eps)
        if states is None:
            keys, values = self._states(encoder_hidden_states)
            queries, keys = qk_norm_rotary(queries, keys, self.query_norm, self.key_norm, k_positions=encoder_positions, **norm)
        else:
            keys, values = states
            queries, _ = qk_norm_rotary(queries, None, self.query_norm, **norm)
        mask = encoder_attention_mask
        if mask is not None and mask.dtype != torch.bool:
            mask = mask > 0
        return self.dense(cross_attention(queries, keys, values, mask).flatten(2))


class EncoderLayer(nn.Module):
    """attention + residual, LookupFFN + residual (PL/layer.py:66-78)."""

    def __init__(self, config):
        super().__init__()
        self.hidden_size = config.hidden_size
        self.FFN = LookupFFN(config, self.hidden_size)
        self.attention = Attention(config)
        self.dropout = nn.Dropout(p=config.hidden_dropout_prob)

    def _attention_and_residual(self, hidden_states, attention_mask):
        attention, dropout = self.attention, self.dropout
        if (_plain(attention, Attention) and _plain(dropout, nn.Dropout) and (not dropout.training or dropout.p == 0.0)
                and attention._kernels_apply(hidden_states, attention_mask)):
            # the residual is added where the output projection's results are stored
            return attention._forward_kernels(hidden_states, attention_mask, hidden_states)
        return dropout(attention(hidden_states, attention_mask)) + hidden_states

    def forward(self, hidden_states, attention_mask):
        attn_output = self._attention_and_residual(hidden_states, attention_mask)
        if (not self.training or self.dropout.p == 0.0) and attn_output.dtype == torch.float32:
            # dropout is the identity: the residual add runs inside the FFN's gather kernel
            return self.FFN(attn_output, residual=attn_output)
        return self.dropout(self.FFN(attn_output)) + attn_output


class Encoder(nn.Module):
    """PL/encoder.py:9-19."""

    def __init__(self, config):
        super().__init__()
        self.layer = nn.ModuleList([EncoderLayer(config) for _ in range(config.num_hidden_layers)])
        self.LayerNorm = nn.LayerNorm(config.hidden_size, eps=config.layer_norm_eps)

    def forward(self, hidden_states, attention_mask):
        for layer_module in self.layer:
            hidden_states = layer_module(hidden_states, attention_mask)
        return self.LayerNorm(hidden_states)


class Lookup(nn.Module):
    """PL/encoder.py:21-37: embeddings + encoder; returns (sequence_output, {})."""

    def __init__(self, config):
        super().__init__()
        self.config = config
        self.embeddings = RobertaEmbeddings(config)
        self.encoder = Encoder(config)

    def forward(self, input_ids, token_type_ids, position_ids, attention_mask, **kwargs):
        embedding_output = self.embeddings(input_ids, token_type_ids, position_ids)
        return self.encoder(embedding_output, attention_mask), {}

    def get_input_embeddings(self):
        return self.embeddings.word_embeddings

    def set_input_embeddings(self, value):
        self.embeddings.word_embeddings = value


class MaskedLMHead(nn.Module):
    """What the reference pre-trains its encoder by (src/roberta/tasks/mlm.py:33-112), behind the encoder: a projection, gelu and layer norm of the states, and the projection
    to the vocabulary by the word embeddings with a bias of its own.  With labels the loss, whose logits are not in memory as a whole and whose cost is that of the
    labelled tokens (``linear_cross_entropy``, GPU only; hidden_size a multiple of 8); without, the logits.  The norm is this package's ``layer_norm`` wherever it is the nn.LayerNorm
    that the head was built with and nothing watches its calls, else what stands in its place.

    ``config``: hidden_size, vocab_size, layer_norm_eps."""

    def __init__(self, config):
        super().__init__()
        self.dense = nn.Linear(config.hidden_size, config.hidden_size)
        self.LayerNorm = nn.LayerNorm(config.hidden_size, eps=config.layer_norm_eps)
        self.bias = nn.Parameter(torch.zeros(config.vocab_size))

    def forward(self, hidden_states, word_embeddings, labels=None, *, ignore_index=-100, reduction="mean"):
        """hidden_states [..., hidden], word_embeddings [vocabulary, hidden], labels [...] (ignore_index: not asked for) -> the loss, by ``reduction``; without labels
        the logits [..., vocabulary]."""
        hidden, norm = F.gelu(self.dense(hidden_states)), self.LayerNorm
        if _plain(norm, nn.LayerNorm) and hidden.is_cuda and ops.row_format(hidden.dtype) is not None and norm.normalized_shape == hidden.shape[-1:]:
            hidden = layer_norm(hidden, norm.weight, norm.bias, eps=norm.eps)
        else:
            hidden = norm(hidden)
        if labels is None:
            return F.linear(hidden, word_embeddings, self.bias)
        # (under autocast the states are 16 bits wide, and the projection is as any other's)
        return linear_cross_entropy(hidden, word_embeddings.to(hidden.dtype), self.bias, labels, ignore_index=ignore_index, reduction=reduction)


class LookupForMaskedLM(nn.Module):
    """``Lookup`` and ``MaskedLMHead``, which projects by the encoder's word embeddings: what the reference trains (src/roberta/tasks/mlm.py:33-112).  GPU only, as the
    embeddings' kernels are; forward(..., labels) -> the mean loss of the labelled tokens, without labels the logits.  Nothing is looked at on the host: numbers outside a table
    are rows of zeros (``RobertaEmbeddings``), labels outside the vocabulary are as if not asked for (``linear_cross_entropy``)."""

    def __init__(self, config):
        super().__init__()
        self.encoder = Lookup(config)
        self.encoder.embeddings.kernels = True
        self.head = MaskedLMHead(config)

    def forward(self, input_ids, token_type_ids, position_ids, attention_mask, labels=None, **kwargs):
        states, _ = self.encoder(input_ids, token_type_ids, position_ids, attention_mask, **kwargs)
        return self.head(states, self.encoder.get_input_embeddings().weight, labels)
