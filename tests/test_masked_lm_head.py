"""MaskedLMHead calls what stands in its norm's place; without a GPU."""
from argparse import Namespace

import torch
import torch.nn.functional as F
from torch._subclasses.fake_tensor import FakeTensorMode

from lookupffn_amd import MaskedLMHead

CONFIG = Namespace(hidden_size=64, vocab_size=300, max_position_embeddings=40, type_vocab_size=2, pad_token_id=1, layer_norm_eps=1e-5, hidden_dropout_prob=0.0)


def test_the_norm_is_called_where_it_is_watched():
    head, x, table = MaskedLMHead(CONFIG), torch.randn(3, 64), torch.randn(300, 64)
    seen = []
    head.LayerNorm.register_forward_hook(lambda module, args, out: seen.append(out))
    logits = head(x, table)
    assert len(seen) == 1 and torch.equal(logits, F.linear(seen[0], table, head.bias))
    handle = head.LayerNorm.register_forward_hook(lambda module, args, out: 2 * out)
    assert torch.equal(head(x, table), F.linear(2 * seen[0], table, head.bias))
    handle.remove()


def test_another_norm_is_what_runs():
    head, x, table = MaskedLMHead(CONFIG), torch.randn(3, 64), torch.randn(300, 64)
    head.LayerNorm = torch.nn.Identity()
    assert torch.equal(head(x, table), F.linear(F.gelu(head.dense(x)), table, head.bias))

    class Shifted(torch.nn.LayerNorm):
        def forward(self, x):
            return super().forward(x) + 1

    head.LayerNorm = Shifted(64)
    want = F.layer_norm(F.gelu(head.dense(x)), (64,), head.LayerNorm.weight, head.LayerNorm.bias, 1e-5) + 1
    assert torch.equal(head(x, table), F.linear(want, table, head.bias))


def test_logits_of_a_type_that_no_kernel_takes():
    with FakeTensorMode():
        torch.set_default_dtype(torch.float64)
        try:
            with torch.device("cuda"):
                head, x, table = MaskedLMHead(CONFIG), torch.randn(3, 64), torch.randn(300, 64)
        finally:
            torch.set_default_dtype(torch.float32)
        out = head(x, table)
    assert out.shape == (3, 300) and out.dtype == torch.float64
