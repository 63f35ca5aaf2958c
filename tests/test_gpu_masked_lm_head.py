"""MaskedLMHead: its norm by this package's kernel, or by the module where that is watched or another; with labels."""
from argparse import Namespace

import pytest
import torch

import lookupffn_amd
from lookupffn_amd import MaskedLMHead

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
CONFIG = Namespace(hidden_size=64, vocab_size=300, layer_norm_eps=1e-5)


def test_hooks_on_the_norm(monkeypatch):
    torch.manual_seed(0)
    head, x, table = MaskedLMHead(CONFIG).to(DEV), torch.randn(40, 64, device=DEV), torch.randn(300, 64, device=DEV) / 8
    y = torch.randint(0, 300, (40,), device=DEV)
    calls = []
    inner = lookupffn_amd.encoder.layer_norm
    monkeypatch.setattr(lookupffn_amd.encoder, "layer_norm", lambda *a, **k: calls.append(1) or inner(*a, **k))
    loss = head(x, table, y)
    assert len(calls) == 1
    seen, grads = [], []
    handles = [head.LayerNorm.register_forward_hook(lambda m, a, out: seen.append(out)), head.LayerNorm.register_full_backward_hook(lambda m, gi, go: grads.append(go))]
    watched = head(x.clone().requires_grad_(), table, y)
    watched.backward()
    # (both norms are rounded in fp32: a loss of 6 of logits of 5, whose errors are some 2^-20 of them)
    assert len(calls) == 1 and len(seen) == len(grads) == 1 and abs(loss.item() - watched.item()) <= 6 * 2.0 ** -18
    for h in handles:
        h.remove()
    head.LayerNorm = torch.nn.Identity()
    assert head(x, table, y) != loss and len(calls) == 1
