"""Which tables RobertaEmbeddings reads by this package's kernels, and which are torch's; without a GPU, by tensors that have no memory."""
import pickle
from argparse import Namespace

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import lookupffn_amd
from lookupffn_amd.encoder import RobertaEmbeddings

CONFIG = Namespace(hidden_size=64, vocab_size=300, max_position_embeddings=40, type_vocab_size=2, pad_token_id=1, layer_norm_eps=1e-5, hidden_dropout_prob=0.0)


@pytest.mark.parametrize("dtype,by_kernels", [(torch.float32, 3), (torch.float16, 3), (torch.bfloat16, 3), (torch.float64, 0)])
def test_types(dtype, by_kernels, monkeypatch):
    calls = []
    inner = lookupffn_amd.encoder.embedding
    monkeypatch.setattr(lookupffn_amd.encoder, "embedding", lambda *a, **k: calls.append(1) or inner(*a, **k))
    with FakeTensorMode():
        torch.set_default_dtype(dtype)
        try:
            with torch.device("cuda"):
                module = RobertaEmbeddings(CONFIG, kernels=True)
        finally:
            torch.set_default_dtype(torch.float32)
        ids = torch.zeros(2, 5, dtype=torch.int64, device="cuda")
        out = module(ids, ids, ids)
    assert len(calls) == by_kernels and out.shape == (2, 5, 64) and out.dtype == dtype


def test_a_module_that_was_pickled_without_the_choice():
    module = RobertaEmbeddings(CONFIG)
    del module.__dict__["kernels"]
    again = pickle.loads(pickle.dumps(module))
    ids = torch.zeros(2, 5, dtype=torch.int64)
    assert not again.kernels and torch.equal(again(ids, ids, ids), RobertaEmbeddings.forward(module, ids, ids, ids))
