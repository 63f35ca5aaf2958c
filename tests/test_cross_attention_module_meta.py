"""CrossAttention made without memory and given it afterwards: its rotation, which no state_dict holds, is there.  Without a GPU."""
from argparse import Namespace

import pytest
import torch

import lookupffn_amd

CONFIG = dict(hidden_size=96, num_attention_heads=6, attention_head_size=16, attention_probs_dropout_prob=0.1, layer_norm_eps=1e-5, rotary_columns=16, max_position_embeddings=50)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_rotation_is_made_again(dtype):
    want = lookupffn_amd.CrossAttention(Namespace(**CONFIG)).to(dtype)
    with torch.device("meta"):
        module = lookupffn_amd.CrossAttention(Namespace(**CONFIG)).to(dtype)
    assert module.rotary.is_meta
    parent = torch.nn.ModuleList([module]).to_empty(device="cpu")
    parent[0].load_state_dict(want.state_dict())
    assert module.rotary.dtype == torch.float32 and torch.equal(module.rotary, want.rotary)
    assert all(torch.equal(a, b) for a, b in zip(module.parameters(), want.parameters()))
