"""CrossAttention converted to other types: its rotation stays in float32, as the operator has it.  Without a GPU."""
import copy
from argparse import Namespace

import pytest
import torch

import lookupffn_amd

CONFIG = dict(hidden_size=96, num_attention_heads=6, num_key_value_heads=2, attention_head_size=16, attention_probs_dropout_prob=0.1, layer_norm_eps=1e-5,
              rotary_columns=16, max_position_embeddings=50)


@pytest.mark.parametrize("convert", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.to(torch.bfloat16), lambda m: m.to("cpu", torch.float16),
                                     lambda m: torch.nn.ModuleList([m]).bfloat16()[0], lambda m: copy.deepcopy(m).half().float(), lambda m: m.double()])
def test_the_rotation_keeps_its_numbers(convert):
    module = lookupffn_amd.CrossAttention(Namespace(**CONFIG))
    want = module.rotary.clone()
    module = convert(module)
    assert module.rotary.dtype == torch.float32 and torch.equal(module.rotary, want)
    assert module._buffers["rotary"] is module.rotary and "rotary" not in module.state_dict()


def test_without_rotation_and_without_memory():
    module = lookupffn_amd.CrossAttention(Namespace(**{**CONFIG, "rotary_columns": 0})).bfloat16()
    assert module.rotary is None and module.query_norm.dtype == torch.bfloat16
    module = lookupffn_amd.CrossAttention(Namespace(**CONFIG)).to("meta").half()
    assert module.rotary.device.type == "meta" and module.rotary.dtype == torch.float32
    assert module.to_empty(device="cpu").rotary.device.type == "cpu"
