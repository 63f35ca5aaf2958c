"""CrossAttention held in 16 bits, with rotation: forward, kept states, training, against the same weights in float32."""
from argparse import Namespace

import pytest
import torch

import lookupffn_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("columns", [0, 32, 64])
def test_in_16_bits(columns, dtype):
    torch.manual_seed(0)
    config = Namespace(hidden_size=192, num_attention_heads=3, num_key_value_heads=1, attention_head_size=64, attention_probs_dropout_prob=0.1, layer_norm_eps=1e-5,
                       rotary_columns=columns, max_position_embeddings=300)
    module = lookupffn_amd.CrossAttention(config).to(DEV, dtype)
    whole = lookupffn_amd.CrossAttention(config).to(DEV)
    whole.load_state_dict(module.state_dict())
    x, states = (torch.randn(2, n, 192, device=DEV).to(dtype) for n in (40, 100))
    mask = torch.arange(100, device=DEV) < torch.tensor([[100], [37]], device=DEV)
    positions = torch.arange(40, device=DEV) + 250
    want = whole(x.float(), states.float(), mask, positions=positions)
    out = module(x, states, mask, positions=positions)
    assert out.dtype == dtype
    # roundings of the hidden states, projections, queries, keys and values, weights, results: 8 half steps, each with its own sign, twice for what the norms spread
    u = torch.finfo(dtype).eps / 2
    assert (out.float() - want).norm() <= 8 * u * want.norm()
    # gradients: the same roundings again on the way back, and of ds what its two terms have in common, four times their difference
    g = torch.randn_like(want)
    names = [n for n, _ in module.named_parameters()]
    grads = torch.autograd.grad(out, list(module.parameters()), g.to(dtype))
    gradients = torch.autograd.grad(want, list(whole.parameters()), g)
    for name, a, b in zip(names, grads, gradients):
        assert a.dtype == dtype and a.isfinite().all()
        if name != "key.bias":          # (what a norm and a softmax leave of it is little beside its terms)
            assert (a.float() - b).norm() <= 32 * u * b.norm(), name
    with torch.no_grad():
        kept = module.states(states)
        step = module(x[:, 3:4], None, mask, states=kept, positions=positions[3:4])
        assert (step[:, 0].float() - want[:, 3]).norm() <= 8 * u * want[:, 3].norm()
