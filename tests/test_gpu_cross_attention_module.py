"""CrossAttention: norms, rotation and attention together, as a decoder reads an encoder's states."""
from argparse import Namespace

import pytest
import torch

import lookupffn_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _config(**change):
    config = dict(hidden_size=192, num_attention_heads=3, attention_head_size=64, attention_probs_dropout_prob=0.1, layer_norm_eps=1e-5)
    return Namespace(**{**config, **change})


def _module(config, dtype=torch.float32):
    torch.manual_seed(0)
    module = lookupffn_amd.CrossAttention(config).to(DEV)
    with torch.no_grad():
        module.query_norm.add_(0.1 * torch.randn_like(module.query_norm))
        module.key_norm.add_(0.1 * torch.randn_like(module.key_norm))
    return module.to(dtype) if dtype != torch.float32 else module


def _turn(x, positions, columns):
    half = columns // 2
    angle = positions.double()[..., None] * 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    cos, sin = angle.cos()[..., None, :], angle.sin()[..., None, :]
    a, b = x[..., :half], x[..., half:columns]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., columns:]), -1)


def _reference(module, config, x, states, mask, positions, state_positions):
    """The definition in 64 bits, differentiable."""
    p = {n: t.detach().double().cpu().requires_grad_() for n, t in module.named_parameters()}
    heads, key_heads, size = config.num_attention_heads, module.num_key_value_heads, config.attention_head_size
    linear = lambda t, name: torch.nn.functional.linear(t, p[name + ".weight"], p[name + ".bias"])  # noqa: E731
    rms = lambda t, w: t / (t.pow(2).mean(-1, keepdim=True) + config.layer_norm_eps).sqrt() * w  # noqa: E731
    h = torch.nn.functional.layer_norm(x, x.shape[-1:], p["LayerNorm.weight"], p["LayerNorm.bias"], config.layer_norm_eps)
    q = rms(linear(h, "query").unflatten(-1, (heads, size)), p["query_norm"])
    k = rms(linear(states, "key").unflatten(-1, (key_heads, size)), p["key_norm"])
    v = linear(states, "value").unflatten(-1, (key_heads, size))
    columns = getattr(config, "rotary_columns", 0)
    if columns:
        q, k = _turn(q, positions, columns), _turn(k, state_positions, columns)
    k, v = (t.repeat_interleave(heads // key_heads, 2) for t in (k, v))
    s = torch.einsum("bihd,bjhd->bhij", q, k) / size ** 0.5
    s = s.masked_fill(~mask[:, None, None], -1e300)
    w = torch.softmax(s, -1) * mask.any(1)[:, None, None, None]
    return linear(torch.einsum("bhij,bjhd->bihd", w, v).flatten(2), "dense"), p


@pytest.mark.parametrize("change", [{}, dict(num_key_value_heads=1, rotary_columns=32, max_position_embeddings=300, encoder_hidden_size=96),
                                    dict(rotary_columns=64, max_position_embeddings=200)])
def test_training_against_64_bits(change):
    config = _config(**change)
    module = _module(config)
    B, L, S, width = 3, 37, 150, getattr(config, "encoder_hidden_size", 192)
    x, states = torch.randn(B, L, 192, device=DEV), torch.randn(B, S, width, device=DEV)
    lengths = torch.tensor([S, 60, 0])
    mask = torch.arange(S) < lengths[:, None]
    positions, state_positions = torch.arange(L) + 11, torch.arange(S)
    x.requires_grad_(), states.requires_grad_()
    out = module(x, states, mask.to(DEV).float(), positions=positions.to(DEV), encoder_positions=None)
    g = torch.randn(B, L, 192, device=DEV)
    names = [n for n, _ in module.named_parameters()]
    grads = torch.autograd.grad(out, (x, states, *module.parameters()), g)
    x64, s64 = x.detach().double().cpu().requires_grad_(), states.detach().double().cpu().requires_grad_()
    want, p = _reference(module, config, x64, s64, mask, positions, state_positions)
    gradients = torch.autograd.grad(want, (x64, s64, *(p[n] for n in names)), g.double().cpu())
    # a chain of six fp32 operators, each off by some 2^-21 of its result's norm (the library's products too); softmax gradients lose what their two terms have in
    # common, up to ten times; a key bias has no gradient but for that (its terms add up to zero in a head without norms, not here)
    assert (out.double().cpu() - want).norm() <= 5e-6 * want.norm()
    for name, a, b in zip(("x", "states", *names), grads, gradients):
        assert (a.double().cpu() - b).norm() <= 2e-5 * b.norm(), name


@pytest.mark.parametrize("change", [{}, dict(num_key_value_heads=1, rotary_columns=32, max_position_embeddings=300)])
def test_steps_over_kept_states(change):
    """One token at a time over states that are kept gives what the whole sequence gives."""
    module = _module(_config(**change)).eval()
    B, L, S = 2, 5, 200
    x, states = torch.randn(B, L, 192, device=DEV), torch.randn(B, S, 192, device=DEV)
    mask = torch.arange(S, device=DEV) < torch.tensor([[S], [33]], device=DEV)
    with torch.no_grad():
        whole = module(x, states, mask)
        kept = module.states(states)
        for i in range(L):
            step = module(x[:, i:i + 1], None, mask, states=kept, positions=torch.full((B, 1), i, device=DEV))
            # (another kernel, and other sizes of the library's products: fp32 both, 2^-20 of the result)
            assert (step[:, 0] - whole[:, i]).norm() <= 2e-6 * whole[:, i].norm()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_under_autocast(dtype):
    module = _module(_config(rotary_columns=64, max_position_embeddings=300))
    x, states = torch.randn(2, 40, 192, device=DEV), torch.randn(2, 100, 192, device=DEV)
    want = module(x, states)
    with torch.autocast("cuda", dtype):
        out = module(x, states)
    assert out.dtype == dtype
    # five roundings to the type on the way, each at most half a step, and the softmax's weights: of either sign, 4 half steps
    assert (out.float() - want).norm() <= 4 * torch.finfo(dtype).eps / 2 * want.norm() * 2
    out.float().square().mean().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in module.parameters())
