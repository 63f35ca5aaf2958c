"""What hooks on saved tensors give back, laid out in their own way, is read as it lies."""
import pytest
import torch

import lookupffn_amd
from lookupffn_amd import cross_attention, qk_norm_rotary, rotary_table

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("host", [True, False])
@pytest.mark.parametrize("L,keys", [(1, 90), (40, 70), (300, 200)])
def test_strided_and_shifted(L, keys, host, dtype, monkeypatch):
    if host:
        assert lookupffn_amd._lib.host()
    else:
        monkeypatch.setattr(lookupffn_amd._lib, "loaded_host", False)
    gen = torch.Generator(device=DEV).manual_seed(0)
    q, k, v, g = (torch.randn(2, n, h, 64, generator=gen, device=DEV).to(dtype) for n, h in ((L, 4), (keys, 2), (keys, 2), (L, 4)))
    w = 1 + 0.1 * torch.randn(64, generator=gen, device=DEV)
    table, mask = rotary_table(400, 32, device=DEV), torch.rand(2, keys, generator=gen, device=DEV) < 0.8

    def step(unpack):
        leaves = [t.clone().requires_grad_() for t in (q, k, v, w)]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), unpack):
            a, b = qk_norm_rotary(leaves[0], leaves[1], leaves[3], leaves[3], table=table)
            out = cross_attention(a, b, leaves[2], mask)
        return (out.detach(), *torch.autograd.grad(out, leaves, g))

    want = step(lambda t: t)
    # every number beside itself (the larger array holds whatever is read of it), and one number further
    for unpack in (lambda t: torch.stack((t, t), -1)[..., 0], lambda t: torch.cat((t.flatten()[:1], t.flatten()))[1:].view(t.shape)):
        assert all(torch.equal(a, b) for a, b in zip(step(unpack), want))


@pytest.mark.parametrize("host", [True, False])
@pytest.mark.parametrize("unpack", [lambda t: t.half() if t.dtype == torch.float32 else t, lambda t: t.float() if t.dtype == torch.float16 else t,
                                    lambda t: t[:1] if t.dim() == 4 else t, lambda t: t[:64] if t.dtype == torch.uint8 else t, lambda t: t[..., :8] if t.dtype == torch.bool else t,
                                    lambda t: t.int() if t.dtype == torch.int64 else t])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_another_type_or_shape_is_refused(dtype, unpack, host, monkeypatch):
    """Before anything is read by it (where it is what was saved, the gradients are what they were)."""
    if host:
        assert lookupffn_amd._lib.host()
    else:
        monkeypatch.setattr(lookupffn_amd._lib, "loaded_host", False)
    gen = torch.Generator(device=DEV).manual_seed(0)
    q, k, v, g = (torch.randn(2, n, h, 64, generator=gen, device=DEV).to(dtype) for n, h in ((40, 4), (70, 2), (70, 2), (40, 4)))
    w, table, mask = torch.ones(64, device=DEV), rotary_table(400, 32, device=DEV), torch.rand(2, 70, generator=gen, device=DEV) < 0.8
    at = torch.arange(40, device=DEV), torch.arange(70, device=DEV)
    seen = []

    def watched(t):
        given = unpack(t)
        seen.append(given.dtype != t.dtype or given.shape != t.shape)
        return given

    for call, inputs in ((lambda q, k, w: qk_norm_rotary(q, k, w, w, table=table, q_positions=at[0], k_positions=at[1])[0], (q, k, w)),
                         (lambda q, k, v: cross_attention(q, k, v, mask), (q, k, v))):
        leaves = [t.clone().requires_grad_() for t in inputs]
        want = torch.autograd.grad(call(*leaves), leaves, g)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), watched):
            out = call(*leaves)
        seen.clear()
        try:
            got = torch.autograd.grad(out, leaves, g)
        except (RuntimeError, AssertionError):
            assert any(seen)
        else:
            # (positions of 32 bits say the same)
            assert all(torch.equal(a, b) for a, b in zip(got, want)) and (not any(seen) or unpack(at[0]).dtype == torch.int32)
