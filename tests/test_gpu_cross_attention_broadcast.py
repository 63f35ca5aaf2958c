"""Queries, keys and values that sequences, heads or tokens share by a stride of zero: their gradients."""
import pytest
import torch

import lookupffn_amd
from lookupffn_amd import cross_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True, params=["host", "python"])
def either_path(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(lookupffn_amd._lib, "loaded_host", False)
    else:
        assert lookupffn_amd._lib.host()


def _randn(*shape, dtype, seed):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("what", ["one sequence's keys", "one sequence's values", "one sequence's both", "one head's keys", "one head's values", "one query"])
@pytest.mark.parametrize("L,keys", [(1, 200), (90, 150), (200, 70)])
def test_gradients_of_what_is_shared(L, keys, what, dtype):
    """The sum of the gradients of copies of it."""
    B, H, Hk, D = 3, 4, 2, 64
    q, k, v, g = (_randn(B, n, h, D, dtype=dtype, seed=s) for s, (n, h) in enumerate(((L, H), (keys, Hk), (keys, Hk), (L, H))))
    if "sequence" in what:
        dim, shape = 0, (B, -1, -1, -1)
    elif "head" in what:
        dim, shape = 2, (-1, -1, Hk, -1)
    else:
        dim, shape = 1, (-1, L, -1, -1)
    shared = [t.narrow(dim, 0, 1).clone().requires_grad_() if name in what or "both" in what and name != "query" else t
              for name, t in zip(("query", "keys", "values"), (q, k, v))]
    leaves = [t for t in shared if t.requires_grad]
    assert leaves
    out = cross_attention(*(t.expand(shape) if t.requires_grad else t for t in shared))
    got = torch.autograd.grad(out, leaves, g)
    copies = [(t.detach().repeat([n if i == dim else 1 for i, n in enumerate((B, L, Hk, 1))]) if t.requires_grad else t).requires_grad_(t.requires_grad) for t in shared]
    want_out = cross_attention(*copies)
    assert torch.equal(out, want_out)
    each = torch.autograd.grad(want_out, [t for t in copies if t.requires_grad], g)
    for a, b in zip(got, each):
        want = b.double().sum(dim, keepdim=True)
        n = b.shape[dim]
        # the copies' gradients, which have the same bits, are added in fp32 (n - 1 additions) and rounded to the type
        bound = (n - 1) * 2.0 ** -24 * b.double().abs().sum(dim, keepdim=True) + torch.finfo(dtype).eps / 2 * want.abs() + (2.0 ** -24 if dtype == torch.float16 else 1e-37)
        if dtype != torch.float32:      # (the engine may add in the type)
            bound = bound + (n - 1) * torch.finfo(dtype).eps / 2 * b.double().abs().sum(dim, keepdim=True)
        assert ((a.double() - want).abs() <= bound).all()
