"""linear_cross_entropy whose logits' gradients are formed in several pieces of the vocabulary that the pieces do not divide, with several tiles of columns, every token labelled and some:
against 64 bits."""
import math

import pytest
import torch

import lookupffn_amd
from lookupffn_amd import linear_cross_entropy

from _loss_reference import reference, worst

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True, params=["host", "python"])
def either_path(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(lookupffn_amd._lib, "loaded_host", False)
    else:
        assert lookupffn_amd._lib.host()


@pytest.mark.parametrize("N,dtype,share,factor", [(24000, torch.float16, 1.0, 1.0), (24000, torch.bfloat16, 0.9, 1.0), (12000, torch.float32, 1.0, 1.0), (12000, torch.float32, 0.95, 1e9)])
def test_pieces_that_the_tiles_do_not_divide_into(N, dtype, share, factor):
    """196 tiles of the vocabulary in three pieces of 66, 66 and 64: the last one has fewer of dh's shares."""
    V, K = 50000, 264
    gen = torch.Generator(device=DEV).manual_seed(N)
    randn = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    h, w, b = randn(N, K), (1.5 / math.sqrt(K) * randn(V, K)).to(dtype), 0.3 * randn(V)
    h[77] *= factor
    h = h.to(dtype)
    y = torch.randint(0, V, (N,), generator=gen, device=DEV)
    y = torch.where(torch.rand(N, generator=gen, device=DEV) < share, y, -100)
    leaves = [t.requires_grad_() for t in (h, w, b)]
    loss = linear_cross_entropy(h, w, b, y, reduction="sum")
    grads = torch.autograd.grad(loss, leaves)
    want, bounds = reference(h, w, b, y, torch.ones(N, device=DEV))
    # (the losses' sum is in 64 bits and rounded once)
    assert abs(loss.item() - want[0].sum().item()) <= bounds[0].sum().item() + 2.0 ** -24 * abs(want[0].sum().item())
    off = [worst(got, want[i], bounds[i]) for i, got in enumerate(grads, 1)]
    assert max(off) <= 1, off
    assert (grads[0][y < 0] == 0).all()
