"""linear_cross_entropy of logits so large that every token's softmax is one entry, against 64 bits: losses, and what the gradients are made of."""
import pytest
import torch

import lookupffn_amd
from lookupffn_amd import linear_cross_entropy

from _loss_reference import reference, worst

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# few tokens whose logits are kept; tiles of 64 and of 256; several tiles of columns
SIZES = [(40, 300, 64), (60, 300, 16), (70, 300, 72), (300, 777, 136), (130, 520, 264), (5000, 300, 64)]


@pytest.fixture(autouse=True, params=["host", "python"])
def either_path(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(lookupffn_amd._lib, "loaded_host", False)
    else:
        assert lookupffn_amd._lib.host()


def _randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed + sum(shape)), device=DEV)


def _labels(N, V, seed=5):
    return torch.randint(0, V, (N,), generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


@pytest.mark.parametrize("size", [1e3, 1e4, 6e4])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,K", SIZES)
def test_losses(N, V, K, dtype, size):
    """Logits from some millions to some tens of billions, below and above 2^30."""
    h, w, b = (size * _randn(N, K).clamp(-1, 1)).to(dtype), (size * _randn(V, K, seed=1).clamp(-1, 1)).to(dtype), _randn(V, seed=2)
    for y in (_labels(N, V), (h.double() @ w.double().T + b).argmax(1)):
        want, bounds = reference(h, w, b, y, torch.ones(N, device=DEV))
        assert worst(linear_cross_entropy(h, w, b, y, reduction="none"), want[0], bounds[0]) <= 1


@pytest.mark.parametrize("sign", [1, -1])
def test_one_token_among_others(sign):
    """A token's logits of any size are that token's: the others' losses are as they were, bit for bit, its own one finite."""
    N, V, K = 300, 777, 136
    h, w, b, y = _randn(N, K), 0.25 * _randn(V, K, seed=1), _randn(V, seed=2), _labels(N, V)
    before = linear_cross_entropy(h, w, b, y, reduction="none")
    for size in (1e6, 2.0 ** 28, 2.0 ** 30, 1e10, 1e20, 1e37):
        t = h.clone()
        t[5] *= sign * size
        losses = linear_cross_entropy(t, w, b, y, reduction="none")
        want, bounds = reference(t[5:6], w, b, y[5:6], torch.ones(1, device=DEV))
        assert worst(losses[5:6], want[0], bounds[0]) <= 1
        losses[5] = before[5]
        assert torch.equal(losses, before)


@pytest.mark.parametrize("dtype", DTYPES)
def test_logits_on_both_sides_of_a_level_s_units(dtype):
    """Every entry's logit around 2^30 by themselves: the largest is found, wherever the others are."""
    V, K = 600, 8
    w = torch.zeros(V, K, device=DEV)
    w[:, 0] = torch.linspace(0.5, 2.0, V, device=DEV)
    for sign in (1, -1):
        h = torch.zeros(70, K, device=DEV)
        h[:, 0] = sign * 2.0 ** 15
        # (the last one, 2^16, is no finite number of half: its largest, 65504)
        hd, wd = h.to(dtype), (w * 2.0 ** 15).clamp(max=torch.finfo(dtype).max).to(dtype)
        y = _labels(70, V)
        want, bounds = reference(hd, wd, None, y, torch.ones(70, device=DEV))
        assert worst(linear_cross_entropy(hd, wd, None, y, reduction="none"), want[0], bounds[0]) <= 1


@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("N,V,K", [*SIZES, (60, 300, 96), (64, 2000, 120)])
def test_gradients(N, V, K, dtype):
    """Both directions see a token's one entry at the same height, whichever kernels form their logits."""
    h, w, y = (1e4 * _randn(N, K)).to(dtype), (1e4 * _randn(V, K, seed=1)).to(dtype), _labels(N, V)
    g = torch.full((N,), 2.0 ** -6, device=DEV)
    leaves = h.requires_grad_(), w.requires_grad_()
    grads = torch.autograd.grad(linear_cross_entropy(h, w, None, y, reduction="none"), leaves, g)
    want, bounds = reference(h, w, None, y, g)
    assert max(worst(got, want[i], bounds[i]) for i, got in enumerate(grads, 1)) <= 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [7, 300])
def test_no_label_and_a_gradient_that_is_no_number(N, dtype):
    """Tokens without a label have no part in anything, whatever the loss's gradient is."""
    h, w, b = ((t / 8).to(dtype).requires_grad_() for t in (_randn(N, 64), _randn(200, 64, seed=1), _randn(200, seed=2)))
    y = torch.full((N,), -100, device=DEV)
    for g in (float("inf"), float("nan")):
        for reduction in ("mean", "sum", "none"):
            loss = linear_cross_entropy(h, w, b, y, reduction=reduction)
            assert all((t == 0).all() for t in torch.autograd.grad(loss, (h, w, b), torch.full_like(loss, g)))
