"""linear_cross_entropy where numbers are far apart: a token, an entry or a token's gradient of another size than the rest, logits that are large everywhere.  What one of them is must not
reach the others' gradients.  Against 64 bits."""
import math

import pytest
import torch

import lookupffn_amd
from lookupffn_amd import linear_cross_entropy

from _loss_reference import reference, worst

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(autouse=True, params=["host", "python"])
def either_path(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(lookupffn_amd._lib, "loaded_host", False)
    else:
        assert lookupffn_amd._lib.host()


def _randn(*shape, dtype=torch.float32, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed + sum(shape)), device=DEV).to(dtype)


def _labels(N, V, seed=5):
    return torch.randint(0, V, (N,), generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


def _check(h, w, b, y, g=None):
    """Losses of each token and, with `g` by token or a mean over the labelled ones, the gradients; the same bits twice."""
    leaves = [t.requires_grad_() for t in (h, w, b) if t is not None]
    live = (y >= 0) & (y < len(w))
    with torch.no_grad():
        losses = linear_cross_entropy(h, w, b, y, reduction="none")

    def step():
        loss = linear_cross_entropy(h, w, b, y, reduction="mean" if g is None else "none")
        return torch.autograd.grad(loss, leaves, g)

    grads = step()
    want, bounds = reference(h, w, b, y, 1 / live.sum().clamp(min=1).expand(len(y)) if g is None else g)
    assert worst(losses, want[0], bounds[0]) <= 1
    off = [worst(got, want[i], bounds[i]) for i, got in enumerate(grads, 1)]
    assert max(off) <= 1, off
    assert (grads[0][~live] == 0).all()
    assert all(torch.equal(p, q) for p, q in zip(grads, step()))


# few tokens whose logits are kept; few, but more than columns; tiles of 64 and of 256; sums over the tokens that are cut; several tiles of columns
SIZES = [(40, 300, 64), (60, 300, 16), (70, 300, 72), (300, 777, 136), (130, 520, 264), (5000, 300, 64)]


@pytest.mark.parametrize("factor", [2.0 ** 10, 2.0 ** 15, 1e6, 1e9, 1e12, 1e20])
@pytest.mark.parametrize("N,V,K", SIZES)
def test_a_large_token(N, V, K, factor):
    h, w, b, y = _randn(N, K), 0.25 * _randn(V, K, seed=1), 0.5 * _randn(V, seed=2), _labels(N, V)
    h[5] *= factor
    h[N - 3] *= -factor
    if N >= 70:
        y[::3] = -100
    _check(h, w, b, y)


@pytest.mark.parametrize("factor", [2.0 ** 15, 1e9, 1e20])
@pytest.mark.parametrize("N,V,K", SIZES)
def test_a_large_entry(N, V, K, factor):
    """An entry of the vocabulary that no token is near, and that is one token's label."""
    h, w, b, y = _randn(N, K), 0.25 * _randn(V, K, seed=1), 0.5 * _randn(V, seed=2), _labels(N, V - 1)
    h[:, 0] = h[:, 0].abs() + 1
    w[V - 1] = w[V - 1] / 64
    w[V - 1, 0] = -1
    w[V - 1] *= factor
    y[7] = V - 1
    _check(h, w, b, y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,K", SIZES)
def test_large_logits_everywhere(N, V, K, dtype):
    """Logits of 10^8 and more: every token's softmax is one entry, and both directions have to see the same one at the same height."""
    h, w, y = (1e4 * _randn(N, K)).to(dtype), (1e4 * _randn(V, K, seed=1)).to(dtype), _labels(N, V)
    _check(h, w, None, y, torch.full((N,), 2.0 ** -6, device=DEV))


@pytest.mark.parametrize("steps", [7, 30, 60])
@pytest.mark.parametrize("N,V,K", SIZES)
def test_tokens_gradients_of_many_sizes(N, V, K, steps):
    """Each token's gradient as exact as if it were alone: sizes from 1 down to 2^-steps, both signs, zeros."""
    h, w, b, y = _randn(N, K), 1.5 / math.sqrt(K) * _randn(V, K, seed=1), 0.5 * _randn(V, seed=2), _labels(N, V)
    n = torch.arange(N, device=DEV)
    g = 2.0 ** -(n * 7 % (steps + 1)).float() * torch.where(n % 2 == 0, 1.0, -1.0)
    g[9] = 0
    _check(h, w, b, y, g)


def test_in_pieces_of_the_vocabulary():
    """So many tokens that the logits' gradients are formed in two pieces."""
    N, V, K = 65536, 5000, 8
    h, w, b, y = _randn(N, K), _randn(V, K, seed=1), 0.5 * _randn(V, seed=2), _labels(N, V)
    h[77] *= 1e9
    _check(h, w, b, y)


def test_only_what_is_wanted():
    N, V, K = 90, 700, 136
    parts = [_randn(N, K), 0.25 * _randn(V, K, seed=1), _randn(V, seed=2)]
    parts[0][5] *= 1e9
    y = _labels(N, V)
    every = [t.clone().requires_grad_() for t in parts]
    want = torch.autograd.grad(linear_cross_entropy(*every, y), every)
    for i in range(3):
        args = [t.clone().requires_grad_(n == i) for n, t in enumerate(parts)]
        assert torch.equal(torch.autograd.grad(linear_cross_entropy(*args, y), args[i])[0], want[i])


@pytest.mark.parametrize("N", [50, 300])
def test_layouts(N):
    """Rows and entries apart in memory, in reverse order of tokens' and columns' strides, one row for all tokens, one dimension more."""
    V, K = 300, 104
    h, w, b, y = _randn(N, 2 * K), 0.25 * _randn(V, 2 * K, seed=1), _randn(2 * V, seed=2), _labels(N, V)
    w[7] *= 1e8
    h[3] *= 1e7
    for hv, wv, bv in ((h[:, :K], w[:, :K], b[:V]), (h[:, K:], w[:, K:], b[::2]), (h[:, ::2], w[:, 1:K + 1], None), (h[:1, :K].expand(N, K), w[:, :K], None)):
        hv, wv = hv.detach(), wv.detach()
        _check(hv, wv, None if bv is None else bv.detach(), y)
    leaves = [t.detach().clone().requires_grad_() for t in (h[:, :K], w[:, :K])]
    flat = torch.autograd.grad(linear_cross_entropy(*leaves, None, y), leaves)
    deep = torch.autograd.grad(linear_cross_entropy(leaves[0].view(2, -1, K), leaves[1], None, y.view(2, -1)), leaves)
    assert all(torch.equal(p, q) for p, q in zip(flat, deep))


@pytest.mark.parametrize("N", [40, 300])
def test_replays_of_other_sizes(N, either_path):
    """Whether numbers are far apart is the replay's, not the capture's."""
    if lookupffn_amd._lib.host_module() is None:
        pytest.skip("without the host library no forward with gradients is captured")
    V, K = 500, 136
    base, w, b, y = _randn(N, K), (0.25 * _randn(V, K, seed=1)).requires_grad_(), _randn(V, seed=2).requires_grad_(), _labels(N, V)
    inputs = []
    for factor in (1.0, 1e9, 1.0, 1e15):
        inputs.append(base.clone())
        inputs[-1][7] *= factor
    h = base.clone().requires_grad_()

    def step(h):
        loss = linear_cross_entropy(h, w, b, y)
        return loss.detach(), *torch.autograd.grad(loss, (h, w, b))

    want = [step(t.clone().requires_grad_()) for t in inputs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(h)
    for t, expected in zip(inputs, want):
        with torch.no_grad():
            h.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, expected))
        torch.randn(1 << 20, device=DEV).sum().item()
