"""Softmax cross entropy of a projection to a vocabulary (csrc/linear_cross_entropy.hip), forward and backward, against 64 bits."""
import math

import pytest
import torch

import lookupffn_amd
from lookupffn_amd import linear_cross_entropy

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


def _reference(h, w, b, y, ignore, reduction, g):
    """-> ((loss, grad h, grad w, grad b), their bounds), e = 2^-24.
    A logit: K products (exact of 16 bits; of two terms off by 2^-21 of their sizes, and by 2^-37 of the largest number), K / 8 + 8 roundings of sums that are at most all the
    products' sizes.  Levels and exponentials: a softmax moves by twice the logits' errors, and each exponential by its argument's rounding and 2^-21.  d: rounded to the type, of half
    precision (and in the second term) also by 2^-38 of the largest gradient of a token.  Gradients: those errors times the other operand, and the roundings of their sums.  A rounding to
    the type at the end."""
    e, u, half = 2.0 ** -24, torch.finfo(h.dtype).eps / 2, h.dtype == torch.float16
    two = h.dtype == torch.float32
    tiny = torch.finfo(h.dtype).smallest_normal * 2.0 ** -8
    bu = torch.finfo(h.dtype if b is None else b.dtype).eps / 2
    h, w, g, y = h.detach().double().cpu(), w.detach().double().cpu(), g.double().cpu(), y.long().cpu()
    b = torch.zeros(len(w), dtype=torch.float64) if b is None else b.detach().double().cpu()
    (N, K), V = h.shape, len(w)
    live = (y != ignore) & (y >= 0) & (y < V)
    h = torch.where(live[:, None], h, 0.0)
    at = torch.where(live, y, 0)[:, None]
    logits = h @ w.T + b
    sizes = h.abs() @ w.abs().T
    of_logit = (K / 8 + 8) * e * sizes + 2 * e * (sizes + b.abs())
    if two:
        of_logit += 2.0 ** -21 * sizes + 2.0 ** -37 * (h.abs().amax() * w.abs().sum(1) + w.abs().amax() * h.abs().sum(1, keepdim=True))
    of_logit = of_logit.amax(1, keepdim=True)
    lse = torch.logsumexp(logits, 1, keepdim=True)
    span = (lse - logits).amax(1, keepdim=True) + lse.abs()
    of_p = 2 * of_logit + span * 4 * e + 2.0 ** -20                       # relative
    loss = torch.where(live, (lse - logits.gather(1, at))[:, 0], 0.0)
    of_loss = torch.where(live, (2 * of_logit + span * 4 * e + 2.0 ** -20)[:, 0], 0.0) + 1e-30
    count = max(1, int(live.sum()))
    coefficient = torch.where(live, g.expand(N) / (count if reduction == "mean" else 1), 0.0)[:, None]
    p = (logits - lse).exp()
    d = p.clone()
    d[torch.arange(N), at[:, 0]] -= 1
    d, of_d = d * coefficient, (p * of_p + e) * coefficient.abs()
    of_d += (2.0 ** -21 if two else u) * d.abs() + (2.0 ** -37 * coefficient.abs().max() if half or two else 0.0) * live[:, None]
    gh, gw, gb = d @ w, d.T @ h, d.sum(0)
    of_gh = of_d @ w.abs() + (V / 8 + 80) * e * (d.abs() @ w.abs())
    of_gw = of_d.T @ h.abs() + (N / 8 + 80) * e * (d.abs().T @ h.abs())
    of_gb = of_d.sum(0) + (N / 2 + 80) * e * d.abs().sum(0)
    if two:
        of_gh += (2.0 ** -21 * d.abs() @ w.abs()) + 2.0 ** -37 * w.abs().amax() * d.abs().sum(1, keepdim=True)
        of_gw += (2.0 ** -21 * d.abs().T @ h.abs()) + 2.0 ** -37 * h.abs().amax() * d.abs().sum(0)[:, None]
    if reduction != "none":
        of_loss = of_loss.sum() / (count if reduction == "mean" else 1) + e * loss.sum().abs()
        loss = loss.sum() / (count if reduction == "mean" else 1)
    return ((loss, gh, gw, gb), (of_loss + e * loss.abs(), u * gh.abs() + of_gh + tiny, u * gw.abs() + of_gw + tiny, bu * gb.abs() + of_gb + tiny))


def _close(got, want, bound):
    assert got.shape == want.shape and got.isfinite().all()
    worst = ((got.double().cpu() - want).abs() / bound).max().item() if got.numel() else 0.0
    assert worst <= 1, worst


def _check(h, w, b, y, reduction="mean", ignore=-100, g=None):
    leaves = [t.requires_grad_() for t in (h, w, b) if t is not None]
    call = lambda: linear_cross_entropy(h, w, b, y, ignore_index=ignore, reduction=reduction)  # noqa: E731
    loss = call()
    assert loss.dtype == torch.float32 and loss.shape == (y.shape if reduction == "none" else ())
    g = torch.ones_like(loss) if g is None else g
    grads = torch.autograd.grad(loss, leaves, g)
    assert all(a.dtype == t.dtype and a.shape == t.shape for a, t in zip(grads, leaves))
    if y.numel() == 0:
        assert (loss == 0).all() and all((t == 0).all() for t in grads)
        return loss, grads
    flat = g.reshape(-1) if reduction == "none" else g
    want, bounds = _reference(h.reshape(-1, h.shape[-1]), w, b, y.reshape(-1), ignore, reduction, flat)
    _close(loss.detach().reshape(want[0].shape), want[0], bounds[0])
    for got, i in zip(grads, (1, 2, 3)):
        _close(got.reshape(want[i].shape), want[i], bounds[i])
    with torch.no_grad():
        assert torch.equal(call(), loss)
    again = torch.autograd.grad(call(), leaves, g)
    assert all(torch.equal(p, q) for p, q in zip(again, grads))
    return loss, grads


# tokens, vocabulary, columns, share of the tokens that have a label: one of each; sizes below, at and beyond a tile's; tokens that are counted in a launch of their own; many tiles; tokens
# whose sums are cut; few labelled ones; few with kept logits, in pieces of the vocabulary
SIZES = [(1, 1, 8, 1.0), (1, 300, 64, 1.0), (5, 7, 16, 0.8), (64, 1000, 72, 1.0), (255, 255, 40, 1.0), (256, 256, 64, 1.0), (257, 513, 136, 0.5), (300, 777, 520, 0.3), (33, 5003, 264, 1.0),
         (4200, 600, 64, 0.1), (700, 2100, 776, 0.9), (130, 4096, 1032, 1.0), (40, 70001, 24, 0.9), (64, 300, 1208, 1.0), (64, 300, 1216, 1.0), (20, 300, 2432, 1.0), (32, 40, 2424, 0.9),
         (64, 300, 608, 1.0), (64, 300, 616, 1.0), (32, 40, 1216, 0.9), (20, 9000, 1224, 1.0), (1100, 300, 40, 1.0), (5000, 300, 72, 1.0), (9001, 40, 264, 0.9),
         (4097, 1100, 24, 0.6), (300, 777, 72, 0.1), (129, 1500, 520, 0.45), (90, 1030, 1400, 0.5), (4, 2200000, 8, 1.0)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,K,share", SIZES)
def test_against_64_bits(N, V, K, share, dtype):
    gen = torch.Generator(device=DEV).manual_seed(N)
    h, w = _randn(N, K, dtype=dtype), (2 / math.sqrt(K) * _randn(V, K, seed=1)).to(dtype)
    b = None if N == 33 else (0.5 * _randn(V, seed=2)).to(torch.float32 if N % 2 else dtype)
    y = torch.randint(0, V, (N,), generator=gen, device=DEV)
    y = torch.where(torch.rand(N, generator=gen, device=DEV) < share, y, -100)
    scale = 1024.0 if dtype == torch.float16 else 1.0
    _check(h, w, b, y, "mean", g=torch.tensor(scale, device=DEV))
    _check(h, w, b, y.int(), "sum", g=torch.tensor(-0.5, device=DEV))
    _check(h, w, b, y, "none", g=(_randn(N, seed=3) * 3).float())


@pytest.mark.parametrize("dtype", DTYPES)
def test_pieces_of_the_vocabulary(dtype):
    """So many tokens that the logits' gradients are formed in several pieces: with every token labelled, and with few, which need fewer pieces than launches."""
    N, V, K = (131072, 5000, 8) if dtype != torch.float32 else (65536, 5000, 8)
    h, w = _randn(N, K, dtype=dtype), _randn(V, K, dtype=dtype, seed=1)
    b = 0.5 * _randn(V, seed=2)
    y = torch.randint(0, V, (N,), device=DEV)
    few = torch.where(torch.arange(N, device=DEV) % 50 == 0, y, -100)
    at = few >= 0
    leaves = [t.requires_grad_() for t in (h, w, b)]
    got = torch.autograd.grad(linear_cross_entropy(h, w, b, few, reduction="sum"), leaves)
    rows = h.detach()[at].requires_grad_()
    want = torch.autograd.grad(linear_cross_entropy(rows, w, b, few[at], reduction="sum"), (rows, w, b))
    # the same tokens by themselves: shares of sums may be others, so compared with bounds
    ref, bounds = _reference(h.detach()[at], w, b, few[at], -100, "sum", torch.tensor(1.0))
    _close(got[0][at], ref[1], bounds[1])
    _close(got[1], ref[2], bounds[2])
    _close(got[2], ref[3], bounds[3])
    assert (got[0][~at] == 0).all() and want[0].shape == rows.shape
    # all tokens: those of a part of them in any place have their gradients, and the weights' are the parts' sums
    every = torch.autograd.grad(linear_cross_entropy(h, w, b, y, reduction="sum"), leaves)
    total_w, total_b, sizes = 0.0, 0.0, 0.0
    for i in range(0, N, 4096):
        part = h.detach()[i:i + 4096].requires_grad_()
        one = torch.autograd.grad(linear_cross_entropy(part, w, b, y[i:i + 4096], reduction="sum"), (part, w, b))
        # (both are roundings of sums of the same d: within two roundings, and the roundings of sums of 5000 numbers of W)
        u = torch.finfo(dtype).eps
        assert ((every[0][i:i + 4096].double() - one[0].double()).abs() <= u * one[0].double().abs() + 2000 * 2.0 ** -24 * 2 * w.detach().double().abs().amax()).all()
        total_w, total_b, sizes = total_w + one[1].double(), total_b + one[2].double(), sizes + one[1].double().abs()
    # every part's gradient is a rounding, so is the whole's; sums of N numbers of size 1 and K = 8, some N / 8 roundings of 2^-24 of at most N / V 10 + 1 labels' and sums of p
    slack = 2 * torch.finfo(dtype).eps * (sizes + every[1].double().abs()) + 2.0 ** -24 * (N / 8) * 4 * (4 * N / V + 10)
    assert ((every[1].double() - total_w).abs() <= slack).all()
    # an entry's bias: a lane adds N / 2 numbers d in pairs, N / 4 roundings of sums that are at most the sum of their sizes, which is the labels' of the entry twice and the gradient
    # itself (d is p, or p - 1 at a label); a part's have a sixteenth as many, so both together less than twice that; and the rounding of each to fp32
    most = every[2].double().abs() + 2 * torch.bincount(y, minlength=V)
    assert ((every[2].double() - total_b).abs() <= 2 * (N / 4) * 2.0 ** -24 * most + 2.0 ** -20 * every[2].double().abs()).all()


def test_labels():
    N, V, K = 200, 300, 64
    h, w, b = _randn(N, K), 0.3 * _randn(V, K, seed=1), _randn(V, seed=2)
    y = torch.randint(0, V, (N,), device=DEV)
    for ignore in (-100, 0, 7, V + 5, -1 << 40, 1 << 40):
        t = y.clone()
        t[::3] = ignore
        t[1::10], t[2::10] = -1, V              # no numbers of the vocabulary: as if ignored
        t[4::10] = -1 << 33
        loss, _ = _check(h, w, b, t, "none", ignore)
        out = (t == ignore) | (t < 0) | (t >= V)
        assert (loss[out] == 0).all() and (loss[~out] > 0).all()
    for t in (torch.full_like(y, -100), torch.full_like(y, V - 1), torch.zeros_like(y)):
        for reduction in ("mean", "sum", "none"):
            loss, grads = _check(h, w, b, t, reduction)
            if t[0] == -100:
                assert (loss == 0).all() and all((g == 0).all() for g in grads)


def test_ignored_rows_may_hold_anything():
    N, V, K = 300, 400, 72
    for dtype in DTYPES:
        h, w, b = _randn(N, K, dtype=dtype), (0.3 * _randn(V, K, seed=1)).to(dtype), _randn(V, seed=2)
        y = torch.randint(0, V, (N,), device=DEV)
        y[::2] = -100
        plain = _check(h.clone(), w.clone(), b.clone(), y)
        h = h.detach().clone()
        h[::4], h[2::4] = float("nan"), float("inf")
        wild = linear_cross_entropy(h.requires_grad_(), w.requires_grad_(), b.requires_grad_(), y)
        grads = torch.autograd.grad(wild, (h, w, b))
        assert torch.equal(wild, plain[0]) and all(torch.equal(p, q) for p, q in zip(grads, plain[1]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,K", [(7, 64), (60, 16), (130, 64)])
def test_no_token_has_a_label(N, K, dtype):
    h, w, b = (_randn(N, K, dtype=dtype).requires_grad_(), _randn(200, K, dtype=dtype, seed=1).requires_grad_(), _randn(200, seed=2).requires_grad_())
    y = torch.full((N,), -100, device=DEV)
    for reduction in ("mean", "sum", "none"):
        loss = linear_cross_entropy(h, w, b, y, reduction=reduction)
        assert (loss == 0).all() and all((t == 0).all() for t in torch.autograd.grad(loss, (h, w, b), torch.ones_like(loss)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [40, 300])
def test_an_infinite_token_leaves_the_others(N, dtype):
    """A token's infinite numbers, or an infinite gradient of its loss, reach that token's loss and gradient, and no other's."""
    V, K = 500, 64
    h, w, b = _randn(N, K, dtype=dtype), _randn(V, K, dtype=dtype, seed=1) / 4, _randn(V, seed=2)
    y, g = torch.randint(0, V, (N,), device=DEV), _randn(N, seed=3)
    h[3, 5], h[N - 2, 1] = float("inf"), float("nan")
    g[7] = float("inf")
    leaf = h.clone().requires_grad_()
    loss = linear_cross_entropy(leaf, w, b, y, reduction="none")
    grad, = torch.autograd.grad(loss, leaf, g)
    lost = [3, N - 2]
    assert not loss[lost].isfinite().any() and not grad[lost + [7]].isfinite().all(1).any()
    others = torch.tensor([n not in (*lost, 7) for n in range(N)], device=DEV)
    want, bounds = _reference(h[others], w, b, y[others], -100, "none", g[others])
    _close(loss.detach()[others], want[0], bounds[0])
    _close(grad[others], want[1], bounds[1])


def test_masked_vocabulary():
    """Entries that a bias of the lowest value, or minus infinity, takes out: whole tiles of them, and a token whose label is one."""
    N, V, K = 50, 900, 64
    h, w, y = _randn(N, K), 0.3 * _randn(V, K, seed=1), torch.randint(600, 900, (N,), device=DEV)
    for low in (-math.inf, torch.finfo(torch.float32).min):
        b = _randn(V, seed=2)
        b[:600] = low
        leaves = [t.detach().clone().requires_grad_() for t in (h, w, b)]
        loss = linear_cross_entropy(*leaves, y, reduction="none")
        grads = torch.autograd.grad(loss.sum(), leaves)
        fewer = [t.detach().clone().requires_grad_() for t in (h, w[600:], b[600:])]
        ref, bounds = _reference(*fewer, y - 600, -100, "none", torch.ones(N))
        _close(loss.detach(), ref[0], bounds[0])
        _close(grads[0], ref[1], bounds[1])
        _close(grads[1][600:], ref[2], bounds[2])
        _close(grads[2][600:], ref[3], bounds[3])
        assert (grads[1][:600] == 0).all() and (grads[2][:600] == 0).all()
        away = linear_cross_entropy(h, w, b, torch.zeros_like(y), reduction="none")
        assert (away == math.inf).all() if low == -math.inf else (away > 1e38).all()


def test_large_logits():
    """Logits of some hundreds: a softmax of one entry; gradients stay finite."""
    N, V, K = 90, 700, 128
    for dtype in DTYPES:
        h, w = (10 * _randn(N, K)).to(dtype), (3 * _randn(V, K, seed=1)).to(dtype)
        best = (h.double() @ w.double().T).argmax(1)
        _check(h, w, None, best, "sum")
        _check(h, w, None, torch.randint(0, V, (N,), device=DEV), "sum")


def test_numbers_of_many_sizes():
    """fp32: rows of very different sizes, large and small ones, zeros."""
    N, V, K = 100, 500, 96
    h, w = _randn(N, K), 0.1 * _randn(V, K, seed=1)
    h = h * 2.0 ** (torch.arange(N, device=DEV) % 12 - 8)[:, None]
    w = w * 2.0 ** (torch.arange(V, device=DEV) % 9 - 6)[:, None]
    h[5], w[7] = 0, 0
    y = torch.randint(0, V, (N,), device=DEV)
    _check(h, w, None, y, "sum")
    _check(h * 1e-15, w * 1e15, None, y, "sum")
    _check(torch.zeros_like(h), w, None, y, "sum")
    _check(h, torch.zeros_like(w), None, y, "sum")


def test_shapes_and_layouts():
    B, L, V, K = 3, 40, 300, 104
    h, w, b = _randn(B, L, 2 * K, dtype=torch.float16), (0.2 * _randn(V, 2 * K, seed=1)).half(), _randn(2 * V, seed=2).half()
    y = torch.randint(0, V, (B, L), device=DEV)
    for hv, wv, bv, yv in ((h[..., :K], w[:, :K], b[:V], y), (h[..., K:], w[:, K:], b[::2], y), (h[..., 3:K + 3], w[:, 1:K + 1], b[1:V + 1], y), (h[:, ::2, :K], w[:, ::2], None, y[:, ::2]),
                           (h.transpose(0, 1)[..., :K], w[:, :K], None, y.t()), (h[:1, :1, :K].expand(B, L, K), w[:1, :K].expand(V, K), None, y), (h[0, 0, :K], w[:, :K], None, y[0, 0]),
                           (h[:, :0, :K], w[:, :K], b[:V], y[:, :0])):
        for reduction in ("mean", "none"):
            _check(hv.detach(), wv.detach(), None if bv is None else bv.detach(), yv, reduction)


def test_only_what_is_wanted():
    N, V, K = 60, 500, 64
    for dtype in DTYPES:
        parts = [_randn(N, K, dtype=dtype), (0.2 * _randn(V, K, seed=1)).to(dtype), _randn(V, seed=2)]
        y = torch.randint(0, V, (N,), device=DEV)
        every = [t.clone().requires_grad_() for t in parts]
        want = torch.autograd.grad(linear_cross_entropy(*every, y), every)
        for i in range(3):
            args = [t.clone().requires_grad_(n == i) for n, t in enumerate(parts)]
            assert torch.equal(torch.autograd.grad(linear_cross_entropy(*args, y), args[i])[0], want[i])


def test_the_gradient_is_the_slope():
    N, V, K = 40, 120, 16
    h, w, b = _randn(N, K), _randn(V, K, seed=1) / 2, _randn(V, seed=2) / 2
    y = torch.randint(0, V, (N,), device=DEV)
    leaves = [t.requires_grad_() for t in (h, w, b)]
    grads = torch.autograd.grad(linear_cross_entropy(*leaves, y, reduction="sum"), leaves)
    for n, (t, grad) in enumerate(zip(leaves, grads)):
        way = _randn(*t.shape, seed=10 + n)
        step = 2.0 ** -6 / way.norm().item()
        at = lambda s: linear_cross_entropy(*[(q.detach() + s * step * way if k == n else q.detach()) for k, q in enumerate(leaves)], y, reduction="none").double().sum().item()  # noqa: E731
        slope = (at(1) - at(-1)) / 2
        # losses of size 5 are off by 2^-21 each, 40 of them; the third derivative of a sum of log sums over a way of length 2^-6 is below 40 * 2^-18 * 5
        assert abs(slope - (grad * way).double().sum().item() * step) <= 40 * 5 * 2.0 ** -21 + 40 * 5 * 2.0 ** -18 / 6


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,K", [(40, 300, 256), (300, 700, 64), (5000, 300, 64)])
def test_replays_with_other_labels(N, V, K, dtype, either_path):
    """How many tokens have a label is the replay's, not the capture's: none, few, all; each as the eager call has it, with the program's own work between."""
    if lookupffn_amd._lib.host_module() is None:
        pytest.skip("without the host library no forward with gradients is captured")
    h, w, b = (_randn(N, K, dtype=dtype).requires_grad_(), (_randn(V, K, seed=1) / 8).to(dtype).requires_grad_(), _randn(V, seed=2).requires_grad_())
    full = torch.randint(0, V, (N,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(3))
    some = [torch.where(torch.rand(N, device=DEV, generator=torch.Generator(device=DEV).manual_seed(4)) < share, full, -100) for share in (1.0, 0.1, 0.0, 0.5, 1.0)]

    def step(y):
        loss = linear_cross_entropy(h, w, b, y)
        return loss.detach(), *torch.autograd.grad(loss, (h, w, b))

    want = [step(y) for y in some]
    y = full.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(y)
    for labels, expected in zip(some, want):
        y.copy_(labels)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, expected))
        torch.randn(1 << 20, device=DEV).sum().item()
