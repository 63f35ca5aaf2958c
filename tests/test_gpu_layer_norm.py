"""Layer norm of rows (csrc/layer_norm_rows.hip), forward and backward, against 64 bits."""
import pytest
import torch

import lookupffn_amd
from lookupffn_amd import layer_norm

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


def _reference(x, w, b, eps, g):
    """-> ((y, grad x, grad w, grad b), their bounds).  A sum over a row goes through at most D additions: 32 of a thread (or one in 256 columns of a wide row), 6 between lanes, 4
    between wavefronts; so a mean is off by D 2^-24 of the numbers' sizes, and what follows by what it takes from there, to first order, half as much again for the rest.  Sums over the
    rows: those of a workgroup, four within it, 32 and 16 of the workgroups'.  A rounding to the type at the end."""
    e, u = 2.0 ** -24, torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal * 2.0 ** -8
    x, g = (t.detach().double().cpu().reshape(-1, x.shape[-1]) for t in (x, g))
    n = x.shape[1]
    D, R = 48 + n / 256, len(x) / 512 + 64
    uw = u if w is None and b is None else torch.finfo((b if w is None else w).dtype).eps / 2
    w = torch.ones(n, dtype=torch.float64) if w is None else w.detach().double().cpu()
    b = torch.zeros(n, dtype=torch.float64) if b is None else b.detach().double().cpu()
    mean = lambda t: t.mean(1, keepdim=True)  # noqa: E731
    d = x - mean(x)
    var = mean(d * d)
    r = (var + eps) ** -0.5
    z = d * r
    y, h = z * w + b, g * w
    s1, s2 = mean(h), mean(h * z)
    gx = r * (h - s1 - z * s2)
    of_mean = D * e * mean(x.abs())
    of_r = 0.5 * (2 * mean(d.abs()) * of_mean + of_mean ** 2 + (D + 3) * e * var) / (var + eps) + 4 * e          # relative
    of_z = r * (of_mean + e * d.abs()) + z.abs() * (of_r + 2 * e)
    of_y = w.abs() * of_z + 2 * e * ((z * w).abs() + b.abs())
    of_s1, of_s2 = D * e * mean(h.abs()), mean(h.abs() * of_z) + (D + 2) * e * mean((h * z).abs())
    of_gx = gx.abs() * of_r + r * (of_s1 + of_z * s2.abs() + z.abs() * of_s2 + 4 * e * (h.abs() + s1.abs() + (z * s2).abs()))
    of_gw, of_gb = (g.abs() * of_z).sum(0) + R * e * (g * z).abs().sum(0), R * e * g.abs().sum(0)
    gw, gb = (g * z).sum(0), g.sum(0)
    return (y, gx, gw, gb), (u * y.abs() + 1.5 * of_y + tiny, u * gx.abs() + 1.5 * of_gx + tiny, uw * gw.abs() + 1.5 * of_gw + tiny, uw * gb.abs() + 1.5 * of_gb + tiny)


def _close(got, want, bound):
    assert got.isfinite().all()
    worst = ((got.double().cpu().reshape(want.shape) - want).abs() / bound).max().item() if got.numel() else 0.0
    assert worst <= 1, worst


def _check(x, w, b, g, eps=1e-5):
    leaves = [t.requires_grad_() for t in (x, w, b) if t is not None]
    out = layer_norm(x, w, b, eps=eps)
    grads = torch.autograd.grad(out, leaves, g)
    assert out.shape == x.shape and out.dtype == x.dtype and all(a.dtype == t.dtype and a.shape == t.shape for a, t in zip(grads, leaves))
    want, bounds = _reference(x, w, b, eps, g)
    rest = [i for i, t in ((1, x), (2, w), (3, b)) if t is not None]
    for got, i in zip((out.detach(), *grads), (0, *rest)):
        _close(got, want[i], bounds[i])
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, eps=eps), out)
    again = torch.autograd.grad(layer_norm(x, w, b, eps=eps), leaves, g)
    assert all(torch.equal(p, q) for p, q in zip(again, grads))


# rows, columns: a lane, a sixteenth of a wavefront, one, several vectors of one, a workgroup, rows that are read again; odd widths of each; more rows than a backward's workgroups
SIZES = [(1, 1), (3, 2), (5, 7), (1, 8), (33, 16), (1, 64), (70, 65), (2100, 24), (17, 128), (19, 129), (300, 389), (4, 512), (601, 768), (5, 701), (2, 1000), (3, 1024), (530, 1026), (9, 2048),
         (7, 2049), (2, 4096), (3, 5003), (1, 8192), (2, 8200), (600, 9000), (5, 20001), (70, 70000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,columns", SIZES)
def test_against_64_bits(rows, columns, dtype):
    x = (0.5 + _randn(rows, 1) + _randn(rows, columns)).to(dtype)
    of = torch.float32 if rows % 2 else dtype
    w, b = (1 + 0.2 * _randn(columns, seed=1)).to(of), (0.3 * _randn(columns, seed=2)).to(of)
    # (of one or two columns the squares' mean may be nothing but the mean's rounding: with a large eps they do not matter)
    _check(x, w, b, _randn(rows, columns, dtype=dtype, seed=3), 1.0 if columns < 8 else 1e-5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_weights(dtype):
    for w, b in ((None, None), (1.5, None), (None, 0.5)):
        w, b = (None if t is None else t + 0.1 * _randn(130, seed=4) for t in (w, b))
        _check(_randn(37, 130, dtype=dtype), w, b, _randn(37, 130, dtype=dtype, seed=1))


def test_shapes_and_layouts():
    x = _randn(4, 6, 200, dtype=torch.float16)
    w, b = 1 + 0.1 * _randn(300, seed=1), 0.1 * _randn(300, seed=2)
    g = _randn(4, 6, 200, dtype=torch.float16, seed=3)
    for view, gv in ((x, g), (x[:, :, 8:136], g[:, :, 8:136]), (x[:, :, 3:100], g[:, :, 3:100]), (x[:, ::2], g[:, ::2]), (x.transpose(0, 1), g.transpose(0, 1)), (x[0, 0], g[0, 0]),
                     (x[..., ::2], g[..., ::2]), (x[:1].expand(5, 6, 200), g[:1].expand(5, 6, 200)), (x.transpose(0, 2), g.transpose(0, 2)), (x, g[:1, :1, :1].expand(4, 6, 200))):
        n = view.shape[-1]
        _check(view.detach(), w[:n].clone(), b[n:2 * n:1][:n].clone() if 2 * n <= 300 else None, gv, 1e-3)
        _check(view.detach(), w[1:n + 1].detach().half(), None, gv, 1e-3)            # a weight whose address 16 bytes do not divide
    for shape in ((0, 40), (3, 0, 40)):                                             # no rows: zeros for the weights
        x, w, b = torch.empty(shape, device=DEV).requires_grad_(), torch.ones(40, device=DEV).requires_grad_(), torch.ones(40, device=DEV).requires_grad_()
        grads = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), torch.empty(shape, device=DEV))
        assert grads[0].shape == shape and (grads[1] == 0).all() and (grads[2] == 0).all()


def test_only_what_is_wanted():
    x, w, b, g = _randn(50, 96), 1 + _randn(96, seed=1), _randn(96, seed=2), _randn(50, 96, seed=3)
    every = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(layer_norm(*every), every, g)
    for i in range(3):
        args = [t.clone().requires_grad_(n == i) for n, t in enumerate((x, w, b))]
        assert torch.equal(torch.autograd.grad(layer_norm(*args), args[i], g)[0], want[i])


def test_far_numbers():
    """Means far from zero, large and small numbers, infinities in one row of several."""
    g = _randn(6, 1024, seed=1)
    _check(100 + _randn(6, 1024), None, None, g)
    _check(1e15 * _randn(6, 1024), None, None, g)
    _check(1e-3 * _randn(6, 1024), None, None, g, 1e-8)
    x = _randn(6, 1024)
    x[2, 5], x[4, 7] = float("inf"), float("nan")
    out = layer_norm(x)
    assert out[2].isnan().any() and out[4].isnan().all() and torch.equal(out[[0, 1, 3, 5]], layer_norm(x[[0, 1, 3, 5]]))
