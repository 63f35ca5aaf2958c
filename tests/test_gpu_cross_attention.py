"""Attention to an encoder's states (csrc/cross_attention*.hip), forward and backward, against 64 bits."""
import math

import pytest
import torch

import lookupffn_amd
from lookupffn_amd import cross_attention, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
@pytest.fixture(autouse=True, params=["host", "python"])
def either_path(request, monkeypatch):
    """The calls with the host path in C++ and without."""
    if request.param == "python":
        monkeypatch.setattr(lookupffn_amd._lib, "loaded_host", False)
    else:
        assert lookupffn_amd._lib.host()
    return request.param


DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _randn(*shape, dtype=torch.float32, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + sum(shape))
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def _mask(kind, B, Lk, seed=0):
    if kind is None:
        return None
    g = torch.Generator().manual_seed(seed + Lk)
    keys = torch.arange(Lk)
    if kind == "padded":            # the last sequence has no state at all
        lengths = torch.randint(1, Lk + 1, (B, 1), generator=g)
        lengths[-1] = 0 if B > 1 else lengths[-1]
        mask = keys < lengths
    elif kind == "holes":
        mask = torch.rand(B, Lk, generator=g) < 0.5
    else:                           # "late": the first keys take no part, whole steps of them where there are enough
        mask = keys >= (2 * Lk) // 3
        mask = mask.expand(B, Lk).clone()
    return mask.to(DEV)


def _reference(q, k, v, mask, scale, g=None):
    """In 64 bits; gradients by their formulas.  -> (out, grads, bounds): how far 16-bit or fp32 arithmetic with fp32 sums may be off."""
    u = 0.0 if q.dtype == torch.float32 else torch.finfo(q.dtype).eps / 2      # a rounding to the type
    rest = 2.0 ** -24 if q.dtype == torch.float32 else u
    tiny = 2.0 ** -24 if q.dtype == torch.float16 else 1e-37                   # half's smallest step
    dims = (0, 2, 1, 3)
    group = q.shape[2] // k.shape[2]
    q, k, v = (t.detach().double().cpu().permute(*dims) for t in (q, k, v))
    if mask is not None:            # what takes no part is not looked at
        k, v = (torch.where(mask.cpu()[:, None, :, None], t, 0.0) for t in (k, v))
    k, v = (t.repeat_interleave(group, 1) for t in (k, v))
    s = scale * q @ k.transpose(-1, -2)
    keep = torch.ones_like(s, dtype=torch.bool) if mask is None else mask.cpu()[:, None, None].expand_as(s)
    s = s.masked_fill(~keep, -math.inf)
    m = s.amax(-1, keepdim=True) if s.shape[-1] else s.sum(-1, keepdim=True)
    m = torch.where(m.isfinite(), m, 0.0)
    e = (s - m).exp()
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    out = p @ v
    # A score is off by 2^-20 of the sum of its products' sizes: each product to 2^-22 (fp32), the sum in at most 48 steps of 2^-24, either sign (7 of them).
    # The row's level and the exponentials are off by 2^-23 of the scores' size.
    size = scale * q.abs() @ k.abs().transpose(-1, -2)
    top = size.amax(-1, keepdim=True) if size.shape[-1] else torch.zeros_like(m)
    off = 2.0 ** -20 * top + 2.0 ** -22 * (m.abs() + 10)
    weights = u + 2.0 ** -21 + 2 * off                                          # a weight, relative
    bound = weights * (p @ v.abs()) + rest * out.abs() + tiny
    back = lambda t: t.permute(*dims)  # noqa: E731
    if g is None:
        return back(out), None, (back(bound),)
    g = g.double().cpu().permute(*dims)
    shared = lambda t: back(t.unflatten(1, (-1, group)).sum(2))  # noqa: E731
    dp = g @ v.transpose(-1, -2)
    ds = p * (dp - (g * out).sum(-1, keepdim=True))
    off_ds = weights * ds.abs() + p * (2.0 ** -20 * (g.abs() @ v.abs().transpose(-1, -2)) + (rest + 2.0 ** -20) * (g.abs() * out.abs()).sum(-1, keepdim=True)
                                       + (g.abs() * bound).sum(-1, keepdim=True))
    gq, gk, gv = scale * ds @ k, shared(scale * ds.transpose(-1, -2) @ q), shared(p.transpose(-1, -2) @ g)
    bq = back(scale * off_ds @ k.abs()) + rest * back(gq).abs() + tiny
    bk = shared(scale * off_ds.transpose(-1, -2) @ q.abs()) + rest * gk.abs() + tiny
    bv = shared((weights * p).transpose(-1, -2) @ g.abs()) + rest * gv.abs() + tiny
    return back(out), (back(gq), gk, gv), (back(bound), bq, bk, bv)


def _run(q, k, v, mask, scale=None, g=None):
    if g is None:
        return cross_attention(q, k, v, mask, scale=scale), ()
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = cross_attention(*leaves, mask, scale=scale)
    return out.detach(), torch.autograd.grad(out, leaves, g)


def _close(got, want, bound):
    assert got.shape == want.shape and got.isfinite().all()
    worst = ((got.double().cpu() - want).abs() / bound).max().item() if got.numel() else 0.0
    assert worst <= 1, worst


# Lengths around a step's 64 keys (32 of fp32 heads beyond 64 columns), a workgroup's 128 rows and a wavefront's 32, a block of 64 steps; few rows, whose keys
# are shared out, and few keys, whose rows are; heads of every kernel's columns and between; shared heads
SIZES = [(1, 1, 1, 1, 1, 8), (2, 1, 65, 4, 2, 64), (3, 33, 64, 3, 3, 32), (2, 129, 127, 2, 1, 64), (1, 130, 513, 8, 2, 128), (2, 5, 1000, 2, 2, 128),
         (1, 1, 5000, 8, 1, 64), (4, 64, 77, 4, 4, 40), (1, 300, 70, 2, 2, 96), (2, 1, 4500, 2, 2, 16), (1, 1000, 3, 6, 2, 24), (2, 700, 260, 2, 2, 64),
         (1, 257, 4200, 1, 1, 112)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mask", [None, "padded", "holes", "late"])
@pytest.mark.parametrize("B,Lq,Lk,H,Hk,D", SIZES)
def test_against_64_bits(B, Lq, Lk, H, Hk, D, mask, dtype):
    q, k, v, g = (_randn(B, n, h, D, dtype=dtype, seed=s) for s, (n, h) in enumerate(((Lq, H), (Lk, Hk), (Lk, Hk), (Lq, H))))
    mask_kind, mask = mask, _mask(mask, B, Lk)
    out, grads = _run(q, k, v, mask, None, g)
    want, gradients, bounds = _reference(q, k, v, mask, D ** -0.5, g)
    for a, b, c in zip((out, *grads), (want, *gradients), bounds):
        _close(a, b, c)
    if dtype == torch.float32:      # errors of either sign: far below the sum of their sizes
        # (of one key p = 1 and ds = g v - g o = 0, of a few nearly so: what is left of two equal terms is relative to them, as the bounds above are)
        spread = Lk >= 64 and mask_kind in (None, "holes")
        for i, (a, b) in enumerate(zip((out, *grads), (want, *gradients))):
            if i in (1, 2) and not spread:
                continue
            assert (a.double().cpu() - b).norm() <= 1e-6 * b.norm()
    again, gradients = _run(q, k, v, mask, None, g)
    assert torch.equal(out, again) and all(torch.equal(a, b) for a, b in zip(grads, gradients))
    assert torch.equal(out, _run(q, k, v, mask)[0])
    if mask is not None:
        assert not grads[1][~mask].any() and not grads[2][~mask].any()
        assert not out[~mask.any(1)].any() and not grads[0][~mask.any(1)].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,Lq,Lk,H,Hk,D", [(3, 1, 300, 4, 4, 64), (3, 70, 200, 4, 2, 64), (3, 140, 90, 2, 2, 128)])
def test_what_takes_no_part_is_not_looked_at(B, Lq, Lk, H, Hk, D, dtype):
    """Infinities, NaN and the type's lowest value in masked keys and values: the same bits as with zeros there, forward and backward."""
    q, k, v, g = (_randn(B, n, h, D, dtype=dtype, seed=s) for s, (n, h) in enumerate(((Lq, H), (Lk, Hk), (Lk, Hk), (Lq, H))))
    mask = torch.arange(Lk, device=DEV) < torch.tensor([[Lk // 2], [0], [Lk - 1]], device=DEV)
    mask[0, 3], mask[2, :66] = False, False
    clean = [torch.where(mask[:, :, None, None], t, 0.0) for t in (k, v)]
    want, gradients = _run(q, *clean, mask, None, g)
    for other in (math.nan, math.inf, -math.inf, torch.finfo(dtype).min):
        out, grads = _run(q, *(torch.where(mask[:, :, None, None], t, other) for t in (k, v)), mask, None, g)
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(grads, gradients))
    # NaN of a key that takes part, or of a query, stays in its sequence and head (and the query's in its row of the result)
    k[2, 70, 0, 1] = math.nan
    q[0, 0, H - 1, 3] = math.nan
    out, _ = _run(q, k, v, mask)
    assert out[2, :, :H // Hk].isnan().all() and out[0, 0, H - 1].isnan().all()
    rest = out.clone()
    rest[2, :, :H // Hk], rest[0, 0, H - 1] = 0, 0
    assert rest.isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_and_small_numbers(dtype):
    """Scores up to some hundred (one key has all the weight), a scale of its own, gradients near either end of half's normal numbers, weights of many keys."""
    B, Lq, Lk, H, D = 2, 100, 700, 2, 64
    q, k, v, g = (_randn(B, n, H, D, dtype=dtype, seed=s) for s, n in enumerate((Lq, Lk, Lk, Lq)))
    for q1, scale, v1, g1 in ((q * 30, None, v, g), (q, 0.01, v, g), (q, None, v * 100, g * 1e-3), (q, None, v, g * 500), (q * 0.01, 3.0, v * 0.01, g * 0.02)):
        out, grads = _run(q1, k, v1, None, scale, g1)
        want, gradients, bounds = _reference(q1, k, v1, None, scale or D ** -0.5, g1)
        for a, b, c in zip((out, *grads), (want, *gradients), bounds):
            _close(a, b, c)
    k, v = (_randn(1, 20000, 1, D, dtype=dtype, seed=s) for s in (7, 8))
    q, g = _randn(1, 60, 1, D, dtype=dtype), _randn(1, 60, 1, D, dtype=dtype, seed=1)
    out, grads = _run(q, k, v, None, None, g)
    want, gradients, bounds = _reference(q, k, v, None, D ** -0.5, g)
    for a, b, c in zip((out, *grads), (want, *gradients), bounds):
        _close(a, b, c)
    if dtype != torch.float32:
        # as near as the type's own rounding has it: 1.5 times the error of results that are rounded once, of either sign
        for a, b in zip((out, *grads), (want, *gradients)):
            assert (a.double().cpu() - b).norm() <= 1.5 * (b.to(dtype).double() - b).norm()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Lq,Lk", [(1, 200), (90, 150)])
def test_layouts(Lq, Lk, dtype):
    """Any strides give the bits of contiguous arrays: one projection of all three, heads first, broadcast keys, odd addresses, a mask's columns apart."""
    B, H, Hk, D = 2, 4, 2, 64
    q, g = _randn(B, Lq, H, D, dtype=dtype), _randn(B, Lq, H, D, dtype=dtype, seed=1)
    k, v = _randn(B, Lk, Hk, D, dtype=dtype, seed=2), _randn(B, Lk, Hk, D, dtype=dtype, seed=3)
    mask = _mask("holes", B, Lk)
    want, gradients = _run(q, k, v, mask, None, g)

    def same(q, k, v, mask, g):
        out, grads = _run(q, k, v, mask, None, g)
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(grads, gradients))

    kv = torch.stack((k, v), 2)
    same(q, kv[:, :, 0], kv[:, :, 1], mask, g)
    first = lambda t: t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)  # noqa: E731
    same(first(q), first(k), first(v), mask, first(g))
    columns_first = lambda t: t.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)  # noqa: E731
    same(columns_first(q), columns_first(k), v, mask, columns_first(g))
    odd = lambda t: torch.cat((t.flatten()[:1], t.flatten()))[1:].view(t.shape)  # noqa: E731
    same(odd(q), odd(k), odd(v), mask, odd(g))
    apart = torch.zeros(B, Lk, 3, dtype=torch.bool, device=DEV)
    apart[:, :, 1] = mask
    same(q, k, v, apart[:, :, 1], g)
    # one sequence's states for all, one key head for all: their gradients are what a user adds up
    out, _ = _run(q, k[:1].expand(B, -1, -1, -1), v[:1].expand(B, -1, -1, -1), mask[:1].expand(B, -1))
    assert torch.equal(out, _run(q, k[:1].repeat(B, 1, 1, 1), v[:1].repeat(B, 1, 1, 1), mask[:1].repeat(B, 1))[0])
    leaf = k[:1].detach().requires_grad_()
    got, = torch.autograd.grad(cross_attention(q, leaf.expand(B, -1, -1, -1), v, mask), leaf, g)
    assert torch.equal(got, gradients[1].sum(0, keepdim=True)) or not torch.equal(k[0], k[1])


@pytest.mark.parametrize("L,apart", [(300, 1 << 24), (600, 1 << 23)])
def test_rows_beyond_32_bits(L, apart):
    """Keys, values and queries that lie further apart than 32 bits reach: 32 MB from one to the next (a copy is made) and 16."""
    D = 64
    base = torch.empty(L, apart, dtype=torch.bfloat16, device=DEV)            # 10 GB, of which 3 x 64 columns are used
    q, k, v = (_randn(1, L, 1, D, dtype=torch.bfloat16, seed=s) for s in range(3))
    far = []
    for i, t in enumerate((q, k, v)):
        base[:, i * 64:(i + 1) * 64] = t[0, :, 0]
        far.append(base[:, i * 64:(i + 1) * 64][None, :, None])
    g = _randn(1, L, 1, D, dtype=torch.bfloat16, seed=3)
    want, gradients = _run(q, k, v, None, None, g)
    out, grads = _run(*far, None, None, g)
    assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(grads, gradients))
    assert torch.equal(_run(far[0][:, :1], *far[1:], None)[0], _run(q[:, :1], k, v, None)[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_to_do(dtype):
    for B, Lq, Lk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k = _randn(B, Lq, 4, 64, dtype=dtype).requires_grad_(), _randn(B, Lk, 2, 64, dtype=dtype).requires_grad_()
        out = cross_attention(q, k, k, torch.ones(B, Lk, dtype=torch.bool, device=DEV))
        assert out.shape == q.shape and not out.any()
        grads = torch.autograd.grad(out, (q, k), torch.ones_like(out))
        assert all(not t.any() for t in grads) and [t.shape for t in grads] == [q.shape, k.shape]


def test_gradients_that_are_wanted():
    q, k, v, g = (_randn(2, n, 2, 64, dtype=torch.float16, seed=s) for s, n in enumerate((50, 70, 70, 50)))
    _, every = _run(q, k, v, None, None, g)
    for wanted in ((0,), (1,), (2,), (0, 2), (1, 2)):
        leaves = [t.detach().requires_grad_(i in wanted) for i, t in enumerate((q, k, v))]
        got = torch.autograd.grad(cross_attention(*leaves), [leaves[i] for i in wanted], g)
        assert all(torch.equal(a, every[i]) for a, i in zip(got, wanted))
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = cross_attention(*leaves)
    grads = torch.autograd.grad(out, leaves, g, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(grads, every))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(grads[0].float().sum(), leaves)
    with torch.no_grad():
        assert not cross_attention(*leaves).requires_grad


def test_gradient_against_differences():
    q, k, v, g = (_randn(2, n, h, 32, seed=s) for s, (n, h) in enumerate(((9, 4), (37, 2), (37, 2), (9, 4))))
    mask = _mask("holes", 2, 37)
    _, grads = _run(q, k, v, mask, None, g)
    for i, x in enumerate((q, k, v)):
        step = _randn(*x.shape, seed=11)
        at = [[t + e * step if j == i else t for j, t in enumerate((q, k, v))] for e in (-0.05, 0.05, -0.1, 0.1)]
        a, b, c, d = ((_run(*s, mask)[0].double() * g.double()).sum().item() for s in at)
        slope = (8 * (b - a) - (d - c)) / (12 * 0.05)             # to the fourth order: 0.05^4 of the fifth derivative's size
        want = (grads[i].double() * step.double()).sum().item()
        # the results' rounding, 2^-22 of some 2300 terms of size 1, either sign, over the step: 2^-22 * 48 * 18 / 0.6; the order's rest 1e-3 of the size
        assert abs(slope - want) <= 2e-3 * max(abs(want), grads[i].norm().item())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("Lq,Lk", [(1, 512), (5, 2000), (200, 150)])
def test_captured_and_replayed(Lq, Lk, dtype):
    """Forward and a training step in two graphs that are replayed in turn, with eager calls and new inputs between them."""
    B, H, D = 2, 4, 64
    q, k, v, g = (_randn(B, n, H, D, dtype=dtype, seed=s) for s, n in enumerate((Lq, Lk, Lk, Lq)))
    mask = _mask("padded", B, Lk)
    _run(q, k, v, mask, None, g)                                    # (a kernel's first call asks for its LDS)
    _run(q, k, v, mask)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, results = [], []
    with torch.cuda.stream(side):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        for train in (False, True):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                if train:
                    out = cross_attention(*leaves, mask)
                    results.append((out.detach(), *torch.autograd.grad(out, leaves, g)))
                else:
                    with torch.no_grad():
                        results.append((cross_attention(q, k, v, mask),))
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        for t in (q, k, v, g):
            t.copy_(_randn(*t.shape, dtype=dtype, seed=20 + i))
        mask.copy_(_mask("holes" if i % 2 else "padded", B, Lk, seed=i))
        out, grads = _run(q, k, v, mask, None, g)
        for graph in graphs if i % 2 else graphs[::-1]:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(results[0][0], out)
        assert all(torch.equal(a, b) for a, b in zip(results[1], (out, *grads)))


def test_on_another_stream():
    q, k, v, g = (_randn(4, n, 4, 64, dtype=torch.bfloat16, seed=s) for s, n in enumerate((300, 1000, 1000, 300)))
    want, gradients = _run(q, k, v, None, None, g)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    late = torch.zeros_like(q)
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        late.copy_(q)                                               # what the call reads is there only when its stream gets to it
        out, grads = _run(late, k, v, None, None, g)
    side.synchronize()
    assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(grads, gradients))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Lq,Lk,D", [(1, 77, 64), (3, 5, 40), (129, 130, 128), (40, 4000, 24)])
def test_nothing_is_written_beside_the_results(Lq, Lk, D, dtype):
    """Through the C entries: results and workspaces inside larger arrays, whose other numbers stay."""
    import ctypes
    lib, B, H = lookupffn_amd._lib.load(), 2, 2
    q, k, v, g = (_randn(B, n, H, D, dtype=dtype, seed=s) for s, n in enumerate((Lq, Lk, Lk, Lq)))
    a = ops._cross_attention_args(q, k, v, None, D ** -0.5)
    n = ctypes.c_int64(0)
    guarded = []

    def room(numbers, dtype):
        t = torch.full((numbers + 128,), 77.0, device=DEV).to(dtype)
        guarded.append((t, numbers))
        return t[64:].data_ptr()

    assert lib.lffn_cross_attention_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) == 0
    stream = torch.cuda.current_stream().cuda_stream
    kept = ctypes.c_int64(0)
    assert lib.lffn_cross_attention_kept_bytes(ctypes.byref(a), ctypes.byref(kept)) == 0 and kept.value == ops._kept_bytes(q)
    out, lse = room(q.numel(), dtype), room(kept.value // 4, torch.float32)
    assert lib.lffn_cross_attention_fwd(ctypes.byref(a), out, lse, room(n.value // 4, torch.float32), n.value, stream) == 0
    assert lib.lffn_cross_attention_bwd_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) == 0
    grads = [room(t.numel(), dtype) for t in (q, k, v)]
    assert lib.lffn_cross_attention_bwd(ctypes.byref(a), out, lse, g.data_ptr(), *grads, room(n.value // 4, torch.float32), n.value, stream) == 0
    torch.cuda.synchronize()
    for t, numbers in guarded:
        assert (t[:64] == 77).all() and (t[64 + numbers:] == 77).all()
    want, gradients = _run(q, k, v, None, None, g)
    inside = [t[64:64 + numbers] for t, numbers in guarded]
    assert torch.equal(inside[0], want.flatten())
    assert all(torch.equal(a, b.flatten()) for a, b in zip((inside[3], inside[4], inside[5]), gradients))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Lq,Lk", [(1, 2), (300, 5), (40, 3000), (200, 70)])
def test_gradients_of_few_keys_are_as_near(Lq, Lk, dtype):
    """Of few keys ds is what two terms of one size leave: with a sum over the rounded result for one of them it was off by twice a rounding.  Results off by a
    rounding of their own and one of each weight (or ds), of either sign: 1.41 of the first alone."""
    q, k, v, g = (_randn(4, n, 8, 64, dtype=dtype, seed=s) for s, n in enumerate((Lq, Lk, Lk, Lq)))
    out, grads = _run(q, k, v, None, None, g)
    want, gradients, _ = _reference(q, k, v, None, 0.125, g)
    for a, b in zip((out, *grads), (want, *gradients)):
        assert (a.double().cpu() - b).norm() <= 1.5 * (b.to(dtype).double() - b).norm()
