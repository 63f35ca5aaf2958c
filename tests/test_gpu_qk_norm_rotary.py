"""Norms of queries and keys with the rotation to their positions (csrc/qk_norm_rotary.hip), forward and backward, against 64 bits."""
import pytest
import torch

import lookupffn_amd
from lookupffn_amd import qk_norm_rotary, rotary_table

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


def _turn(y, table, positions, interleaved, back=False):
    if table is None:
        return y
    table = table.double().cpu()
    rows = table[positions.long().cpu().clamp(0, table.shape[0] - 1).expand(y.shape[:2])][:, :, None]
    half = table.shape[1] // 2
    cos, sin = rows[..., :half], rows[..., half:] * (-1 if back else 1)
    y = y.clone()
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
    return y


def _reference(x, w, table, positions, eps, interleaved, g):
    """-> ((y, grad x, grad w), their bounds).  A row's sums of at most 256 squares or products are off by 2^-20 of their sizes (at most 8 + 8 additions
    in a lane and the exchanges behind them, 2^-24 each), so is what follows of them; a rounding to the type at the end."""
    u = torch.finfo(x.dtype).eps / 2
    tiny = 2.0 ** -24 if x.dtype == torch.float16 else 1e-37
    x, g = x.detach().double().cpu(), g.double().cpu()
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.detach().double().cpu()
    if positions is None:
        positions = torch.arange(x.shape[1])
    r = 1 / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    y = _turn(x * r * w, table, positions, interleaved)
    h = _turn(g, table, positions, interleaved, back=True)
    gx = r * (h * w - x * r * (h * w * x * r).mean(-1, keepdim=True))
    gw = (h * x * r).sum((0, 1, 2))
    most = lambda t: t.abs().amax(-1, keepdim=True) if t.numel() else t.abs()  # noqa: E731
    sizes = r * (most(h * w) + most(x * r) * (h * w * x * r).abs().mean(-1, keepdim=True))
    return (y, gx, gw), (u * y.abs() + 2.0 ** -20 * 1.5 * most(x * r * w) + tiny, u * gx.abs() + 2.0 ** -19 * sizes + tiny,
                         2.0 ** -18 * (h.abs() * (x * r).abs()).sum((0, 1, 2)) + 1e-37)


def _close(got, want, bound):
    assert got.shape == want.shape and got.isfinite().all()
    worst = ((got.double().cpu() - want).abs() / bound).max().item() if got.numel() else 0.0
    assert worst <= 1, worst


# B, queries, keys, heads, key heads, columns, rotated columns: rows of one to 32 lanes, odd numbers of vectors, one to four heads a lane group, tokens beyond
# the workgroups of a backward
SIZES = [(1, 1, 1, 1, 1, 8, 0), (2, 1, None, 12, 12, 64, 64), (3, 7, 5, 3, 1, 16, 16), (2, 33, 65, 5, 2, 128, 64), (1, 77, 10, 16, 4, 128, 128), (2, 19, 23, 2, 2, 256, 256),
         (4, 50, 3, 7, 7, 40, 32), (2, 129, 64, 4, 4, 96, 16), (1, 3, 200, 2, 1, 24, 0), (8, 900, 1100, 12, 4, 64, 64), (3, 2100, 1, 16, 1, 72, 48)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,Lq,Lk,H,Hk,D,R", SIZES)
def test_against_64_bits(B, Lq, Lk, H, Hk, D, R, interleaved, dtype):
    q, gq = _randn(B, Lq, H, D, dtype=dtype), _randn(B, Lq, H, D, dtype=dtype, seed=1)
    k, gk = (None, None) if Lk is None else (_randn(B, Lk, Hk, D, dtype=dtype, seed=2), _randn(B, Lk, Hk, D, dtype=dtype, seed=3))
    qw, kw = 1 + 0.2 * _randn(D, seed=4), None if Lk is None or D == 24 else 1 + 0.2 * _randn(D, seed=5)
    table = rotary_table(500, R, device=DEV) if R else None
    qp = torch.randint(-3, 510, (B, Lq), device=DEV)                # (some outside the table)
    kp = None if Lk is None or D == 16 else torch.randint(0, 500, (Lk,), device=DEV, dtype=torch.int32)
    leaves = [t.requires_grad_() for t in (q, k, qw, kw) if t is not None]
    run = lambda: qk_norm_rotary(q, k, qw, kw, table=table, q_positions=qp, k_positions=kp, eps=1e-5, interleaved=interleaved)  # noqa: E731
    out = run()
    assert (out[1] is None) == (k is None)
    outs, gs = [t for t in out if t is not None], [t for t in (gq, gk) if t is not None]
    grads = torch.autograd.grad(outs, leaves, gs)
    of_x, of_w = list(grads[:len(gs)]), list(grads[len(gs):])
    for i, (x, w, p, g) in enumerate(((q, qw, qp, gq), (k, kw, kp, gk))):
        if x is None:
            continue
        (y, gx, gw), bounds = _reference(x, w, table, p, 1e-5, interleaved, g)
        _close(outs[i].detach(), y, bounds[0])
        _close(of_x[i], gx, bounds[1])
        if w is not None:
            _close(of_w.pop(0), gw, bounds[2])
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(outs, run()))
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad([t for t in run() if t is not None], leaves, gs)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts_and_types(dtype):
    """Any strides give the bits of contiguous arrays; weights of q's type and positions of either width; zeros and large numbers."""
    B, L, H, Hk, D = 2, 9, 4, 2, 64
    q, k = _randn(B, L, H, D, dtype=dtype), _randn(B, L, Hk, D, dtype=dtype, seed=1)
    table, qw = rotary_table(50, 32, device=DEV), 1 + 0.2 * _randn(D, seed=4)
    at = torch.randint(0, 50, (B, L), device=DEV)
    want = qk_norm_rotary(q, k, qw, qw, table=table, q_positions=at, k_positions=at)

    def same(q, k, at=at, kat=at):
        assert all(torch.equal(a, b) for a, b in zip(qk_norm_rotary(q, k, qw, qw, table=table, q_positions=at, k_positions=kat), want))

    qkv = torch.cat((q, k, k), 2)
    same(qkv[:, :, :H], qkv[:, :, H:H + Hk])
    first = lambda t: t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)  # noqa: E731
    same(first(q), first(k))
    odd = lambda t: torch.cat((t.flatten()[:1], t.flatten()))[1:].view(t.shape)  # noqa: E731
    same(odd(q), odd(k))
    same(q, k, at.int(), at)
    same(q, k, at.int(), at.int())
    same(q, k, torch.stack((at, at), 2)[:, :, 0])
    row = qk_norm_rotary(q, k, qw, qw, table=table, q_positions=at[0], k_positions=at[0])
    all_rows = qk_norm_rotary(q, k, qw, qw, table=table, q_positions=at[:1].expand(B, -1), k_positions=at[0])
    assert all(torch.equal(a, b) for a, b in zip(row, all_rows))
    own = qw.to(dtype)
    assert torch.equal(qk_norm_rotary(q, None, own)[0], qk_norm_rotary(q, None, own.float())[0])
    x = torch.zeros(1, 2, 1, D, device=DEV, dtype=dtype)
    assert not qk_norm_rotary(x)[0].any()
    x[0, 1] = 100.0
    y = qk_norm_rotary(x, eps=0.0)[0]
    assert y[0, 0].isnan().all() and (y[0, 1].float() - 1).abs().max() <= torch.finfo(dtype).eps       # 0 / 0, as the formula has it


def test_nothing_to_do():
    for B, Lq, Lk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k = _randn(B, Lq, 4, 64).requires_grad_(), _randn(B, Lk, 2, 64).requires_grad_()
        w = torch.ones(64, device=DEV, requires_grad=True)
        a, b = qk_norm_rotary(q, k, w, w)
        assert a.shape == q.shape and b.shape == k.shape
        grads = torch.autograd.grad((a, b), (q, k, w), (torch.ones_like(a), torch.ones_like(b)))
        assert [t.shape for t in grads] == [q.shape, k.shape, w.shape] and grads[2].isfinite().all()


def test_one_of_two_gradients():
    q, k, w = _randn(2, 3, 4, 64).requires_grad_(), _randn(2, 5, 2, 64, seed=1).requires_grad_(), torch.ones(64, device=DEV, requires_grad=True)
    g = _randn(2, 3, 4, 64, seed=2)
    a, b = qk_norm_rotary(q, k, w, w)
    gq, gk, gw = torch.autograd.grad(a, (q, k, w), g)
    alone = torch.autograd.grad(qk_norm_rotary(q, None, w)[0], (q, w), g)
    assert torch.equal(gq, alone[0]) and torch.equal(gw, alone[1]) and not gk.any()
    a, b = qk_norm_rotary(q, k, w, w)
    got = torch.autograd.grad((a, b), (q, k), (g, torch.ones_like(b)), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(got[0].sum(), q)


def test_captured_and_replayed():
    q, k = (_randn(3, n, 4, 64, dtype=torch.float16, seed=n).requires_grad_() for n in (70, 90))
    w, table = torch.ones(64, device=DEV, requires_grad=True), rotary_table(100, 64, device=DEV)
    at = torch.randint(0, 100, (3, 70), device=DEV)
    gs = [torch.ones(3, n, 4, 64, device=DEV, dtype=torch.float16) for n in (70, 90)]

    def step(q, k, w):
        out = qk_norm_rotary(q, k, w, w, table=table, q_positions=at)
        return (*(t.detach() for t in out), *torch.autograd.grad(out, (q, k, w), gs))

    step(q, k, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step(q, k, w)
    for i in range(4):
        with torch.no_grad():
            for t in (q, k, *gs):
                t.copy_(_randn(*t.shape, seed=i).half())
            w.copy_(1 + 0.1 * _randn(64, seed=i))
            at.copy_(torch.randint(0, 100, at.shape, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        fresh = [t.detach().clone().requires_grad_() for t in (q, k, w)]
        assert all(torch.equal(a, b) for a, b in zip(got, step(*fresh)))


def test_rows_beyond_32_bits():
    base = torch.empty(300, 1 << 24, dtype=torch.bfloat16, device=DEV)
    x = _randn(1, 300, 1, 64, dtype=torch.bfloat16)
    base[:, 64:128] = x[0, :, 0]
    far = base[:, 64:128][None, :, None]
    table = rotary_table(300, 64, device=DEV)
    assert torch.equal(qk_norm_rotary(far, far, table=table)[1], qk_norm_rotary(x, x, table=table)[0])
