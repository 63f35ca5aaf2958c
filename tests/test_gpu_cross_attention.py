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
