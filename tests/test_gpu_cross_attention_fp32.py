"""fp32 attention to an encoder's states where its numbers are two terms of half precision (csrc/cross_attention.h): many rows and keys forward, any sizes
backward; numbers of very different sizes; against 64 bits."""
import math

import pytest
import torch

from lookupffn_amd import cross_attention
from test_gpu_cross_attention import _close, _mask, _randn, _reference, _run

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# 256 rows of a key head or more, 5e8 products or more; every kernel's columns and between, shared heads, odd lengths
SIZES = [(1, 512, 1100, 8, 8, 128), (2, 600, 2100, 4, 2, 64), (8, 257, 700, 8, 8, 32), (3, 300, 1000, 4, 4, 120), (16, 2000, 77, 4, 4, 72)]


@pytest.mark.parametrize("mask", [None, "padded", "holes", "late"])
@pytest.mark.parametrize("B,Lq,Lk,H,Hk,D", SIZES)
def test_against_64_bits(B, Lq, Lk, H, Hk, D, mask):
    q, k, v, g = (_randn(B, n, h, D, seed=s) for s, (n, h) in enumerate(((Lq, H), (Lk, Hk), (Lk, Hk), (Lq, H))))
    spread, mask = mask in (None, "holes"), _mask(mask, B, Lk)
    out, grads = _run(q, k, v, mask, None, g)
    want, gradients, bounds = _reference(q, k, v, mask, D ** -0.5, g)
    for i, (a, b, c) in enumerate(zip((out, *grads), (want, *gradients), bounds)):
        _close(a, b, c)
        if spread or i in (0, 3):       # (of few keys dq and dk are what two terms of one size leave)
            assert (a.double().cpu() - b).norm() <= 1e-6 * b.norm()
    again, repeated = _run(q, k, v, mask, None, g)
    assert torch.equal(out, again) and all(torch.equal(a, b) for a, b in zip(grads, repeated))


def _two_terms(q, k, v, g, mask, scale):
    """What the bounds of fp32 arithmetic take on: a number that passes is held to 2^-36 of the longest row of its head, where that is more than 2^-22 of itself;
    weights, in the forward, to 2^-33 of their row's largest (half's last step, 2^-25, of at least 2^8); weights and ds, in the backward, to 2^-36 of
    their row's or key's largest (2^-25 of at least 2^11).  -> addends of the bounds of out, dq, dk, dv."""
    group, dims = q.shape[2] // k.shape[2], (0, 2, 1, 3)
    q, k, v, g = (t.double().cpu().permute(*dims) for t in (q, k, v, g))
    k, v = (t.repeat_interleave(group, 1) for t in (k, v))
    keep = torch.ones(q.shape[0], k.shape[2], dtype=torch.bool) if mask is None else mask.cpu()
    keep = keep[:, None, :, None]

    def held(t, shared=False):          # [B, H, 1, 1]
        rows = torch.where(keep, t, 0.0) if t.shape[2] == k.shape[2] and (t is k or t is v) else t
        longest = rows.norm(dim=-1).amax(-1)
        if shared:
            longest = longest.unflatten(1, (-1, group)).amax(2).repeat_interleave(group, 1)
        return 2.0 ** -36 * longest[:, :, None, None]

    hq, hk, hv, hg = held(q, True), held(k), held(v), held(g, True)
    s = (scale * q @ k.transpose(-1, -2)).masked_fill(~keep.transpose(-1, -2), -math.inf)
    p = s.softmax(-1)
    k, v = torch.where(keep, k, 0.0), torch.where(keep, v, 0.0)
    out = p @ v
    sums = lambda t: t.abs().sum(-1, keepdim=True)  # noqa: E731
    off = 2 * scale * (sums(q) * hk + (sums(k) * hq).transpose(-1, -2).amax(-1, keepdim=True)).amax(-1, keepdim=True)      # of a weight, relative; level and score
    b_out = off * (p @ v.abs()) + hv + 2.0 ** -33 * p.amax(-1, keepdim=True) * v.abs().sum(2, keepdim=True)
    ds = p * (g @ v.transpose(-1, -2) - (g * out).sum(-1, keepdim=True))
    off_ds = off * ds.abs() + p * (sums(g) * hv + (sums(v) * hg).transpose(-1, -2) + (g.abs() * b_out).sum(-1, keepdim=True))
    top_row, top_key = 2.0 ** -36 * ds.abs().amax(-1, keepdim=True), 2.0 ** -36 * ds.abs().amax(-2, keepdim=True).transpose(-1, -2)
    shared_k = lambda t: t.unflatten(1, (-1, group)).sum(2)  # noqa: E731
    t = lambda x: x.transpose(-1, -2)  # noqa: E731
    b_q = scale * (off_ds @ k.abs() + sums(ds) * hk + top_row * k.abs().sum(2, keepdim=True))
    b_k = scale * shared_k(t(off_ds) @ q.abs() + sums(t(ds)) * hq + top_key * q.abs().sum(2, keepdim=True))
    b_v = shared_k(t(off * p) @ g.abs() + sums(t(p)) * hg + 2.0 ** -36 * t(p.amax(-2, keepdim=True)) * g.abs().sum(2, keepdim=True))
    return [x.permute(*dims) for x in (b_out, b_q, b_k, b_v)]


def _held(q, k, v, g, mask=None, scale=None):
    scale = scale or q.shape[-1] ** -0.5
    out, grads = _run(q, k, v, mask, scale, g)
    want, gradients, bounds = _reference(q, k, v, mask, scale, g)
    for a, b, c, more in zip((out, *grads), (want, *gradients), bounds, _two_terms(q, k, v, g, mask, scale)):
        _close(a, b, c + more)


@pytest.mark.parametrize("B,Lq,Lk,H,Hk,D", [(1, 256, 2100, 8, 8, 128), (2, 300, 2000, 4, 2, 64), (2, 40, 130, 2, 1, 40)])
def test_numbers_of_many_sizes(B, Lq, Lk, H, Hk, D):
    """Rows from 2^-12 to 1 times the longest, columns from 2^-8 to 1; all of a tensor near either end of fp32's range; heads and sequences of sizes of their own."""
    q, k, v, g = (_randn(B, n, h, D, seed=s) for s, (n, h) in enumerate(((Lq, H), (Lk, Hk), (Lk, Hk), (Lq, H))))
    gen = torch.Generator(device=DEV).manual_seed(9)

    def powers(*shape, low):
        return 2.0 ** (low * torch.rand(*shape, generator=gen, device=DEV))
    for which in range(4):              # one tensor's rows and columns
        t = [q, k, v, g]
        t[which] = t[which] * powers(B, t[which].shape[1], t[which].shape[2], 1, low=-12) * powers(D, low=-8)
        _held(*t)
    _held(q * 1e-20, k * 1e20, v * 1e-25, g * 1e25)
    _held(q * 1e18, k * 1e-18, v * 1e18, g * 1e-12)
    _held(q * 1e-30, k * 1e-10, v, g)   # (scores of nothing)
    _held(q, k, v * 1e-34, g)           # (results near the end of the range, whose scaling back is no fp32 number)
    _held(q * 1e-16, k * 1e16, v * 1e-16, g * 1e-17)
    _held(q * powers(B, 1, H, 1, low=-20), k * powers(B, 1, Hk, 1, low=-20), v * powers(B, 1, Hk, 1, low=-20), g * powers(B, 1, H, 1, low=-20))


def test_weights_of_little():
    """Keys that hardly any query attends to: their gradients are as near as any key's."""
    q, k, v, g = (_randn(2, n, 4, 64, seed=s) for s, n in enumerate((300, 2000, 2000, 300)))
    k[:, 100:] = k[:, 100:] * 0.01 - 1.5 * q.mean(1, keepdim=True)
    q = q + 4.0
    k[:, ::2] -= 1.0                    # scores some 32 lower
    _held(q, k, v, g)


@pytest.mark.parametrize("which", range(4))
def test_zeros(which):
    t = [_randn(2, n, 4, 64, seed=s) for s, n in enumerate((300, 2000, 2000, 300))]
    t[which].zero_()
    _held(*t)
    t = [_randn(2, n, 4, 64, seed=s) for s, n in enumerate((300, 2000, 2000, 300))]
    t[which][:, 64:] = 0
    t[which][1, :, 2] = 0
    _held(*t)


def test_what_takes_no_part_is_not_looked_at():
    """Infinities, NaN and the lowest number in masked keys and values do not count among the longest rows; those that take part stay in their head."""
    B, Lq, Lk, H, Hk, D = 3, 300, 2000, 4, 2, 64
    q, k, v, g = (_randn(B, n, h, D, seed=s) for s, (n, h) in enumerate(((Lq, H), (Lk, Hk), (Lk, Hk), (Lq, H))))
    mask = torch.arange(Lk, device=DEV) < torch.tensor([[Lk // 2], [0], [Lk - 1]], device=DEV)
    mask[0, 3], mask[2, :66] = False, False
    clean = [torch.where(mask[:, :, None, None], t, 0.0) for t in (k, v)]
    want, gradients = _run(q, *clean, mask, None, g)
    for other in (math.nan, math.inf, -math.inf, torch.finfo(torch.float32).min):
        out, grads = _run(q, *(torch.where(mask[:, :, None, None], t, other) for t in (k, v)), mask, None, g)
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(grads, gradients))
    for bad in (math.nan, math.inf):
        v2, q2 = v.clone(), q.clone()
        v2[2, 70, 0, 1] = bad           # of a value: in its column, where it has weight
        q2[0, 0, H - 1, 3] = bad        # of a query: in its row
        out, _ = _run(q2, k, v2, mask)
        same = torch.ones_like(out, dtype=torch.bool)
        same[2, :, :H // Hk], same[0, 0, H - 1] = False, False
        assert not out[2, :, :H // Hk, 1].isfinite().any() and out[0, 0, H - 1].isnan().all()
        assert torch.equal(out[same], want[same])
        assert (out[2, :, :H // Hk, 2:] - want[2, :, :H // Hk, 2:]).abs().max() <= 1e-5


def test_captured_and_replayed():
    q, k, v, g = (_randn(2, n, 4, 64, seed=s) for s, n in enumerate((300, 2000, 2000, 300)))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]

    def step():
        out = cross_attention(*leaves)
        return (out.detach(), *torch.autograd.grad(out, leaves, g))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step()
    for n in range(4):
        with torch.no_grad():
            for t, new in zip(leaves, (q, k, v)):
                t.copy_(new * 10.0 ** (n - 2))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in results]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
