"""Rows of an embedding table by token number (csrc/embedding.hip) and the table's gradient, against 64 bits."""
import pytest
import torch

import lookupffn_amd
from lookupffn_amd import embedding

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(autouse=True, params=["host", "python"])
def either_path(request, monkeypatch):
    """The calls with the host path in C++ and without."""
    if request.param == "python":
        monkeypatch.setattr(lookupffn_amd._lib, "loaded_host", False)
    else:
        assert lookupffn_amd._lib.host()


def _randn(*shape, dtype=torch.float32, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed + sum(shape)), device=DEV).to(dtype)


def _close(got, want, bound):
    assert got.shape == want.shape and got.isfinite().all()
    assert ((got.double().cpu() - want).abs() <= bound).all()


def _check(ids, w, scale, padding, g):
    """A result is a product in fp32 and a rounding to the type.  A sum of m numbers in fp32, in any order, is off by m 2^-24 of their sizes' sum, its product with the scale
    by another 2^-24; a rounding to the type at the end."""
    u, tiny = torch.finfo(w.dtype).eps / 2, torch.finfo(w.dtype).smallest_normal * 2.0 ** -8
    w.requires_grad_()
    out = embedding(ids, w, scale=scale, padding_idx=padding)
    grad, = torch.autograd.grad(out, w, g)
    assert out.dtype == w.dtype and grad.dtype == w.dtype and grad.shape == w.shape
    flat, rows = ids.reshape(-1).long().cpu(), w.shape[0]
    there = (flat >= 0) & (flat < rows)
    table = w.detach().double().cpu()
    want = torch.where(there[:, None], table[torch.where(there, flat, 0)] * scale, 0.0) if rows else torch.zeros(flat.numel(), w.shape[1], dtype=torch.float64)
    _close(out.detach().reshape(want.shape), want, (u + 2.0 ** -24) * want.abs() + tiny)
    if scale == 1:
        assert torch.equal(out.detach().reshape(want.shape).double().cpu(), want)
    use = there if padding is None else there & (flat != padding % rows)
    gs = g.double().cpu().reshape(-1, w.shape[1])[use]
    total = torch.zeros(w.shape, dtype=torch.float64).index_add_(0, flat[use], gs)
    sizes = torch.zeros(w.shape, dtype=torch.float64).index_add_(0, flat[use], gs.abs())
    count = torch.zeros(rows, dtype=torch.float64).index_add_(0, flat[use], torch.ones(len(gs), dtype=torch.float64))[:, None]
    _close(grad, total * scale, u * (total * scale).abs() + (count + 1) * 2.0 ** -24 * abs(scale) * sizes + tiny)
    assert (grad[(count == 0)[:, 0].to(DEV)] == 0).all()
    with torch.no_grad():
        assert torch.equal(embedding(ids, w, scale=scale, padding_idx=padding), out)
    again, = torch.autograd.grad(embedding(ids, w, scale=scale, padding_idx=padding), w, g)
    assert torch.equal(again, grad)


# tokens, rows, columns: none and one; a run through every piece; several workgroups of a sort; one, two and three passes; rows of one lane, of many blocks; odd widths; more chunks than each adds up by itself
SIZES = [(0, 5, 8), (1, 1, 1), (1, 50265, 768), (7, 3, 16), (17, 511, 24), (33, 512, 40), (385, 8191, 389), (1024, 700, 24), (1025, 9000, 16), (2048, 100, 64), (2049, 1, 129), (4096, 50265, 32), (4097, 3000, 8), (5000, 600, 512), (9001, 50265, 96),
         (40000, 2, 72), (3000, 300001, 9), (300, 20, 2056), (700, 31, 1030), (600001, 700, 8)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,rows,columns", SIZES)
def test_against_64_bits(tokens, rows, columns, dtype):
    gen = torch.Generator(device=DEV).manual_seed(tokens + rows)
    # some numbers often, most of them rarely, some outside the table
    ids = (rows * torch.rand(tokens, generator=gen, device=DEV) ** 6).long() - (torch.rand(tokens, generator=gen, device=DEV) < 0.03).long() * 2
    ids = torch.where(torch.rand(tokens, generator=gen, device=DEV) < 0.03, rows, ids)
    w, g = _randn(rows, columns, dtype=dtype), _randn(tokens, columns, dtype=dtype, seed=1)
    padding, scale = (None, 1.0) if tokens % 2 else (rows // 3, 0.75 if tokens % 4 else columns ** 0.5)
    _check(ids, w, scale, padding, g)


@pytest.mark.parametrize("ids", ["one", "distinct", "descending", "all outside", "all padding"])
def test_numbers(ids):
    n, rows = 3000, 4000
    ids = {"one": torch.full((n,), 3999), "distinct": torch.randperm(rows)[:n], "descending": torch.arange(n).flip(0), "all outside": torch.full((n,), rows),
           "all padding": torch.full((n,), 5)}[ids].to(DEV)
    _check(ids, _randn(rows, 64), -1.5, 5, _randn(n, 64, seed=2))


def test_shapes_types_and_layouts():
    w = _randn(90, 136, dtype=torch.float16)
    ids = torch.randint(0, 90, (3, 5, 7), device=DEV)
    g = _randn(3, 5, 7, 136, dtype=torch.float16, seed=1)
    _check(ids, w.clone(), 2.0, -1, g)
    _check(ids.int(), w.clone(), 1.0, 0, g)
    _check(ids.transpose(0, 2), w.clone(), 1.0, None, g.transpose(0, 2))
    _check(ids[..., ::2], w.clone(), 1.0, None, g[..., ::2, :])
    _check(ids[0, 0, 0], w.clone(), 1.0, None, g[0, 0, 0])
    for view in (w[:, 8:72], w[:, 3:68], w[::2], w.t()[:90], w[:1].expand(90, 136), w.flatten()[1:-1].view(-1, 2)):     # unaligned, strided, turned, one row
        _check(ids, view.detach(), 1.0, None, _randn(3, 5, 7, view.shape[1], dtype=torch.float16, seed=3))
    _check(ids, w.clone(), 1.0, None, g[:1, :1, :1, :1].expand(3, 5, 7, 136))
    _check(ids, w.clone(), 1.0, None, _randn(3 * 5 * 7 * 136 + 1, dtype=torch.float16)[1:].view(3, 5, 7, 136))
    out = embedding(ids, torch.empty(0, 24, device=DEV))                    # a table without rows
    assert out.shape == (3, 5, 7, 24) and (out == 0).all()


def test_a_sum_of_many():
    """One row of 100000 tokens: parts of pieces, added up by a launch of their own."""
    n = 100000
    g = (1 + _randn(n, 48, seed=4).abs())
    w = _randn(3, 48).requires_grad_()
    grad, = torch.autograd.grad(embedding(torch.full((n,), 1, device=DEV), w), w, g)
    want = g.double().sum(0)
    # a piece's 128 numbers, then a wavefront's share of 782 parts, 98, then 8: some 240 roundings of 2^-24 of sums of positive numbers
    assert ((grad[1].double() - want).abs() <= 240 * 2.0 ** -24 * want).all() and (grad[::2] == 0).all()


def test_infinities_stay_in_their_rows():
    w = _randn(10, 32).requires_grad_()
    ids = torch.tensor([1, 2, 2, 11, 3, 4], device=DEV)
    g = _randn(6, 32, seed=5)
    g[1] = float("inf")
    g[3] = float("nan")                 # of a token without a row
    g[5] = float("nan")                 # of the padding
    grad, = torch.autograd.grad(embedding(ids, w, padding_idx=4), w, g)
    assert grad[2].isinf().all() and grad[[0, 1, 3, 4, 5, 6, 7, 8, 9]].isfinite().all() and torch.equal(grad[1], g[0])
