"""Gradients of attention to an encoder's states where the queries of a key head are 128 at most: one kernel for all three (csrc/cross_attention_bwd.hip),
against 64 bits and against the kernels that form them apart."""
import math

import pytest
import torch

from lookupffn_amd import cross_attention
import test_gpu_cross_attention as attention
from test_gpu_cross_attention import _close, _mask, _randn, _reference, _run

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float16, torch.bfloat16]
# rows of a key head 1 to 128, around a wavefront's 32; keys around a step's 32 and beyond a block of 64 steps; 33 to 64 columns; shared heads; keys shared out
SIZES = [(3, 31, 65, 2, 2, 64), (2, 32, 64, 3, 3, 56), (2, 33, 31, 2, 2, 40), (2, 127, 200, 2, 1, 48), (2, 32, 257, 8, 2, 64), (1, 128, 4100, 1, 1, 64), (2, 1, 33, 4, 4, 64),
         (5, 96, 1, 2, 2, 64), (40, 20, 2150, 8, 8, 64), (3, 64, 129, 16, 8, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mask", [None, "padded", "holes", "late"])
@pytest.mark.parametrize("B,Lq,Lk,H,Hk,D", SIZES)
def test_against_64_bits(B, Lq, Lk, H, Hk, D, mask, dtype):
    q, k, v, g = (_randn(B, n, h, D, dtype=dtype, seed=s) for s, (n, h) in enumerate(((Lq, H), (Lk, Hk), (Lk, Hk), (Lq, H))))
    mask = _mask(mask, B, Lk)
    out, grads = _run(q, k, v, mask, None, g)
    want, gradients, bounds = _reference(q, k, v, mask, D ** -0.5, g)
    for a, b, c in zip((out, *grads), (want, *gradients), bounds):
        _close(a, b, c)
    if mask is not None:
        dead = ~mask[:, :, None, None].expand_as(k)
        assert not grads[1][dead].any() and not grads[2][dead].any()
    again, repeated = _run(q, k, v, mask, None, g)
    assert torch.equal(out, again) and all(torch.equal(a, b) for a, b in zip(grads, repeated))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,Lq,Lk,H,Hk,D", [(3, 1, 300, 4, 4, 64), (3, 90, 200, 4, 4, 64), (3, 40, 90, 6, 2, 40)])
def test_what_takes_no_part_is_not_looked_at(B, Lq, Lk, H, Hk, D, dtype):
    """Infinities, NaN and the type's lowest value in masked keys and values: the same bits as with zeros there; NaN of a query or its gradient stays in its sequence
    and key head, infinities of one key in its sequence and head."""
    q, k, v, g = (_randn(B, n, h, D, dtype=dtype, seed=s) for s, (n, h) in enumerate(((Lq, H), (Lk, Hk), (Lk, Hk), (Lq, H))))
    mask = torch.arange(Lk, device=DEV) < torch.tensor([[Lk // 2], [0], [Lk - 1]], device=DEV)
    mask[0, 3], mask[2, :66] = False, False
    clean = [torch.where(mask[:, :, None, None], t, 0.0) for t in (k, v)]
    want, gradients = _run(q, *clean, mask, None, g)
    for other in (math.nan, math.inf, -math.inf, torch.finfo(dtype).min):
        out, grads = _run(q, *(torch.where(mask[:, :, None, None], t, other) for t in (k, v)), mask, None, g)
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(grads, gradients))
    group = H // Hk
    for which in range(2):
        t = [q.clone(), g.clone()]
        t[which][0, Lq - 1, group - 1] = math.nan        # of sequence 0, key head 0
        _, grads = _run(t[0], *clean, mask, None, t[1])
        for i, (a, b, heads) in enumerate(zip(grads, gradients, (group, 1, 1))):
            same = torch.ones_like(a, dtype=torch.bool)
            same[0, :, :heads] = False
            assert torch.equal(a[same], b[same])
            if i:
                dead = ~mask[0]
                assert not a[0, dead, 0].any()           # zeros for keys that take no part, also here


@pytest.mark.parametrize("dtype", DTYPES)
def test_apart_and_together(dtype):
    """The gradients of queries alone and of keys and values alone, by kernels of their own: off by the roundings of either."""
    q, k, v, g = (_randn(4, n, 6, 64, dtype=dtype, seed=s) for s, n in enumerate((100, 333, 333, 100)))
    mask = _mask("holes", 4, 333)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = cross_attention(*leaves, mask)
    together = torch.autograd.grad(out, leaves, g, retain_graph=True)
    only_q = q.clone().requires_grad_()
    apart = [*torch.autograd.grad(cross_attention(only_q, k, v, mask), only_q, g)]
    only = [t.clone().requires_grad_() for t in (k, v)]
    apart += torch.autograd.grad(cross_attention(q, *only, mask), only, g)
    _, _, bounds = _reference(q, k, v, mask, 0.125, g)
    for a, b, c in zip(together, apart, bounds[1:]):
        assert ((a.double() - b.double()).abs().cpu() <= 2 * c).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_and_replayed(dtype):
    q, k, v, g = (_randn(3, n, 4, 64, dtype=dtype, seed=s) for s, n in enumerate((77, 500, 500, 77)))
    mask = _mask("padded", 3, 500)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]

    def step():
        out = cross_attention(*leaves, mask)
        return (out.detach(), *torch.autograd.grad(out, leaves, g))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step()
    for n in range(3):
        with torch.no_grad():
            for t, new in zip(leaves, (q, k, v)):
                t.copy_(new * (n + 1))
            mask.copy_(_mask("holes" if n else "late", 3, 500))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in results]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Lq,Lk,D", [(37, 45, 40), (128, 31, 64), (5, 2100, 64)])
def test_nothing_is_written_beside_the_results(Lq, Lk, D, dtype):
    attention.test_nothing_is_written_beside_the_results(Lq, Lk, D, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("mask", [None, "holes"])
@pytest.mark.parametrize("B,L,keys,H,D", [(4, 1000, 2900, 8, 64), (24, 20, 1600, 8, 32), (25, 32, 1537, 8, 64)])
def test_shared_out_with_a_tile_for_every_compute_unit(B, L, keys, H, D, mask, dtype):
    """Rows that fill the chip once and many keys, which are shared out over two to five workgroups each: against the same queries a few at a time, whose results are
    off by no more than the bounds against 64 bits."""
    q, k, v = (_randn(B, n, H, D, dtype=dtype, seed=s) for s, n in enumerate((L, keys, keys)))
    mask = _mask(mask, B, keys)
    out = cross_attention(q, k, v, mask)
    some = torch.arange(0, L, 97 if L > 100 else 1, device=DEV)
    want, _, (bound,) = _reference(q[:, some], k, v, mask, D ** -0.5)
    _close(out[:, some], want, bound)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("L,D", [(1, 64), (5, 16), (70, 64), (200, 64), (150, 128)])
def test_a_single_key(L, D, dtype):
    """It has all the weight: its values are the result, and the gradients of queries and keys are zeros, not what two sums of the same terms differ by."""
    q, k, v, g = (_randn(3, n, 4, D, dtype=dtype, seed=s) for s, n in enumerate((L, 1, 1, L)))
    for mask in (None, torch.tensor([[True], [False], [True]], device=DEV)):
        out, (gq, gk, gv) = _run(q, k, v, mask, None, g)
        want, gradients, bounds = _reference(q, k, v, mask, D ** -0.5, g)
        _close(out, want, bounds[0])
        _close(gv, gradients[2], bounds[3])
        assert not gq.any() and not gk.any()
