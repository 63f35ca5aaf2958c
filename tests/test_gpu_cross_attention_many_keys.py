"""fp32 attention to so many keys, by so many rows, that a lane adds the weights of all of a row's keys up: what a sum's length costs, against 64 bits."""
import pytest
import torch

from lookupffn_amd import cross_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def _reference(q, k, v, g, scale, mask):
    """One head after the other, in 64 bits on the GPU."""
    out, gq, gk, gv = (torch.zeros_like(t, dtype=torch.float64) for t in (q, q, k, v))
    for b in range(q.shape[0]):
        for h in range(q.shape[2]):
            qh, kh, vh, gh = (t[b, :, h].double() for t in (q, k, v, g))
            s = scale * (qh @ kh.T.contiguous())
            if mask is not None:
                s.masked_fill_(~mask[b], -torch.inf)
            p = s.softmax(1)
            out[b, :, h] = p @ vh
            gv[b, :, h] = p.T.contiguous() @ gh
            ds = scale * p * (gh @ vh.T.contiguous() - (gh * out[b, :, h]).sum(1, keepdim=True))
            gq[b, :, h] = ds @ kh
            gk[b, :, h] = ds.T.contiguous() @ qh
    return out, gq, gk, gv


# tiles of 128 rows that fill the chip, so that keys are not shared out; a step has 32 keys beyond 32 columns, else 64
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("L,keys,H,D,step", [(4096, 16384, 8, 72, 32), (6400, 8192, 8, 32, 64), (12800, 9000, 4, 64, 32)])
def test_the_sum_of_the_weights(L, keys, H, D, step, masked):
    gen = torch.Generator(device=DEV).manual_seed(L)
    q, k, v, g = (torch.randn(1, n, H, D, generator=gen, device=DEV) for n in (L, keys, keys, L))
    mask = torch.rand(1, keys, generator=gen, device=DEV) < 0.9 if masked else None
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = cross_attention(*leaves, mask)
    grads = torch.autograd.grad(out, leaves, g)
    q, k, v, out = (t.detach() for t in (q, k, v, out))
    want, *gradients = _reference(q, k, v, g, D ** -0.5, mask)
    # What is wrong with a row's sum scales the row: its part along the row, which the errors of the D columns' own sums hardly enter (1 / sqrt(D) of
    # theirs, U sqrt(keys / 8) at most: three products of 16 keys each are added one to the other).  The running sum is rounded once a step, by U of itself at
    # most, in a growing sum: sqrt(steps / 3) of them of either sign, each U / sqrt(3) in the mean.  Beside it the weights' own errors, the exponentials', U / 2 each, which
    # average out, and the level's and scores', a rounding of the scaled score each: 2 U.
    steps = (keys + step - 1) // step
    off = ((out.double() - want) * want).sum(-1) / want.pow(2).sum(-1)
    bound = U * ((steps / 9) ** 0.5 + (keys / 8 / D) ** 0.5 / 3 ** 0.5 + 2)
    assert off.pow(2).mean().sqrt() <= bound, (off.pow(2).mean().sqrt().item(), bound)
    # and all of it: the columns' sums, U / sqrt(3) a product of 16 in a sum that grows as a random walk, keys * 3 / 16 of them
    rest = U / 3 ** 0.5 * (3 * keys / 16 / 2) ** 0.5
    assert (out.double() - want).norm() <= (bound + rest) * want.norm()
    for name, a, b in zip("qkv", grads, gradients):
        # sums over keys (of q) or rows (of k and v), whose terms have the weights' errors (2^-21: two terms of 22 bits, a level), and their own
        n = L if name != "q" else keys
        own = U / 3 ** 0.5 * (3 * n / 16 / 2) ** 0.5
        assert (a.double() - b).norm() <= (bound + own + 2.0 ** -21) * b.norm(), name
