"""A sequence whose mask leaves one key: it has all the weight, whatever the length of the array, in every kernel of the backward."""
import pytest
import torch

from test_gpu_cross_attention import _close, _randn, _reference, _run

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


# the kernels for all gradients together (16 bits, up to 128 rows, 33 to 64 columns) and apart, in pairs of wavefronts and alone, keys shared out and not
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("L,keys,H,Hk,D", [(1, 300, 4, 4, 64), (50, 2, 4, 2, 64), (5, 70, 4, 4, 16), (70, 700, 4, 2, 64), (200, 333, 4, 4, 64), (150, 9000, 2, 2, 128),
                                           (140, 4500, 2, 1, 32)])
def test_zeros(L, keys, H, Hk, D, dtype):
    """Gradients of queries and keys are zeros, not what two sums of the same terms differ by; those of a sequence with two keys are not."""
    B = 6
    q, k, v, g = (_randn(B, n, h, D, dtype=dtype, seed=s) for s, (n, h) in enumerate(((L, H), (keys, Hk), (keys, Hk), (L, H))))
    mask = torch.zeros(B, keys, dtype=torch.bool, device=DEV)
    mask[0, 0] = mask[1, -1] = mask[2, keys // 2] = True         # early, late and between
    mask[3, 0] = mask[3, -1] = True                              # two
    mask[4] = True                                               # (of sequence 5, none)
    out, (gq, gk, gv) = _run(q, k, v, mask, None, g)
    for n in (gq, gk):
        assert not n[:3].any() and not n[5].any()
        assert n[3].any() and n[4].any()
    want, gradients, bounds = _reference(q, k, v, mask, D ** -0.5, g)
    for a, b, c in zip((out, gq, gk, gv), (want, *gradients), bounds):
        _close(a, b, c)
    for b, key in enumerate((0, keys - 1, keys // 2)):           # one key alone gives what one of many does
        alone = _run(q[b:b + 1], k[b:b + 1, key:key + 1], v[b:b + 1, key:key + 1], None, None, g[b:b + 1])
        _close(alone[1][2], gradients[2][b:b + 1, key:key + 1], bounds[3][b:b + 1, key:key + 1])
        assert not alone[1][0].any() and not alone[1][1].any()


def test_captured_and_replayed_with_other_masks():
    """How many keys take part is found out on every replay."""
    q, k, v, g = (_randn(2, n, 4, 64, dtype=torch.float16, seed=s) for s, n in enumerate((40, 5000, 5000, 40)))
    mask = torch.zeros(2, 5000, dtype=torch.bool, device=DEV)
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def step():
        from lookupffn_amd import cross_attention
        out = cross_attention(*leaves, mask)
        return (out.detach(), *torch.autograd.grad(out, leaves, g))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for n in (1, 2, 5000, 0, 1):
        mask.zero_()
        mask[0, 5000 - n:] = True
        mask[1, :max(n, 2)] = True
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(replayed, step()))
        assert replayed[1][0].any().item() == replayed[2][0].any().item() == (n > 1)
