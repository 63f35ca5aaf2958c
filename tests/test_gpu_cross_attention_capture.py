"""Training steps that are captured while other graphs of the same leaves live, on other streams, two at once."""
import pytest
import torch

import lookupffn_amd
from lookupffn_amd import cross_attention, qk_norm_rotary

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _leaves(dtype=torch.float32, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(2, n, 4, 64, generator=g, device=DEV).to(dtype).requires_grad_() for n in (40, 70, 70)]


def test_a_graph_from_before_the_capture_is_refused():
    """While an eager graph holds the leaves their gradients accumulate on its stream, which a captured backward must not wait for: the captured forward is
    refused, nothing is put into the graph, and once the eager graph is gone the capture works."""
    assert lookupffn_amd._lib.host()
    q, k, v = _leaves()
    eager = cross_attention(q, k, v)
    normed = qk_norm_rotary(q, k)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(RuntimeError, match="graph from before the capture"):
            cross_attention(q, k, v)
        with pytest.raises(RuntimeError, match="graph from before the capture"):
            qk_norm_rotary(q, k)
        with torch.no_grad():               # without gradients there is nothing to wait for
            inside = cross_attention(q, k, v)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(inside, eager)
    want = torch.autograd.grad(eager, (q, k, v), torch.ones_like(eager))
    del eager, normed
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = cross_attention(q, k, v)
        grads = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, inside) and all(torch.equal(a, b) for a, b in zip(grads, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_two_captured_graphs_replayed_in_turn(dtype):
    """Workspaces are each graph's own."""
    made = []
    for seed in range(2):
        leaves = _leaves(dtype, seed)
        eager = cross_attention(*leaves)
        want = (eager.detach().clone(), *torch.autograd.grad(eager, leaves, torch.ones_like(eager)))
        del eager
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = cross_attention(*leaves)
            got = (out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out)))
        made.append((graph, got, want, leaves))
    for _ in range(3):
        for graph, _, _, _ in made:
            graph.replay()
        torch.cuda.synchronize()
        for _, got, want, _ in made:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        torch.randn(1 << 20, device=DEV).sum().item()


def test_two_streams_at_once():
    streams = [torch.cuda.Stream() for _ in range(2)]
    sets = [_leaves(torch.bfloat16, seed) for seed in range(2)]
    want = []
    for leaves in sets:
        out = cross_attention(*leaves)
        want.append((out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out))))
    del out
    got = [None, None]
    for _ in range(10):
        for i, (stream, leaves) in enumerate(zip(streams, sets)):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                out = cross_attention(*leaves)
                got[i] = (out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out)))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_one_tensor_for_several_arguments():
    """Keys that are their own values, and queries that are both: gradients add up."""
    x = torch.randn(2, 90, 4, 64, device=DEV).requires_grad_()
    g = torch.randn(2, 90, 4, 64, device=DEV)
    got, = torch.autograd.grad(cross_attention(x, x, x), x, g)
    three = [x.detach().clone().requires_grad_() for _ in range(3)]
    each = torch.autograd.grad(cross_attention(*three), three, g)
    total = sum(t.double() for t in each)
    # two additions in fp32 of terms no larger than their sizes' sum
    assert ((got.double() - total).abs() <= 2.0 ** -23 * sum(t.abs() for t in each).double()).all()
    states = torch.randn(2, 33, 2, 64, device=DEV).requires_grad_()
    query = torch.randn(2, 1, 4, 64, device=DEV)
    out = cross_attention(query.expand(2, 5, 4, 64), states, states)         # the same query five times, by a stride of zero
    assert torch.equal(out, out[:, :1].expand_as(out))
    out.sum().backward()
    assert states.grad.isfinite().all()
