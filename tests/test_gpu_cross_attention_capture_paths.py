"""Captured training forwards on Python's path: those whose leaves a graph from before the capture holds are refused there as on the host path, before anything is put
into the graph (their backward would end the process)."""
import pytest
import torch

import lookupffn_amd
from lookupffn_amd import _lib, cross_attention, qk_norm_rotary, rotary_table

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _leaves(dtype=torch.float16):
    g = torch.Generator(device=DEV).manual_seed(0)
    return [torch.randn(2, n, 4, 64, generator=g, device=DEV).to(dtype).requires_grad_() for n in (40, 70, 70)]


def _captured(call, side):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = call()
    return graph, got


def _refused(call, side, match="graph from before the capture"):
    def inside():
        with pytest.raises(RuntimeError, match=match):
            call()
        return torch.zeros(1, device=DEV)           # (a graph with nothing in it is warned about)
    _captured(inside, side)[0].replay()
    torch.cuda.synchronize()


def _works(call, inputs, side, want):
    def step():
        out = call()
        return (out.detach(), *torch.autograd.grad(out, inputs, torch.ones_like(out)))
    graph, got = _captured(step, side)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def _eager(call, inputs):
    out = call()
    return (out.detach(), *torch.autograd.grad(out, inputs, torch.ones_like(out), retain_graph=True)), out


# what leaves the host path: it is switched off; weights of the model's type; positions of two types; no host library at all is test_without_the_host_library
@pytest.mark.parametrize("what", ["attention", "norms", "weights", "positions"])
def test_refused_and_then_not(what, monkeypatch):
    q, k, v = _leaves()
    w = torch.ones(64, device=DEV, dtype=torch.float16, requires_grad=True)
    table = rotary_table(100, 64, device=DEV)
    at = torch.arange(40, device=DEV), torch.arange(70, device=DEV, dtype=torch.int32)
    if what in ("attention", "norms"):
        monkeypatch.setattr(_lib, "loaded_host", False)
    else:
        assert _lib.host()
    call, inputs = {"attention": (lambda: cross_attention(q, k, v), (q, k, v)),
                    "norms": (lambda: qk_norm_rotary(q, k)[1], (k,)),
                    "weights": (lambda: qk_norm_rotary(q.detach(), None, w)[0], (w,)),
                    "positions": (lambda: qk_norm_rotary(q, k, table=table, q_positions=at[0], k_positions=at[1])[0], (q,))}[what]
    side = torch.cuda.Stream()
    want, held = _eager(call, inputs)
    side.wait_stream(torch.cuda.current_stream())
    _refused(call, side)
    with torch.no_grad():
        graph, got = _captured(call, side)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want[0])
    del held
    _works(call, inputs, side, want)


def test_a_weight_that_is_not_read_holds_nothing_up():
    """That of keys, where there are none."""
    q, _, _ = _leaves()
    w, other = torch.ones(64, device=DEV, requires_grad=True), torch.ones(64, device=DEV, dtype=torch.float16, requires_grad=True)
    call = lambda: qk_norm_rotary(q, None, w.half(), other)[0]  # noqa: E731
    held = other * 2
    want, out = _eager(call, (q,))
    del out
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    _works(call, (q,), side, want)
    assert held.requires_grad


def test_without_the_host_library(monkeypatch):
    """Nothing tells then whether a graph holds a leaf: captured training forwards are refused; all else works."""
    monkeypatch.setattr(_lib, "loaded_host", False)
    monkeypatch.setattr(_lib, "host_module", lambda: None)
    q, k, v = _leaves()
    call = lambda: cross_attention(q, k, v)  # noqa: E731
    want, _ = _eager(call, (q, k, v))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    _refused(call, side, "only with the host library")
    _refused(lambda: qk_norm_rotary(q, k), side, "only with the host library")
    with torch.no_grad():
        graph, got = _captured(call, side)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want[0])
    again, _ = _eager(call, (q, k, v))
    assert all(torch.equal(a, b) for a, b in zip(again, want))


def test_the_host_library_is_found():
    assert _lib.host_module() is not None and lookupffn_amd._lib.host_module().refuse_foreign_leaves(None, torch.zeros(1)) is None
