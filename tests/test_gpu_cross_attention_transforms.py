"""qk_norm_rotary and cross_attention under what stands around PyTorch's operators: forward mode, torch.func, hooks on saved tensors, modes, torch.compile."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch.utils.checkpoint import checkpoint

import lookupffn_amd
from lookupffn_amd import cross_attention, qk_norm_rotary, rotary_table

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True, params=["host", "python"])
def either_path(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(lookupffn_amd._lib, "loaded_host", False)
    else:
        assert lookupffn_amd._lib.host()


def _inputs(dtype=torch.float16):
    gen = torch.Generator(device=DEV).manual_seed(0)
    return [torch.randn(2, n, h, 64, generator=gen, device=DEV).to(dtype) for n, h in ((40, 4), (70, 2), (70, 2))]


def _block(q, k, v, w, table, mask):
    q, k = qk_norm_rotary(q, k, w, w, table=table)
    return cross_attention(q, k, v, mask)


def _parts(dtype=torch.float16):
    return (*_inputs(dtype), 1 + 0.1 * torch.randn(64, device=DEV), rotary_table(100, 32, device=DEV), torch.arange(70, device=DEV) < torch.tensor([[70], [33]], device=DEV))


def _step(call, parts):
    leaves = [t.detach().clone().requires_grad_() for t in parts[:4]]
    out = call(*leaves, *parts[4:])
    return (out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out)))


@pytest.mark.parametrize("recorded", [False, True])
def test_a_tangent_is_refused(recorded):
    q, k, v = _inputs()
    w = torch.ones(64, device=DEV)
    with torch.set_grad_enabled(recorded), fwAD.dual_level():
        for i in range(3):
            inputs = [fwAD.make_dual(t, torch.ones_like(t)) if n == i else t for n, t in enumerate((q, k, v))]
            with pytest.raises((NotImplementedError, RuntimeError)):
                cross_attention(*inputs)
            with pytest.raises((NotImplementedError, RuntimeError)):
                qk_norm_rotary(inputs[0], inputs[1], fwAD.make_dual(w, w) if i == 2 else w)
        assert torch.equal(cross_attention(q, k, v), cross_attention(q, k, v))
    for call in (lambda t: cross_attention(t, k, v), lambda t: qk_norm_rotary(t, k)[0]):
        with pytest.raises((NotImplementedError, RuntimeError)):
            torch.func.jvp(call, (q,), (torch.ones_like(q),))


def test_torch_func():
    """Mapped over batches attention is one call after the other; the norms, whose operator has a list of results, and torch.func's gradients raise."""
    q, k, v = _inputs()
    mapped = torch.vmap(lambda a, b, c: cross_attention(a[None], b[None], c[None])[0])(q, k, v)
    assert torch.equal(mapped, torch.cat([cross_attention(q[i:i + 1], k[i:i + 1], v[i:i + 1]) for i in range(2)]))
    with pytest.raises(RuntimeError):
        torch.vmap(lambda a: qk_norm_rotary(a[None])[0][0])(q)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: cross_attention(t, k, v).float().sum())(q)


def test_hooks_on_saved_tensors_and_checkpoints():
    parts = _parts()
    want = _step(_block, parts)
    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t.cpu()) or packed[-1], lambda t: t.to(DEV)):
        got = _step(_block, parts)
    assert packed and all(torch.equal(a, b) for a, b in zip(got, want))
    got = _step(lambda *a: checkpoint(_block, *a, use_reentrant=False), parts)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_an_input_that_changes_before_the_backward_is_noticed():
    q, k, v = _inputs()
    for n in range(3):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        inputs = [t * 1 for t in leaves]
        out = cross_attention(*inputs)
        inputs[n].zero_()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.float().sum().backward()


def test_watched_calls():
    class Seen(torch.utils._python_dispatch.TorchDispatchMode):
        names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            Seen.names.append(str(func))
            return func(*args, **(kwargs or {}))

    parts = _parts()
    want = _step(_block, parts)
    with Seen():
        got = _step(_block, parts)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert {"lookupffn.cross_attention.default", "lookupffn.cross_attention_bwd.default", "lookupffn.qk_norm_rotary.default",
            "lookupffn.qk_norm_rotary_bwd.default"} <= set(Seen.names)


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled(backend):
    torch._dynamo.reset()
    parts = _parts()
    compiled = torch.compile(_block, backend=backend, fullgraph=True)
    with torch.no_grad():
        assert torch.equal(compiled(*parts), _block(*parts))
    want = _step(_block, parts)
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(_step(compiled, parts), want))


def test_batched_gradients_are_refused_and_a_jacobian_is_not():
    """Gradients of many vectors in one pass, which the backward does not take; one after the other they are those of the formula."""
    q, k, v = (t[:1, :3, :2, :16].float().clone() for t in _inputs())
    leaf = q.clone().requires_grad_()
    out = cross_attention(leaf, k, v)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, leaf, torch.eye(out.numel(), device=DEV).view(-1, *out.shape), is_grads_batched=True)
    got = torch.autograd.functional.jacobian(lambda t: cross_attention(t, k, v), q)
    q64, k64, v64 = (t.double().cpu() for t in (q, k, v))
    want = torch.autograd.functional.jacobian(lambda t: torch.einsum("bhij,bjhd->bihd", (torch.einsum("bihd,bjhd->bhij", t, k64) / 4).softmax(-1), v64), q64)
    # sums of three keys and sixteen columns, of terms of size 1 to 4: some ten roundings of 2^-24
    assert (got.double().cpu() - want).abs().max() <= 2.0 ** -19
    leaf = q.clone().requires_grad_()
    y, _ = qk_norm_rotary(leaf)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, leaf, torch.eye(y.numel(), device=DEV).view(-1, *y.shape), is_grads_batched=True)
