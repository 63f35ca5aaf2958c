"""Forward-mode derivatives of qk_norm_rotary and cross_attention, which have none: raised, never dropped.  Without a GPU, on tensors that have no memory."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode

from lookupffn_amd import cross_attention, qk_norm_rotary


def _inputs():
    gpu = lambda *shape, dtype=torch.float16: torch.empty(*shape, dtype=dtype, device="cuda")  # noqa: E731
    attention = dict(q=gpu(2, 3, 4, 64), k=gpu(2, 5, 2, 64), v=gpu(2, 5, 2, 64))
    norm = dict(q=gpu(2, 3, 4, 64), k=gpu(2, 5, 2, 64), q_weight=gpu(64, dtype=torch.float32), k_weight=gpu(64))       # (a weight of q's type as well)
    return attention, norm


CASES = [(cross_attention, 0, n) for n in ("q", "k", "v")] + [(qk_norm_rotary, 1, n) for n in ("q", "k", "q_weight", "k_weight")]


@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("call,which,name", CASES)
def test_a_tangent_is_refused(call, which, name, recorded):
    with FakeTensorMode(), torch.set_grad_enabled(recorded):
        inputs = _inputs()[which]
        with fwAD.dual_level():
            call(**inputs)                  # nothing to lose
            inputs[name] = fwAD.make_dual(inputs[name], torch.ones_like(inputs[name]))
            with pytest.raises((NotImplementedError, RuntimeError)):
                call(**inputs)


@pytest.mark.parametrize("call,which,name", CASES)
def test_a_tangent_of_torch_func_is_refused(call, which, name):
    with FakeTensorMode():
        inputs = _inputs()[which]
        x = inputs.pop(name)
        with pytest.raises((NotImplementedError, RuntimeError)):
            torch.func.jvp(lambda t: call(**inputs, **{name: t}), (x,), (torch.ones_like(x),))
