"""The operators behind qk_norm_rotary and cross_attention check types and shapes themselves, as the package's others do: arrays that do not fit would be read beyond
their ends.  Without a GPU, on tensors that have no memory."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from lookupffn_amd import ops


def _gpu(*shape, dtype=torch.float16):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def _attention():
    q, k = _gpu(2, 3, 4, 64), _gpu(2, 5, 2, 64)
    return dict(q=q, k=k, v=_gpu(2, 5, 2, 64), key_mask=_gpu(2, 5, dtype=torch.bool), scale=0.125)


def _attention_bwd():
    a = _attention()
    return dict(a, out=_gpu(2, 3, 4, 64), kept=_gpu(ops._kept_bytes(a["q"]), dtype=torch.uint8), g=_gpu(2, 3, 4, 64), of_queries=True, of_keys=True)


def _norm():
    return dict(q=_gpu(2, 3, 4, 64), k=_gpu(2, 5, 2, 64), q_weight=_gpu(64, dtype=torch.float32), k_weight=_gpu(64, dtype=torch.float32), table=_gpu(9, 32, dtype=torch.float32),
                q_positions=_gpu(2, 3, dtype=torch.int64), k_positions=_gpu(5, dtype=torch.int64), eps=1e-6, interleaved=False)


def _norm_bwd():
    a = _norm()
    return dict(a, g_q=_gpu(2, 3, 4, 64), g_k=_gpu(2, 5, 2, 64), want_q_weight=True, want_k_weight=True)


OF_ATTENTION = [("q", (2, 3, 64)), ("q", (2, 3, 4, 32)), ("q", torch.float32), ("q", torch.float64), ("k", (2, 5, 2, 32)), ("k", (3, 5, 2, 64)), ("k", (2, 5, 3, 64)), ("k", torch.float32),
                ("k", torch.bfloat16), ("v", (2, 4, 2, 64)), ("v", (2, 5, 1, 64)), ("v", torch.bfloat16), ("key_mask", (2, 4)), ("key_mask", (1, 5)), ("key_mask", (5,)), ("key_mask", torch.uint8)]
OF_NORM = [("q", (2, 3, 64)), ("q", torch.float64), ("k", (2, 5, 2, 32)), ("k", (3, 5, 2, 64)), ("k", torch.float32), ("q_weight", (32,)), ("q_weight", torch.float16),
           ("k_weight", (1, 64)), ("k_weight", torch.bfloat16), ("table", (288,)), ("table", torch.float16), ("q_positions", (2, 2)), ("q_positions", (2,)),
           ("q_positions", torch.int32), ("q_positions", torch.float32), ("k_positions", (4,)), ("k_positions", torch.int16)]


@pytest.mark.parametrize("impl,args,name,change", [
    *(("_cross_attention_impl", lambda: dict(_attention(), keep=True), *c) for c in OF_ATTENTION), *(("_cross_attention_bwd_impl", _attention_bwd, *c) for c in OF_ATTENTION),
    *(("_cross_attention_bwd_impl", _attention_bwd, *c) for c in (("out", (2, 2, 4, 64)), ("out", torch.float32), ("kept", (64,)), ("kept", torch.float32), ("g", (2, 3, 4, 32)),
                                                                  ("g", torch.float32))),
    *(("_qk_norm_rotary_impl", _norm, *c) for c in OF_NORM), *(("_qk_norm_rotary_bwd_impl", _norm_bwd, *c) for c in OF_NORM),
    *(("_qk_norm_rotary_bwd_impl", _norm_bwd, *c) for c in (("g_q", (2, 2, 4, 64)), ("g_q", torch.float32), ("g_k", (2, 5, 1, 64)), ("g_k", torch.bfloat16), ("g_k", None)))])
def test_refused(impl, args, name, change):
    with FakeTensorMode():
        args = args()
        args[name] = (change if change is None else _gpu(*args[name].shape, dtype=change) if isinstance(change, torch.dtype) else _gpu(*change, dtype=args[name].dtype))
        with pytest.raises(AssertionError):
            getattr(ops, impl)(**args)
