"""What qk_norm_rotary and cross_attention refuse, and the shapes they promise, without a GPU: tensors that have no memory, and the C entries' own checks."""
import ctypes
import math
from argparse import Namespace

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import lookupffn_amd
from lookupffn_amd import _lib, cross_attention, ops, qk_norm_rotary, rotary_table

P = 256                     # not null, 16-byte aligned, never read
BAD, UNSUPPORTED, OK = _lib.LFFN_ERR_BAD_ARG, _lib.LFFN_ERR_UNSUPPORTED, _lib.LFFN_OK


def _gpu(*shape, dtype=torch.float16):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def _attention_cases():
    q, k = (2, 3, 4, 64), (2, 5, 2, 64)
    yield "three dimensions", lambda: cross_attention(_gpu(2, 3, 64), _gpu(*k), _gpu(*k))
    yield "type", lambda: cross_attention(_gpu(*q, dtype=torch.float64), _gpu(*k), _gpu(*k))
    yield "whole numbers", lambda: cross_attention(_gpu(*q, dtype=torch.int32), _gpu(*k, dtype=torch.int32), _gpu(*k, dtype=torch.int32))
    yield "two types", lambda: cross_attention(_gpu(*q), _gpu(*k, dtype=torch.bfloat16), _gpu(*k, dtype=torch.bfloat16))
    yield "batch", lambda: cross_attention(_gpu(*q), _gpu(3, 5, 2, 64), _gpu(3, 5, 2, 64))
    yield "columns of keys", lambda: cross_attention(_gpu(*q), _gpu(2, 5, 2, 32), _gpu(2, 5, 2, 32))
    yield "values of another length", lambda: cross_attention(_gpu(*q), _gpu(*k), _gpu(2, 6, 2, 64))
    yield "heads", lambda: cross_attention(_gpu(*q), _gpu(2, 5, 3, 64), _gpu(2, 5, 3, 64))
    yield "no key heads", lambda: cross_attention(_gpu(*q), _gpu(2, 5, 0, 64), _gpu(2, 5, 0, 64))
    yield "odd columns", lambda: cross_attention(_gpu(2, 3, 4, 12), _gpu(2, 5, 2, 12), _gpu(2, 5, 2, 12))
    yield "many columns", lambda: cross_attention(_gpu(2, 3, 4, 136), _gpu(2, 5, 2, 136), _gpu(2, 5, 2, 136))
    yield "mask of numbers", lambda: cross_attention(_gpu(*q), _gpu(*k), _gpu(*k), _gpu(2, 5))
    yield "mask of another shape", lambda: cross_attention(_gpu(*q), _gpu(*k), _gpu(*k), _gpu(2, 3, dtype=torch.bool))
    for scale in (0.0, -1.0, math.inf, math.nan):
        yield f"scale {scale}", lambda scale=scale: cross_attention(_gpu(*q), _gpu(*k), _gpu(*k), scale=scale)


def _norm_cases():
    q, k = _gpu, lambda: _gpu(2, 5, 2, 64)
    x = lambda: _gpu(2, 3, 4, 64)  # noqa: E731
    table = lambda *shape, dtype=torch.float32: _gpu(*shape, dtype=dtype)  # noqa: E731
    whole = lambda *shape, dtype=torch.int64: _gpu(*shape, dtype=dtype)  # noqa: E731
    yield "three dimensions", lambda: qk_norm_rotary(_gpu(2, 3, 64))
    yield "two types", lambda: qk_norm_rotary(x(), _gpu(2, 5, 2, 64, dtype=torch.float32))
    yield "batch", lambda: qk_norm_rotary(x(), _gpu(3, 5, 2, 64))
    yield "odd columns", lambda: qk_norm_rotary(_gpu(2, 3, 4, 20))
    yield "many columns", lambda: qk_norm_rotary(_gpu(2, 3, 4, 264))
    yield "eps", lambda: qk_norm_rotary(x(), eps=-1.0)
    yield "eps nan", lambda: qk_norm_rotary(x(), eps=math.nan)
    yield "weight's length", lambda: qk_norm_rotary(x(), q_weight=_gpu(32, dtype=torch.float32))
    yield "weight's type", lambda: qk_norm_rotary(x(), q_weight=_gpu(64, dtype=torch.bfloat16))
    yield "key weight's length", lambda: qk_norm_rotary(x(), k(), k_weight=_gpu(32, dtype=torch.float32))
    yield "table's type", lambda: qk_norm_rotary(x(), table=table(9, 64, dtype=torch.float16))
    yield "table's columns", lambda: qk_norm_rotary(x(), table=table(9, 80))
    yield "table's odd columns", lambda: qk_norm_rotary(x(), table=table(9, 24))
    yield "no positions in the table", lambda: qk_norm_rotary(x(), table=table(0, 64))
    yield "table with a gradient", lambda: qk_norm_rotary(x(), table=table(9, 64).requires_grad_())
    yield "positions' type", lambda: qk_norm_rotary(x(), table=table(9, 64), q_positions=whole(2, 3, dtype=torch.int16))
    yield "positions' shape", lambda: qk_norm_rotary(x(), table=table(9, 64), q_positions=whole(3, 2))
    yield "key positions' shape", lambda: qk_norm_rotary(x(), k(), table=table(9, 64), k_positions=whole(3))


@pytest.mark.parametrize("case", [pytest.param(f, id=n) for n, f in (*_attention_cases(), *_norm_cases())])
def test_refusals(case):
    with FakeTensorMode(), pytest.raises(ValueError):
        case()


def test_cpu_tensors_and_tables():
    t = torch.zeros(1, 2, 2, 16)
    for call in (lambda: cross_attention(t, t, t), lambda: qk_norm_rotary(t)):
        with pytest.raises(RuntimeError, match="CPU tensor"):
            call()
    for positions, columns in ((0, 16), (4, 8), (4, 24)):
        with pytest.raises(ValueError):
            rotary_table(positions, columns)
    table = rotary_table(70000, 32)
    angle = 69999 * 10000.0 ** (-torch.arange(16, dtype=torch.float64) / 16)          # (far positions: angles in 64 bits)
    assert table.shape == (70000, 32) and table.dtype == torch.float32
    # 2^-24 is half a step of fp32 numbers below 1; the angles' own rounding in 64 bits is 2^-36
    assert (table[69999].double() - torch.cat((angle.cos(), angle.sin()))).abs().max() <= 2.0 ** -24


def test_shapes_while_tracing():
    with FakeTensorMode():
        q, k = _gpu(2, 3, 4, 64), _gpu(2, 5, 2, 64)
        assert cross_attention(q, k, k, _gpu(2, 5, dtype=torch.bool)).shape == q.shape
        a, b = qk_norm_rotary(q, k, table=_gpu(9, 64, dtype=torch.float32))
        assert a.shape == q.shape and b.shape == k.shape and a.dtype == q.dtype
        assert qk_norm_rotary(q)[1] is None
        out, lse = ops.cross_attention(q, k, k, None, 0.125, True)
        for of_q, of_k in ((True, True), (False, True), (True, False)):
            want = [t.shape for t, wanted in ((q, of_q), (k, of_k), (k, of_k)) if wanted]
            assert [t.shape for t in ops.cross_attention_bwd(q, k, k, None, 0.125, out, lse, out, of_q, of_k)] == want
        grads = ops.qk_norm_rotary_bwd(q, k, None, None, None, None, None, 1e-6, False, q, k, True, False)
        assert [t.shape for t in grads] == [q.shape, k.shape, (64,)] and grads[2].dtype == torch.float32


def _attention(**change):
    a = _lib.CrossAttention(q=P, k=P, v=P, B=2, q_len=3, k_len=5, heads=4, key_heads=2, columns=64, scale=0.125, format=2)
    a.q_strides[:], a.k_strides[:], a.v_strides[:] = (768, 256, 64), (640, 128, 64), (640, 128, 64)
    for name, value in change.items():
        if isinstance(value, tuple):
            getattr(a, name)[:] = value
        else:
            setattr(a, name, value)
    return ctypes.byref(a)


ATTENTION_REFUSALS = [(dict(B=-1), BAD), (dict(key_heads=0), BAD), (dict(heads=5), BAD), (dict(format=3), BAD), (dict(scale=0.0), BAD), (dict(scale=-1.0), BAD),
                      (dict(scale=math.nan), BAD), (dict(scale=math.inf), BAD), (dict(columns=60), UNSUPPORTED), (dict(columns=136), UNSUPPORTED),
                      (dict(q=None), BAD), (dict(k=None), BAD), (dict(v=None), BAD), (dict(q=P + 4), BAD), (dict(v=P + 8), BAD),
                      (dict(q_strides=(768, 252, 64)), BAD), (dict(k_strides=(640, -128, 64)), BAD), (dict(mask_stride=-1), BAD),
                      (dict(q_len=1 << 30), UNSUPPORTED), (dict(heads=1 << 17), UNSUPPORTED), (dict(B=1 << 29, q_len=1 << 20), UNSUPPORTED),
                      (dict(k_strides=(640, 1 << 27, 64)), UNSUPPORTED), (dict(q_strides=(768, 1 << 26, 64)), UNSUPPORTED)]


@pytest.mark.parametrize("change,code", ATTENTION_REFUSALS)
def test_attention_entries_check_their_arguments(change, code):
    lib, n = _lib.load(), ctypes.c_int64(7)
    a = _attention(**change)
    assert lib.lffn_cross_attention_workspace_bytes(a, ctypes.byref(n)) == code
    assert lib.lffn_cross_attention_bwd_workspace_bytes(a, ctypes.byref(n)) == code
    assert lib.lffn_cross_attention_fwd(a, P, None, None, 0, None) == code
    assert lib.lffn_cross_attention_bwd(a, P, P, P, P, P, P, P, 1 << 40, None) == code


def test_attention_entries_check_their_memory():
    lib, n = _lib.load(), ctypes.c_int64(0)
    a = _attention()
    assert lib.lffn_cross_attention_workspace_bytes(a, None) == BAD
    assert lib.lffn_cross_attention_fwd(None, P, None, None, 0, None) == BAD
    assert lib.lffn_cross_attention_fwd(a, None, None, None, 0, None) == BAD
    assert lib.lffn_cross_attention_fwd(a, P + 8, None, None, 0, None) == BAD
    assert lib.lffn_cross_attention_bwd_workspace_bytes(a, ctypes.byref(n)) == OK and n.value > 0
    for args in ((None, P, P, P, P, P, P, n.value), (P, None, P, P, P, P, P, n.value), (P, P, None, P, P, P, P, n.value), (P, P, P, P, P, None, P, n.value),
                 (P, P, P, P, None, P, P, n.value), (P, P, P, P, P, P, None, n.value), (P, P, P, P, P, P, P, n.value - 4), (P, P, P, P + 4, P, P, P, n.value)):
        assert lib.lffn_cross_attention_bwd(a, *args, None) == BAD
    # a few rows and many keys: shares of the keys need memory
    a = _attention(q_len=8, k_len=100000)
    assert lib.lffn_cross_attention_workspace_bytes(a, ctypes.byref(n)) == OK and n.value > 0
    assert lib.lffn_cross_attention_fwd(a, P, None, None, 0, None) == BAD
    assert lib.lffn_cross_attention_fwd(a, P, None, P, n.value - 4, None) == BAD
    # nothing to do
    assert lib.lffn_cross_attention_fwd(_attention(B=0, q=None, k=None, v=None), None, None, None, 0, None) == OK
    assert lib.lffn_cross_attention_fwd(_attention(q_len=0, q=None), None, None, None, 0, None) == OK
    assert lib.lffn_cross_attention_bwd(_attention(B=0, q=None, k=None, v=None), None, None, None, None, None, None, None, 0, None) == OK
    assert lib.lffn_cross_attention_bwd(_attention(), P, P, P, None, None, None, None, 0, None) == OK          # no gradient is wanted


def _norm(**change):
    a = _lib.QkNormRotary(q=P, k=P, table=P, B=2, q_len=3, k_len=5, q_heads=4, k_heads=2, columns=64, rotary=32, table_rows=9, eps=1e-6, format=1)
    a.q_strides[:], a.k_strides[:] = (768, 256, 64), (640, 128, 64)
    for name, value in change.items():
        if isinstance(value, tuple):
            getattr(a, name)[:] = value
        else:
            setattr(a, name, value)
    return ctypes.byref(a)


@pytest.mark.parametrize("change,code", [
    (dict(B=-1), BAD), (dict(format=-1), BAD), (dict(columns=60), UNSUPPORTED), (dict(columns=264), UNSUPPORTED), (dict(rotary=24), UNSUPPORTED),
    (dict(rotary=80), BAD), (dict(eps=-1.0), BAD), (dict(eps=math.nan), BAD), (dict(table=None), BAD), (dict(table=P + 4), BAD), (dict(table_rows=0), BAD),
    (dict(q=None), BAD), (dict(q=P + 2), BAD), (dict(q_weight=P + 4), BAD), (dict(k_strides=(640, 126, 64)), BAD), (dict(q_strides=(768, 256, -64)), BAD),
    (dict(q_heads=1 << 17), UNSUPPORTED), (dict(B=1 << 31), UNSUPPORTED)])
def test_norm_entries_check_their_arguments(change, code):
    lib, n = _lib.load(), ctypes.c_int64(7)
    a = _norm(**change)
    assert lib.lffn_qk_norm_rotary_fwd(a, P, P, None) == code
    assert lib.lffn_qk_norm_rotary_bwd_workspace_bytes(a, ctypes.byref(n)) == code
    assert lib.lffn_qk_norm_rotary_bwd(a, P, P, P, P, P, P, P, 1 << 40, None) == code


def test_norm_entries_check_their_memory():
    lib, n = _lib.load(), ctypes.c_int64(0)
    a = _norm()
    assert lib.lffn_qk_norm_rotary_fwd(a, None, P, None) == BAD
    assert lib.lffn_qk_norm_rotary_fwd(a, P, P + 8, None) == BAD
    assert lib.lffn_qk_norm_rotary_bwd_workspace_bytes(a, ctypes.byref(n)) == OK and n.value > 0
    for args in ((None, P, P, P, P, P, P, n.value), (P, None, P, P, P, P, P, n.value), (P, P, P, None, P, P, P, n.value), (P, P, P, P, P, P, None, n.value),
                 (P, P, P, P, P, P, P, n.value - 4), (P, P, P, P, P + 4, P, P, n.value)):
        assert lib.lffn_qk_norm_rotary_bwd(a, *args, None) == BAD
    assert lib.lffn_qk_norm_rotary_fwd(_norm(B=0, q=None, k=None), None, None, None) == OK
    assert lib.lffn_qk_norm_rotary_bwd(_norm(q_len=0, q=None, k=None), None, None, None, None, P, None, P, 64, None) == BAD       # a sum over no rows


def test_module_surface():
    config = Namespace(hidden_size=96, num_attention_heads=6, num_key_value_heads=2, attention_head_size=16, attention_probs_dropout_prob=0.1, layer_norm_eps=1e-5,
                       encoder_hidden_size=40, rotary_columns=16, max_position_embeddings=50)
    module = lookupffn_amd.CrossAttention(config)
    assert {n: tuple(p.shape) for n, p in module.state_dict().items()} == {
        "LayerNorm.weight": (96,), "LayerNorm.bias": (96,), "query.weight": (96, 96), "query.bias": (96,), "key.weight": (32, 40), "key.bias": (32,),
        "value.weight": (32, 40), "value.bias": (32,), "dense.weight": (96, 96), "dense.bias": (96,), "query_norm": (16,), "key_norm": (16,)}
    assert module.rotary.shape == (50, 16)
    with pytest.raises(ValueError):
        module(torch.zeros(1, 2, 96))


def test_more_threads_than_a_launch_has():
    """2^26 batches of one token: refused with the plan, before anything is launched."""
    lib, n = _lib.load(), ctypes.c_int64(0)
    a = _attention(B=1 << 26, q_len=1, heads=2)
    assert lib.lffn_cross_attention_workspace_bytes(a, ctypes.byref(n)) == UNSUPPORTED
    assert lib.lffn_cross_attention_fwd(a, P, None, None, 0, None) == UNSUPPORTED
    assert lib.lffn_cross_attention_bwd_workspace_bytes(a, ctypes.byref(n)) == UNSUPPORTED
    assert lib.lffn_cross_attention_bwd(a, P, P, P, P, P, P, P, 1 << 60, None) == UNSUPPORTED
    a = _norm(B=1 << 28, q_len=8)
    assert lib.lffn_qk_norm_rotary_fwd(a, P, P, None) == UNSUPPORTED
