"""What embedding, layer_norm and linear_cross_entropy refuse, and the shapes they promise, without a GPU: tensors that have no memory, and the C entries' own checks."""
import ctypes
import math
from argparse import Namespace

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import lookupffn_amd
from lookupffn_amd import _lib, embedding, layer_norm, linear_cross_entropy, ops

P = 256                     # not null, 16-byte aligned, never read
BAD, UNSUPPORTED, OK = _lib.LFFN_ERR_BAD_ARG, _lib.LFFN_ERR_UNSUPPORTED, _lib.LFFN_OK


def _gpu(*shape, dtype=torch.float16):
    return torch.empty(shape, dtype=dtype, device="cuda")


def _ids(*shape, dtype=torch.int64):
    return _gpu(*shape, dtype=dtype)


def _cases():
    w = lambda *s, **k: _gpu(*(s or (90, 64)), **k)  # noqa: E731
    yield "numbers of no whole type", lambda: embedding(_gpu(3), w())
    yield "short numbers", lambda: embedding(_ids(3, dtype=torch.int16), w())
    yield "flags", lambda: embedding(_ids(3, dtype=torch.bool), w())
    yield "table of three dimensions", lambda: embedding(_ids(3), w(3, 90, 64))
    yield "table's type", lambda: embedding(_ids(3), w(dtype=torch.float64))
    yield "table of whole numbers", lambda: embedding(_ids(3), w(dtype=torch.int32))
    yield "no columns", lambda: embedding(_ids(3), w(90, 0))
    yield "many columns", lambda: embedding(_ids(3), w(2, (1 << 20) + 1))
    yield "many rows", lambda: embedding(_ids(3), w((1 << 31) - 1, 1))
    yield "many tokens", lambda: embedding(_ids(1 << 31), w())
    for padding in (90, -91):
        yield f"padding {padding}", lambda padding=padding: embedding(_ids(3), w(), padding_idx=padding)
    yield "padding of no rows", lambda: embedding(_ids(3), w(0, 64), padding_idx=0)
    for scale in (math.inf, math.nan):
        yield f"scale {scale}", lambda scale=scale: embedding(_ids(3), w(), scale=scale)

    x = lambda *s, **k: _gpu(*(s or (5, 64)), **k)  # noqa: E731
    yield "no dimension", lambda: layer_norm(x().sum())
    yield "norm's type", lambda: layer_norm(x(dtype=torch.float64))
    yield "norm of whole numbers", lambda: layer_norm(x(dtype=torch.int64))
    yield "norm of no columns", lambda: layer_norm(x(5, 0))
    yield "norm of many columns", lambda: layer_norm(x(1, (1 << 24) + 1))
    yield "norm of many rows", lambda: layer_norm(x(1 << 24, 1))
    yield "weight's length", lambda: layer_norm(x(), _gpu(32))
    yield "weight's dimensions", lambda: layer_norm(x(), _gpu(1, 64))
    yield "weight's type", lambda: layer_norm(x(), _gpu(64, dtype=torch.bfloat16))
    yield "bias's length", lambda: layer_norm(x(), _gpu(64), _gpu(65))
    yield "bias's type", lambda: layer_norm(x(), None, _gpu(64, dtype=torch.float64))
    yield "weight and bias of two types", lambda: layer_norm(x(), _gpu(64), _gpu(64, dtype=torch.float32))
    for eps in (-1.0, math.nan):
        yield f"eps {eps}", lambda eps=eps: layer_norm(x(), eps=eps)

    y = lambda *s, **k: _ids(*(s or (5,)), **k)  # noqa: E731
    loss = linear_cross_entropy
    yield "loss without tokens' dimension", lambda: loss(_gpu(4).sum(), w(), None, y())
    yield "loss's type", lambda: loss(x(dtype=torch.float64), w(dtype=torch.float64), None, y())
    yield "odd columns", lambda: loss(x(5, 60), w(90, 60), None, y())
    yield "loss of no columns", lambda: loss(x(5, 0), w(90, 0), None, y())
    yield "loss of many columns", lambda: loss(x(5, 65544), w(9, 65544), None, y())
    yield "weight's columns", lambda: loss(x(), w(90, 72), None, y())
    yield "loss's weight's type", lambda: loss(x(), w(dtype=torch.float32), None, y())
    yield "loss's weight's dimensions", lambda: loss(x(), w(1, 90, 64), None, y())
    yield "no vocabulary", lambda: loss(x(), w(0, 64), None, y())
    yield "large vocabulary", lambda: loss(x(5, 8), w((1 << 22) + 1, 8), None, y())
    yield "loss's bias's length", lambda: loss(x(), w(), _gpu(64), y())
    yield "loss's bias's type", lambda: loss(x(), w(), _gpu(90, dtype=torch.bfloat16), y())
    yield "labels' shape", lambda: loss(x(), w(), None, y(4))
    yield "labels' dimensions", lambda: loss(x(), w(), None, y(5, 1))
    yield "labels' type", lambda: loss(x(), w(), None, y(dtype=torch.int16))
    yield "labels of numbers", lambda: loss(x(), w(), None, _gpu(5, dtype=torch.float32))
    yield "labels of shares", lambda: loss(x(), w(), None, _gpu(5, 90, dtype=torch.float32))
    yield "many labelled tokens", lambda: loss(x((1 << 24) + 1, 8), w(9, 8), None, y((1 << 24) + 1))
    yield "many numbers", lambda: loss(x((1 << 20) + 1, 4096), w(9, 4096), None, y((1 << 20) + 1))
    yield "reduction", lambda: loss(x(), w(), None, y(), reduction="average")
    yield "no reduction", lambda: loss(x(), w(), None, y(), reduction=None)
    yield "ignore_index", lambda: loss(x(), w(), None, y(), ignore_index=1.0)
    yield "large ignore_index", lambda: loss(x(), w(), None, y(), ignore_index=1 << 63)


@pytest.mark.parametrize("case", [pytest.param(f, id=n) for n, f in _cases()])
def test_refusals(case):
    with FakeTensorMode(), pytest.raises(ValueError):
        case()


def test_cpu_tensors():
    ids, t = torch.zeros(3, dtype=torch.int64), torch.zeros(3, 8)
    for call in (lambda: embedding(ids, t), lambda: layer_norm(t), lambda: linear_cross_entropy(t, t, None, ids)):
        with pytest.raises(RuntimeError, match="CPU tensor"):
            call()


def test_shapes_while_tracing():
    with FakeTensorMode():
        w = _gpu(90, 64, dtype=torch.bfloat16)
        out = embedding(_ids(2, 3, dtype=torch.int32), w, padding_idx=-1)
        assert out.shape == (2, 3, 64) and out.dtype == w.dtype
        assert ops.embedding_bwd(_ids(6), _gpu(6, 64), 90, 1.0, -1).shape == (90, 64)
        assert layer_norm(out, None, _gpu(64, dtype=torch.float32)).shape == out.shape
        x = _gpu(6, 64)
        assert [t.shape for t in ops.layer_norm_rows_bwd(x, _gpu(64), None, _gpu(6, 2, dtype=torch.float32), x, True, True, False)] == [(6, 64), (64,)]
        for reduction in ops.REDUCTIONS:
            loss = linear_cross_entropy(out, w, None, _ids(2, 3), reduction=reduction)
            assert loss.shape == ((2, 3) if reduction == "none" else ()) and loss.dtype == torch.float32
        args = (x, _gpu(90, 64), _gpu(90, dtype=torch.float32), _ids(6), -100, 1)
        loss, kept = ops.linear_cross_entropy(*args, True)
        for wanted in ((True, True, True), (False, True, False), (True, False, True)):
            got = ops.linear_cross_entropy_bwd(*args, kept, loss, *wanted)
            assert [(t.shape, t.dtype) for t in got] == [(t.shape, t.dtype) for t, use in zip(args, wanted) if use]


def _loss_args():
    return dict(hidden=_gpu(6, 64), weight=_gpu(90, 64), bias=_gpu(90), labels=_ids(6), ignore_index=-100, reduction=1)


OF_LOSS = [("hidden", (6, 32)), ("hidden", (5, 64)), ("hidden", (1, 6, 64)), ("hidden", torch.float32), ("weight", (90, 32)), ("weight", (90 * 64,)), ("weight", torch.bfloat16),
           ("bias", (91,)), ("bias", torch.bfloat16), ("labels", (7,)), ("labels", (6, 1)), ("labels", torch.int16), ("reduction", 3)]
OF_NORM = [("x", (5, 64, 1)), ("x", torch.float64), ("weight", (63,)), ("weight", torch.bfloat16), ("weight", torch.float32), ("bias", (1, 64)), ("bias", torch.float64)]


@pytest.mark.parametrize("impl,args,name,change", [
    *(("_linear_cross_entropy_impl", lambda: dict(_loss_args(), keep=True), *c) for c in OF_LOSS),
    *(("_linear_cross_entropy_bwd_impl", lambda: dict(_loss_args(), kept=_gpu(ops._loss_kept_bytes(_gpu(6, 64), _gpu(90, 64)), dtype=torch.uint8), g=_gpu(dtype=torch.float32), of_hidden=True, of_weight=True,
                                                      of_bias=True), *c) for c in OF_LOSS + [("kept", (64,)), ("kept", torch.int8), ("g", (6,)), ("g", torch.float16), ("bias", None)]),
    *(("_layer_norm_impl", lambda: dict(x=_gpu(5, 64), weight=_gpu(64), bias=_gpu(64), eps=1e-5, keep=True), *c) for c in OF_NORM),
    *(("_layer_norm_rows_bwd_impl", lambda: dict(x=_gpu(5, 64), weight=_gpu(64), bias=_gpu(64), stats=_gpu(5, 2, dtype=torch.float32), g=_gpu(5, 64), of_x=True, of_weight=True, of_bias=True),
       *c) for c in OF_NORM + [("stats", (4, 2)), ("stats", torch.float16), ("g", (5, 63)), ("g", torch.float32), ("weight", None), ("bias", None)]),
    *(("_embedding_impl", lambda: dict(ids=_ids(6), weight=_gpu(90, 64), scale=1.0, padding=-1), *c)
      for c in (("ids", (6, 1)), ("ids", torch.float32), ("weight", (90, 64, 1)), ("weight", torch.float64), ("padding", 90), ("padding", -2))),
    *(("_embedding_bwd_impl", lambda: dict(ids=_ids(6), g=_gpu(6, 64), rows=90, scale=1.0, padding=-1), *c)
      for c in (("ids", (6, 1)), ("ids", torch.int16), ("g", (5, 64)), ("g", (6, 64, 1)), ("g", torch.float64), ("padding", 90), ("rows", -1)))])
def test_operators_check_what_they_are_given(impl, args, name, change):
    with FakeTensorMode():
        args = args()
        if isinstance(change, torch.dtype):
            change = _gpu(*args[name].shape, dtype=change)
        elif isinstance(change, tuple):
            change = _gpu(*change, dtype=args[name].dtype)
        args[name] = change
        with pytest.raises((AssertionError, RuntimeError)):
            getattr(ops, impl)(**args)


def _struct(kind, base, **change):
    return ctypes.byref(kind(**dict(base, **change)))


def test_c_entries_check_their_arguments():
    lib, n = _lib.load(), ctypes.c_int64(0)
    embed = dict(ids=P, weight=P, tokens=5, rows=90, columns=64, stride=64, padding=-1, scale=1.0, format=2, ids_64=1)
    of = lambda **c: _struct(_lib.Embedding, embed, **c)  # noqa: E731
    fwd = lambda a, out=P: lib.lffn_embedding_fwd(a, out, None)  # noqa: E731
    for bad in (dict(ids=None), dict(weight=None), dict(format=3), dict(format=-1), dict(tokens=-1), dict(rows=-1), dict(columns=0), dict(stride=-1)):
        assert fwd(of(**bad)) == BAD, bad
    assert fwd(of(), None) == BAD and fwd(None) == BAD
    for much in (dict(tokens=1 << 31), dict(rows=(1 << 31) - 1), dict(columns=(1 << 20) + 1)):
        assert fwd(of(**much)) == UNSUPPORTED, much
    assert fwd(of(tokens=0, ids=None), None) == OK
    assert lib.lffn_embedding_bwd_workspace_bytes(of(), ctypes.byref(n)) == OK and n.value > 0
    assert lib.lffn_embedding_bwd_workspace_bytes(of(), None) == BAD
    bwd = lambda a, g=P, grad=P, ws=P, size=n.value: lib.lffn_embedding_bwd(a, g, grad, ws, size, None)  # noqa: E731
    assert bwd(of(), g=None) == BAD and bwd(of(), grad=None) == BAD and bwd(of(), ws=None) == BAD and bwd(of(), ws=P + 8) == BAD and bwd(of(), size=n.value - 1) == BAD
    assert bwd(of(), grad=P + 8) == BAD and bwd(of(rows=0)) == OK

    norm = dict(x=P, weight=P, bias=P, rows=5, columns=64, stride=64, eps=1e-5, format=2, weight_f32=1)
    of = lambda **c: _struct(_lib.LayerNormRows, norm, **c)  # noqa: E731
    fwd = lambda a, out=P: lib.lffn_layer_norm_rows_fwd(a, out, None, None)  # noqa: E731
    for bad in (dict(x=None), dict(format=3), dict(rows=-1), dict(columns=0), dict(stride=-1), dict(eps=-1.0), dict(eps=math.nan)):
        assert fwd(of(**bad)) == BAD, bad
    assert fwd(of(), None) == BAD and fwd(None) == BAD and fwd(of(rows=0, x=None), None) == OK
    for much in (dict(rows=1 << 24), dict(columns=(1 << 24) + 1)):
        assert fwd(of(**much)) == UNSUPPORTED, much
    assert lib.lffn_layer_norm_rows_bwd_workspace_bytes(of(), ctypes.byref(n)) == OK and n.value > 0
    bwd = lambda a, stats=P, g=P, gw=P, ws=P, size=n.value: lib.lffn_layer_norm_rows_bwd(a, stats, g, P, gw, None, ws, size, None)  # noqa: E731
    assert bwd(of(), stats=None) == BAD and bwd(of(), g=None) == BAD and bwd(of(), ws=None) == BAD and bwd(of(), ws=P + 4) == BAD and bwd(of(), size=n.value - 1) == BAD

    loss = dict(hidden=P, weight=P, bias=P, labels=P, tokens=5, vocabulary=90, columns=64, hidden_stride=64, weight_stride=64, ignore_index=-100, format=2, bias_format=0, labels_64=1,
                reduction=1)
    of = lambda **c: _struct(_lib.LinearCrossEntropy, loss, **c)  # noqa: E731
    assert lib.lffn_linear_cross_entropy_workspace_bytes(of(), ctypes.byref(n)) == OK and n.value > 0
    fwd = lambda a, out=P, kept=None, ws=P, size=n.value: lib.lffn_linear_cross_entropy_fwd(a, out, kept, ws, size, None)  # noqa: E731
    for bad in (dict(hidden=None), dict(weight=None), dict(labels=None), dict(format=3), dict(bias_format=3), dict(reduction=3), dict(reduction=-1), dict(tokens=-1), dict(vocabulary=0),
                dict(columns=0), dict(weight=P + 8), dict(hidden=P + 2), dict(hidden_stride=65), dict(weight_stride=68), dict(weight_stride=56), dict(hidden_stride=-8)):
        assert fwd(of(**bad)) == BAD, bad
    for much in (dict(columns=60), dict(columns=65544, weight_stride=65544), dict(tokens=(1 << 24) + 1), dict(vocabulary=(1 << 22) + 1), dict(weight_stride=(1 << 22) + 8),
                 dict(tokens=1 << 24, columns=512, weight_stride=512)):
        assert fwd(of(**much)) == UNSUPPORTED, much
    assert fwd(of(), out=None) == BAD and fwd(of(), ws=None) == BAD and fwd(of(), ws=P + 8) == BAD and fwd(of(), size=n.value - 1) == BAD and fwd(of(), kept=P + 4) == BAD
    for format, dtype in ((0, torch.float32), (2, torch.bfloat16)):
        for tokens, vocabulary, columns in ((5, 90, 64), (0, 90, 64), (1, 90, 8), (32, 90, 64), (33, 90, 64), (32, 33, 1216), (32, 33, 1224), (32, 33, 2424), (32, 33, 2432), (64, 1, 608),
                                            (64, 1, 616), (64, 1, 1208), (64, 1, 1216), (64, 1, 128), (64, 1, 120), (65, 90, 512), (255, 90, 64), (256, 90, 64), (257, 90, 64), (70000, 90, 64)):
            a = of(tokens=tokens, vocabulary=vocabulary, columns=columns, hidden_stride=columns, weight_stride=columns, format=format)
            want = ops._loss_kept_bytes(torch.empty(tokens, columns, dtype=dtype, device="meta"), torch.empty(vocabulary, columns, dtype=dtype, device="meta"))
            assert lib.lffn_linear_cross_entropy_kept_bytes(a, ctypes.byref(n)) == OK and n.value == want, (tokens, vocabulary, columns, format)
    assert lib.lffn_linear_cross_entropy_bwd_workspace_bytes(of(), ctypes.byref(n)) == OK and n.value > 0
    bwd = lambda a, kept=P, g=P, gh=P, gw=P, gb=P, ws=P, size=n.value: lib.lffn_linear_cross_entropy_bwd(a, kept, g, gh, gw, gb, ws, size, None)  # noqa: E731
    assert bwd(of(), kept=None) == BAD and bwd(of(), g=None) == BAD and bwd(of(), gw=None) == BAD and bwd(of(), gh=P + 8) == BAD and bwd(of(), gw=P + 8) == BAD
    assert bwd(of(), ws=None) == BAD and bwd(of(), size=n.value - 1) == BAD and bwd(of(tokens=0)) == UNSUPPORTED


def test_modules_parameters():
    config = Namespace(hidden_size=64, num_attention_heads=1, attention_head_size=64, attention_probs_dropout_prob=0.0, hidden_dropout_prob=0.1, layer_norm_eps=1e-5, num_hidden_layers=1,
                       vocab_size=300, max_position_embeddings=40, type_vocab_size=2, pad_token_id=1, ffn_num_table=8, ffn_table_size=256, projection_type="bh4", block_size=1)
    model = lookupffn_amd.LookupForMaskedLM(config)
    names = {n: tuple(p.shape) for n, p in model.named_parameters()}
    assert {n: s for n, s in names.items() if n.startswith("head.")} == {"head.dense.weight": (64, 64), "head.dense.bias": (64,), "head.LayerNorm.weight": (64,), "head.LayerNorm.bias": (64,),
                                                                        "head.bias": (300,)}
    # (one table for both ends) what the encoder had it has
    plain = lookupffn_amd.Lookup(config)
    assert {n[8:] for n in names if n.startswith("encoder.")} == {n for n, _ in plain.named_parameters()}
    assert model.encoder.embeddings.kernels and not plain.embeddings.kernels
    # on the CPU the embeddings are torch's, as they were
    ids = torch.randint(0, 300, (2, 5))
    emb = model.encoder.embeddings.eval()
    want = emb.LayerNorm(emb.word_embeddings(ids) + emb.token_type_embeddings(ids * 0) + emb.position_embeddings(torch.arange(5).expand(2, 5) + 2))
    assert torch.equal(emb(ids, ids * 0, torch.arange(5).expand(2, 5)), want)
