"""The workspaces of linear_cross_entropy are what its documentation says, from the C entries that report them; without a GPU."""
import ctypes

import pytest

from lookupffn_amd import _lib

P = 256
MB, GB = 1 << 20, 1 << 30


def _up(n, to):
    return (n + to - 1) // to * to


def _bytes(query, tokens, vocabulary, columns, format, reduction=1):
    a = _lib.LinearCrossEntropy(hidden=P, weight=P, labels=P, tokens=tokens, vocabulary=vocabulary, columns=columns, hidden_stride=columns, weight_stride=columns, format=format, labels_64=1,
                                reduction=reduction)
    n = ctypes.c_int64(0)
    assert getattr(_lib.load(), query)(ctypes.byref(a), ctypes.byref(n)) == _lib.LFFN_OK
    return n.value


SIZES = [(16384, 50265, 768), (32768, 50265, 512), (130000, 50265, 64), (260000, 50265, 64), (131072, 1000, 4096), (300000, 1000, 1024), (1000, 1 << 22, 64), (1 << 20, 300, 64), (1, 300, 1024),
         (70, 40, 8)]


@pytest.mark.parametrize("format", [0, 1, 2])
@pytest.mark.parametrize("tokens,vocabulary,columns", SIZES)
def test_workspaces(tokens, vocabulary, columns, format):
    size = 4 if format == 0 else 2
    rows = _up(tokens, 256) * _up(columns, 128) * size
    weights = _up(vocabulary, 256) * (_up(columns, 32) * 4 + 8) if format == 0 else vocabulary * 4
    few = 64 * _up(tokens, 256) + 12 * vocabulary + 64 * 1024          # numbers by token and by entry, alignment
    tokens_ = _up(tokens, 256)
    forward = _bytes("lffn_linear_cross_entropy_workspace_bytes", tokens, vocabulary, columns, format)
    tiles = _up(vocabulary, 256) // 256
    parts = max(8 * tokens_ * tiles, 8 * tokens_ * 256 if tokens <= 64 else 0)
    assert forward <= rows + weights + parts + few
    assert forward >= 8 * tokens * tiles or tokens <= 64
    for reduction in (0, 1):
        backward = _bytes("lffn_linear_cross_entropy_bwd_workspace_bytes", tokens, vocabulary, columns, format, reduction)
        # (2048 entries and 64 more of every token, in 16 bits or two terms, if that is more than 1 GB)
        least = tokens_ * (min(2048, _up(vocabulary, 256)) + 64) * size
        d = least if least > GB else min(GB, tokens_ * (_up(vocabulary, 256) + 64) * size)
        sums = max(256 * MB, tokens * columns * 4)
        assert backward <= rows + weights + d + sums + 512 * MB + few
        assert backward >= rows + d
    assert least <= tokens_ * (4300 if size == 2 else 8500)


def test_few_tokens_keep_their_logits_where_they_are_no_more_than_the_weights():
    for format, size in ((0, 4), (2, 2)):
        for tokens, columns in ((64, 768), (64, 64), (64, 128), (64, 120), (19, 768), (65, 768)):
            kept = _bytes("lffn_linear_cross_entropy_kept_bytes", tokens, 50265, columns, format)
            logits = tokens * _up(50265, 32) * 4
            few = 32 + tokens * 4 + 16 + _up(tokens, 256) * 12
            assert kept <= few + (logits if tokens <= 64 and tokens * 4 <= columns * size else 0)
            assert kept <= 20 * tokens + 12 * 256 + 64 or logits <= 50272 * columns * size
