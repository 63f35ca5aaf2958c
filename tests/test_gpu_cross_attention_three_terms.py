"""fp32 products in three bfloat16 terms (csrc/cross_attention.h): what is left out of one is at most 2^-22 of it."""
import pytest
import torch

from lookupffn_amd import cross_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _numbers():
    """Pairs whose lower terms are as large as terms that are cut off can be, as large as rounded ones can be, and any."""
    bits = [(0x3F80FFFF, 0x3F80FFFF), (0x3F80FFFF, 0x3F81FF80), (0x3F807F7F, 0x3F80FFFF), (0x3F80FF7F, 0x3F80FF7F), (0x3F80FF80, 0x3F80FF80), (0x3F817FFF, 0x3F80FFFF)]
    gen = torch.Generator().manual_seed(0)
    random = (torch.randint(0, 1 << 23, (500, 2), generator=gen) + 0x3F800000).tolist()
    return torch.tensor(bits + random, dtype=torch.int32).view(torch.float32).double().unbind(1)


def test_a_product():
    """The score a b beside the next fp32 number t as a second key's score, 1 t, which is exact: the result, the first key's weight, says by how much they differ."""
    a, b = _numbers()
    t = (a * b).float().double()
    q, k, v = torch.zeros(len(a), 5, 1, 8), torch.zeros(len(a), 2, 1, 8), torch.zeros(len(a), 2, 1, 8)
    q[:, :, 0, 0], q[:, :, 0, 1] = a.float()[:, None], 1
    k[:, 0, 0, 0], k[:, 1, 0, 1] = b.float(), t.float()
    v[:, 0] = 1
    scale = 2.0 ** 16
    out = cross_attention(q.to(DEV), k.to(DEV), v.to(DEV), scale=scale)[:, 0, 0, 0].double().cpu()
    off = torch.logit(out) / scale - (a * b - t)
    # beside what is left out, of a b below 4: the running sum, rounded where the last and largest product is added, and once before among numbers 2^-6 of it
    # (2^-24 and 2^-30 of 2^floor(log2 a b) and more: of a b); the exponent's, 2^-24 of a difference of at most 2^-5, and the weight's and result's roundings, 2^-21, both
    # by the scale
    bound = a * b * (2.0 ** -22 + 2.0 ** -24 + 2.0 ** -30) + 2.0 ** -20 / scale
    worst = (off.abs() / bound).max().item()
    assert worst <= 1, (worst, off.abs().max().item() / 2.0 ** -22)


def test_the_ends_of_the_range():
    """Numbers as large as fp32 has them, and below its normal ones, stay what they are."""
    most = torch.finfo(torch.float32).max
    q = torch.zeros(1, 6, 1, 8, device=DEV)
    k = torch.zeros(1, 1, 1, 8, device=DEV)
    for value in (most, -most, 1e-30, 2.0 ** -100):
        v = torch.full((1, 1, 1, 8), value, device=DEV)
        out = cross_attention(q, k, v)
        assert torch.equal(out, v.expand_as(out))
