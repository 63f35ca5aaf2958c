"""Long caches and queries that lie heads first, heads far apart: read where they are."""
import pytest
import torch

import lookupffn_amd
from lookupffn_amd import cross_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True, params=["host", "python"])
def either_path(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(lookupffn_amd._lib, "loaded_host", False)
    else:
        assert lookupffn_amd._lib.host()


def _randn(*shape, dtype, seed):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def test_a_long_cache_that_lies_heads_first_is_read_in_place():
    """Heads of a gigabyte of keys far apart: nothing is copied (the kernels reach every key head by 64 bits)."""
    B, Hk, keys, D = 1, 16, 1 << 18, 128
    cache = torch.empty(2, B, Hk, keys, D, dtype=torch.bfloat16, device=DEV)
    cache.normal_(generator=torch.Generator(device=DEV).manual_seed(0))
    k, v = (t.permute(0, 2, 1, 3) for t in cache)
    q = _randn(B, 1, Hk, D, dtype=torch.bfloat16, seed=1)
    with torch.no_grad():
        cross_attention(q, k, v)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out = cross_attention(q, k, v)
        assert torch.cuda.max_memory_allocated() - before < 64 << 20
        for h in (0, Hk - 1):
            alone = cross_attention(q[:, :, h:h + 1], *(t[:, h:h + 1].permute(0, 2, 1, 3) for t in cache))
            # (other shares of the keys: fp32 sums, one rounding)
            assert ((out[:, :, h:h + 1].double() - alone.double()).abs() <= 2.0 ** -8 * alone.double().abs() + 2.0 ** -20).all()


@pytest.mark.parametrize("Hk", [16, 4])
def test_long_queries_that_lie_heads_first_are_read_in_place(Hk):
    """A gigabyte of them, a key head's own within 32 bits."""
    L, H, D, keys = 1 << 18, 16, 128, 70
    base = torch.empty(1, H, L, D, dtype=torch.bfloat16, device=DEV)
    base.normal_(generator=torch.Generator(device=DEV).manual_seed(0))
    q = base.permute(0, 2, 1, 3)
    k, v = (_randn(1, keys, Hk, D, dtype=torch.bfloat16, seed=s) for s in (1, 2))
    with torch.no_grad():
        cross_attention(q[:, :64], k, v)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out = cross_attention(q, k, v)
        assert torch.cuda.max_memory_allocated() - before < out.nbytes + (64 << 20)
        some = slice(L - 300, L)
        # (the same kernel, tiles and order: the same bits)
        assert torch.equal(out[:, some], cross_attention(q.contiguous(), k, v)[:, some])
