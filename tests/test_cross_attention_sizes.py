"""Sizes beyond what the C entries of cross_attention count in: refused with the plan, whatever else is empty.  Without a GPU, each in a process of its own: an entry must
not end it."""
import subprocess
import sys

import pytest

CALL = """
import ctypes, sys
sys.path.insert(0, "tests")
from test_cross_attention_arguments import P, _attention
from lookupffn_amd import _lib
lib, n = _lib.load(), ctypes.c_int64(0)
a = _attention(**{change})
print([lib.lffn_cross_attention_workspace_bytes(a, ctypes.byref(n)), lib.lffn_cross_attention_kept_bytes(a, ctypes.byref(n)),
       lib.lffn_cross_attention_bwd_workspace_bytes(a, ctypes.byref(n)), lib.lffn_cross_attention_fwd(a, P, None, P, 1 << 60, None),
       lib.lffn_cross_attention_bwd(a, P, P, P, P, P, P, P, 1 << 60, None)])
"""


# key heads that are a multiple of 2^32, or more than there are query heads; products of batches, heads and tiles of keys that pass 64 bits
@pytest.mark.parametrize("change", [dict(heads=0, key_heads=1 << 40), dict(heads=0, key_heads=(1 << 32) + 2), dict(heads=0, key_heads=1 << 17),
                                    dict(heads=65536, key_heads=65536, q_len=0, B=(1 << 30) - 1, k_len=(1 << 30) - 1),
                                    dict(heads=65536, key_heads=65536, q_len=0, B=1 << 25, k_len=1 << 29),
                                    dict(heads=1 << 16, key_heads=1, q_len=1 << 20)])
def test_refused(change):
    from lookupffn_amd import _lib
    out = subprocess.run([sys.executable, "-c", CALL.format(change=change)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    assert eval(out.stdout) == [_lib.LFFN_ERR_UNSUPPORTED] * 5


@pytest.mark.parametrize("change", [dict(heads=0, key_heads=4, q=None), dict(q_len=0, q=None), dict(k_len=0, k=None, v=None)])
def test_nothing_to_do_is_none_of_them(change):
    import ctypes

    from lookupffn_amd import _lib
    from test_cross_attention_arguments import _attention
    lib, n = _lib.load(), ctypes.c_int64(0)
    a = _attention(**change)
    for entry in (lib.lffn_cross_attention_workspace_bytes, lib.lffn_cross_attention_kept_bytes, lib.lffn_cross_attention_bwd_workspace_bytes):
        assert entry(a, ctypes.byref(n)) == _lib.LFFN_OK
