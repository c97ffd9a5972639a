"""Limits of attention with score rules and over caches, refused before anything is launched (no GPU)."""
import ctypes

import pytest

from sparseattnfunctions_amd import _lib
from test_scored_host import INVALID, cached, scored


@pytest.mark.parametrize("over", [dict(cap=2e30), dict(cap=3e38), dict(cap=1e20, sm_scale=1e-20), dict(cap=1e29, sm_scale=1e-10),
                                  dict(cap=0.9e-30)], ids=str)
def test_caps_out_of_range(over):
    lib = _lib.load()
    n = (ctypes.c_int64 * 3)()
    assert lib.sa_attn_scored_sizes(scored(**over), n) == INVALID
    assert lib.sa_attn_scored_fwd(scored(**over), None) == INVALID
    assert lib.sa_attn_scored_bwd(scored(**over), None) == INVALID
    assert lib.sa_attn_cached_workspace(cached(**over), ctypes.byref(ctypes.c_int64())) == INVALID
    assert lib.sa_attn_cached_fwd(cached(**over), None) == INVALID


@pytest.mark.parametrize("over", [dict(cap=0.9e30), dict(cap=1e10, sm_scale=1e-20), dict(cap=1e-20)], ids=str)
def test_caps_in_range(over):
    lib = _lib.load()
    assert lib.sa_attn_scored_sizes(scored(**over), (ctypes.c_int64 * 3)()) == 0
    assert lib.sa_attn_cached_workspace(cached(**over), ctypes.byref(ctypes.c_int64())) == 0


@pytest.mark.parametrize("over", [dict(B=1 << 16, H=1 << 16, Hk=1 << 16, Ln=1), dict(B=1 << 15, H=1 << 17, Hk=1 << 17, Ln=1, Lp=0)],
                         ids=str)
def test_many_sequences_and_key_heads(over):
    lib = _lib.load()
    n = ctypes.c_int64()
    assert lib.sa_attn_cached_workspace(cached(**over), ctypes.byref(n)) == _lib.SA_ERR_UNSUPPORTED
    assert lib.sa_attn_cached_fwd(cached(**over), None) == _lib.SA_ERR_UNSUPPORTED
