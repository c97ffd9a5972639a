"""Rotary frequencies and what `sa_rotary_*` and `sa_block_sparse_bwd` refuse, without a GPU."""
import ctypes
import math

import pytest
import torch

from sparseattnfunctions_amd import _lib
from sparseattnfunctions_amd.utils.rotary import apply_rotary, rotary_frequencies, rotary_table


def test_frequencies():
    f, m = rotary_frequencies(8, 10000.0)
    assert m == 1.0 and f == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-15)
    f, m = rotary_frequencies(8, 10000.0, {"type": "linear", "factor": 4})
    assert m == 1.0 and f == pytest.approx([0.25, 0.025, 0.0025, 0.00025], rel=1e-15)
    # NTK: the fastest pair stays, the slowest is stretched by the factor
    f, m = rotary_frequencies(64, 10000.0, {"type": "ntk", "factor": 4})
    plain, _ = rotary_frequencies(64, 10000.0)
    assert m == 1.0 and f[0] == 1.0 and f[-1] == pytest.approx(plain[-1] / 4, rel=1e-12)
    assert rotary_frequencies(2, 10000.0, {"type": "ntk", "factor": 4})[0] == [1.0]
    # YaRN: many turns over the trained length keep their frequency, few are divided
    f, m = rotary_frequencies(128, 10000.0, {"type": "yarn", "factor": 8, "original_length": 4096})
    plain, _ = rotary_frequencies(128, 10000.0)
    assert m == pytest.approx(0.1 * math.log(8) + 1)
    for a, b in zip(f, plain):
        turns = 4096 * b / (2 * math.pi)
        if turns >= 32:
            assert a == b
        elif turns <= 1:
            assert a == pytest.approx(b / 8)
        else:
            assert b / 8 < a < b
    assert rotary_frequencies(128, 10000.0, {"type": "yarn", "factor": 1, "original_length": 4096})[0] == pytest.approx(plain)


@pytest.mark.parametrize("bad", [
    dict(dims=0), dict(dims=7), dict(dims=-2), dict(dims=8, theta=0.0), dict(dims=8, theta=math.inf),
    dict(dims=8, scaling={"type": "cubic", "factor": 2}), dict(dims=8, scaling={"type": "linear"}),
    dict(dims=8, scaling={"type": "linear", "factor": 0.5}), dict(dims=8, scaling={"type": "linear", "factor": math.nan}),
    dict(dims=8, scaling={"type": "linear", "factor": 2, "beta_fast": 3}), dict(dims=8, scaling={"type": "yarn", "factor": 2}),
    dict(dims=8, scaling={"factor": 2}), dict(dims=8, scaling={"type": "yarn", "factor": 2, "original_length": 10,
                                                                "beta_fast": 1, "beta_slow": 1})], ids=str)
def test_refused_frequencies(bad):
    with pytest.raises(ValueError):
        rotary_frequencies(**bad)


def test_no_cpu_path():
    with pytest.raises(ValueError):
        rotary_table(torch.arange(4), 64)
    q = torch.zeros(1, 1, 4, 64)
    with pytest.raises(ValueError):
        apply_rotary(q, q, torch.zeros(4, 32, 2))


def test_c_argument_checks():
    lib = _lib.load()
    p = ctypes.c_void_p(256)  # never read: the checks come first
    one = (ctypes.c_int32 * 1)(32)
    freq = (ctypes.c_double * 32)(*([1.0] * 32))
    fac = (ctypes.c_double * 1)(1.0)

    def table(pos=p, kind=0, L=4, axes=1, pairs=one, f=freq, m=fac, out=p):
        return lib.sa_rotary_table(pos, kind, _lib.i64(0, 1), L, axes, pairs, f, m, out, None)

    nan = (ctypes.c_double * 32)(*([math.nan] * 32))
    for bad in (dict(pos=None), dict(kind=9), dict(L=0), dict(axes=0), dict(axes=5), dict(pairs=(ctypes.c_int32 * 1)(129)),
                dict(pairs=(ctypes.c_int32 * 1)(0)), dict(f=nan), dict(m=nan), dict(out=None), dict(out=ctypes.c_void_p(4))):
        assert table(**bad) == _lib.SA_ERR_INVALID, bad

    st = _lib.i64(*range(0, 120, 10))

    def turn(dtype=0, q=p, qo=p, k=p, ko=p, B=1, H=1, Hk=1, L=4, D=64, t=p, rows=8, pairs=32, r=None, skip=0):
        return lib.sa_rotary_apply(dtype, q, qo, k, ko, st, B, H, Hk, L, D, t, rows, pairs, r, 0, skip, 0, 0, None)

    for bad in (dict(dtype=3), dict(q=None), dict(ko=None), dict(B=0), dict(H=0), dict(Hk=0), dict(L=0), dict(D=0), dict(D=258),
                dict(t=None), dict(rows=0), dict(pairs=0), dict(pairs=33), dict(skip=-1), dict(skip=5), dict(rows=3),
                dict(r=p, skip=1), dict(H=65535), dict(t=ctypes.c_void_p(4))):
        assert turn(**bad) == _lib.SA_ERR_INVALID, bad

    n = ctypes.c_int64(0)
    assert lib.sa_block_sparse_bwd_workspace(2, 3, 65, ctypes.byref(n)) == 0 and n.value == 2 * 3 * 2 * 128 * 4
    assert lib.sa_block_sparse_bwd_workspace(0, 3, 65, ctypes.byref(n)) == _lib.SA_ERR_INVALID
    strides = [0, 0, 64] * 8

    def bwd(dtype=0, q=p, k=p, dk=p, dv=p, lse=p, stride=strides, L=128, D=64, cnt=2, beg=p, bias=None, scale=0.125, ws=p,
            nbytes=1 << 20, order=None, slots=0):
        return lib.sa_block_sparse_bwd(dtype, q, k, p, p, p, lse, p, dk, dv, _lib.i64(*stride), 1, 1, L, L, D, p, p, cnt,
                                       beg, p, bias, _lib.i64(0, 0), scale, order, slots, order, slots, ws, nbytes, None)

    for bad in (dict(dtype=-1), dict(q=None), dict(lse=None), dict(beg=None), dict(L=0), dict(cnt=0), dict(scale=0.0),
                dict(scale=math.nan), dict(ws=None), dict(ws=ctypes.c_void_p(16)), dict(nbytes=100), dict(order=p, slots=3)):
        assert bwd(**bad) == _lib.SA_ERR_INVALID, bad
    for bad in (dict(D=96), dict(q=ctypes.c_void_p(8)), dict(stride=[0, 0, 65] * 8), dict(stride=[0, 0, 1 << 30] * 8),
                dict(stride=[0, 0, -64] * 8), dict(dtype=2, bias=p)):
        assert bwd(**bad) == _lib.SA_ERR_UNSUPPORTED, bad

    def lse(dtype=0, out=p, bias=None, parts=1, ws=None, nbytes=0, buf=p):
        s = _lib.i64(0, 0, 64)
        return lib.sa_block_sparse_fwd_lse(dtype, p, s, p, s, p, s, out, s, 1, 1, 64, 64, 64, p, p, 1, bias,
                                           _lib.i64(0, 0), 0.125, None, 0, parts, ws, nbytes, buf, None)

    for bad in (dict(dtype=7), dict(buf=None), dict(parts=0), dict(parts=2), dict(out=None),
                dict(dtype=2, ws=p, nbytes=10)):
        assert lse(**bad) == _lib.SA_ERR_INVALID, bad
    for bad in (dict(dtype=2, bias=p), dict(dtype=2, parts=2), dict(bias=p, parts=2, ws=p, nbytes=1 << 30)):
        assert lse(**bad) == _lib.SA_ERR_UNSUPPORTED, bad

    def transpose(idx=p, BH=1, nqb=2, nkb=2, cnt=2):
        return lib.sa_kv_list_transpose(idx, p, BH, nqb, nkb, cnt, p, p, None)

    for bad in (dict(idx=None), dict(BH=0), dict(nqb=0), dict(nkb=0), dict(cnt=0)):
        assert transpose(**bad) == _lib.SA_ERR_INVALID, bad
    for bad in (dict(cnt=65536), dict(nqb=1 << 20, cnt=1 << 12)):
        assert transpose(**bad) == _lib.SA_ERR_UNSUPPORTED, bad
