"""The training calls' struct, rotary frequencies and what `sa_rotary_*` and `sa_block_sparse_bwd` refuse, without a GPU."""
import ctypes
import math
import os
import subprocess

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

    def call(**changed):
        strides = changed.pop("stride", [0, 0, 64] * 8)
        a = dict(dtype=0, B=1, H=1, Lq=128, Lk=128, D=64, max_cnt=2, parts=1, sm_scale=0.125, workspace=256,
                 workspace_bytes=1 << 20)
        a.update((x, 256) for x in ("q", "k", "v", "out", "dout", "dq", "dk", "dv", "lse", "kv_idx", "kv_cnt"))
        t = _lib.AttnTrain(**{**a, **changed})
        t.strides[:] = strides
        return t

    def need(**changed):
        return lib.sa_block_sparse_bwd_workspace(call(**changed), ctypes.byref(n))

    assert need(B=2, H=30, Lq=640, Lk=650, max_cnt=11) == 0  # statistics, list beginnings and entries
    assert n.value == 60 * 10 * 128 * 4 + (60 * 12 * 4 + 255) // 256 * 256 + (60 * 10 * 11 * 4 + 255) // 256 * 256
    assert need(B=2, H=30, Lq=640, Lk=650, max_cnt=11, q_idx=256) == 0 and n.value == 60 * 10 * 128 * 4
    for bad in (dict(B=0), dict(H=0), dict(Lq=0), dict(Lk=0), dict(max_cnt=0), dict(dtype=5), dict(H=1 << 27)):
        assert need(**bad) == _lib.SA_ERR_INVALID, bad
    assert need(D=32) == _lib.SA_ERR_UNSUPPORTED
    assert lib.sa_block_sparse_bwd_workspace(None, ctypes.byref(n)) == _lib.SA_ERR_INVALID
    assert lib.sa_block_sparse_bwd_workspace(call(), None) == _lib.SA_ERR_INVALID

    def bwd(**changed):
        return lib.sa_block_sparse_bwd(call(**changed), None)

    assert lib.sa_block_sparse_bwd(None, None) == _lib.SA_ERR_INVALID
    for bad in (dict(dtype=-1), *(dict([(x, None)]) for x in ("q", "k", "v", "out", "dout", "lse", "kv_idx", "kv_cnt")),
                dict(Lq=0), dict(max_cnt=0), dict(sm_scale=0.0), dict(sm_scale=math.nan), dict(workspace=None),
                dict(workspace=16), dict(workspace_bytes=100), dict(q_order=256, n_q_slots=3), dict(k_order=256),
                dict(q_idx=256), dict(q_cnt=256)):
        assert bwd(**bad) == _lib.SA_ERR_INVALID, bad
    for bad in (dict(D=96), dict(q=8), dict(dv=8), dict(stride=[0, 0, 65] * 8), dict(stride=[0, 0, 1 << 30] * 8),
                dict(stride=[0, 0, -64] * 8), dict(dtype=2, key_bias=256), dict(max_cnt=65536, workspace_bytes=1 << 40),
                dict(sm_scale=1e-31)):
        assert bwd(**bad) == _lib.SA_ERR_UNSUPPORTED, bad

    def lse(**changed):
        return lib.sa_block_sparse_fwd_lse(call(**changed), None)

    assert lib.sa_block_sparse_fwd_lse(None, None) == _lib.SA_ERR_INVALID
    for bad in (dict(dtype=7), dict(lse=None), dict(parts=0), dict(parts=2, workspace=None), dict(out=None), dict(sm_scale=-1.0),
                dict(dtype=2, workspace_bytes=10), dict(Lk=0), dict(mask=256, Lq=0), dict(mask=256, kv_idx=None),
                dict(mask=256, kv_cnt=None), dict(mask=256, Lk=64 * 100, max_cnt=99), dict(mask=256, q_idx=256)):
        assert lse(**bad) == _lib.SA_ERR_INVALID, bad
    for bad in (dict(dtype=2, key_bias=256), dict(dtype=2, parts=2), dict(key_bias=256, parts=2), dict(D=80),
                dict(stride=[0, 0, 66] * 8)):
        assert lse(**bad) == _lib.SA_ERR_UNSUPPORTED, bad

    def transpose(idx=p, BH=1, nqb=2, nkb=2, cnt=2):
        return lib.sa_kv_list_transpose(idx, p, BH, nqb, nkb, cnt, p, p, None)

    for bad in (dict(idx=None), dict(BH=0), dict(nqb=0), dict(nkb=0), dict(cnt=0)):
        assert transpose(**bad) == _lib.SA_ERR_INVALID, bad
    for bad in (dict(cnt=65536), dict(nqb=1 << 20, cnt=1 << 12)):
        assert transpose(**bad) == _lib.SA_ERR_UNSUPPORTED, bad


def test_struct_layout(tmp_path):
    # The binding's fields lie where the header's do.
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    names = [f[0] for f in _lib.AttnTrain._fields_]
    prints = "".join(f'printf("%zu\\n", offsetof(sa_attn_train, {n}));' for n in names)
    source = tmp_path / "layout.c"
    source.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "sa_api.h"\n'
                      f'int main() {{ {prints} printf("%zu\\n", sizeof(sa_attn_train)); return 0; }}\n')
    subprocess.run(["gcc", f"-I{include}", str(source), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    want = [getattr(_lib.AttnTrain, n).offset for n in names] + [ctypes.sizeof(_lib.AttnTrain)]
    assert [int(x) for x in out.split()] == want


def test_biased_calls_need_the_rows_offsets():
    lib = _lib.load()

    def call(**changed):
        a = dict(dtype=0, B=1, H=1, Lq=128, Lk=128, D=64, max_cnt=2, parts=1, sm_scale=0.125, workspace=256,
                 workspace_bytes=1 << 20)
        a.update((x, 256) for x in ("q", "k", "v", "out", "dout", "dq", "dk", "dv", "lse", "kv_idx", "kv_cnt", "key_bias"))
        t = _lib.AttnTrain(**{**a, **changed})
        t.strides[:] = [0, 0, 64] * 8
        return t

    assert lib.sa_block_sparse_fwd_lse(call(), None) == _lib.SA_ERR_INVALID
    assert lib.sa_block_sparse_bwd(call(), None) == _lib.SA_ERR_INVALID
    # with a bias the rows' statistics take twice the room
    sizes = []
    for bias in (None, 256):
        n = ctypes.c_int64(0)
        assert lib.sa_block_sparse_bwd_workspace(call(key_bias=bias, q_idx=256), ctypes.byref(n)) == 0
        sizes.append(n.value)
    assert sizes == [2 * 128 * 4, 2 * 256 * 4]


def test_backward_limits_are_known_before_the_forward_pass():
    lib = _lib.load()

    def check(stride=64, **changed):
        t = _lib.AttnTrain(**{**dict(dtype=0, B=1, H=1, Lq=40, Lk=40, D=64, max_cnt=2, sm_scale=0.125), **changed})
        t.strides[:] = [0, 0, stride] * 8
        return lib.sa_block_sparse_bwd_check(t)

    assert check() == check(sm_scale=1e-30, dk=256, dv=256) == check(max_cnt=65536) == 0
    assert check(max_cnt=65536, dk=256, q_idx=256) == check(stride=0, Lq=1 << 27) == 0
    for bad in (dict(sm_scale=1e-31), dict(dtype=2, key_bias=256), dict(stride=1 << 24), dict(stride=-64), dict(D=96),
                dict(stride=1 << 62), dict(stride=0, Lq=(1 << 27) + 1), dict(stride=0, Lk=(1 << 27) + 1), dict(max_cnt=65536, dk=256), dict(max_cnt=65536, dv=256)):
        assert check(**bad) == _lib.SA_ERR_UNSUPPORTED, bad
    assert check(Lq=0) == check(sm_scale=0.0) == check(sm_scale=math.nan) == lib.sa_block_sparse_bwd_check(None) == _lib.SA_ERR_INVALID


def test_lengths_of_more_than_32_bits():
    # (a length behind which rounding up to a workgroup's tokens would pass 32 bits; the checks come before any launch)
    lib = _lib.load()
    p = ctypes.c_void_p(256)
    st = _lib.i64(*range(0, 120, 10))
    for L in (2 ** 31 - 1, 2 ** 31 - 255):
        rc = lib.sa_rotary_apply(0, p, p, None, None, st, 1, 1, 0, L, 64, p, 8, 32, p, 0, 0, 0, 0, None)
        assert rc == _lib.SA_ERR_INVALID
