"""Attention with score rules and over caches, without a GPU: what its C entries and Python calls refuse, sizes of buffers,
buckets of distances, and the 64-bit reference against autograd."""
import ctypes
import math

import pytest
import torch

import scored_reference as ref
from sparseattnfunctions_amd import _lib
from sparseattnfunctions_amd.utils.cached_attn import cached_attention
from sparseattnfunctions_amd.utils.scored_attn import (MOST_RADIUS, distance_buckets, row_ranges, scored_attention,
                                                       scored_attention_backward, scored_attention_forward)

P = 1 << 20  # an address that is never used: the checks come first


def scored(**over):
    B, H, Hk, Lq, Lk, D = 2, 4, 2, 100, 300, 64
    c = _lib.AttnScored(dtype=0, B=B, H=H, Hk=Hk, Lq=Lq, Lk=Lk, D=D, sm_scale=0.125, q=P, k=P, v=P, out=P, dout=P, dq=P, dk=P,
                        dv=P, lse=P, ranges=P, ranges_stride=Lk, follow=1, plan=P, plan_bytes=1 << 40, workspace=P,
                        workspace_bytes=1 << 40)
    q, k = (H * Lq * D, Lq * D, D), (Hk * Lk * D, Lk * D, D)
    c.strides[:] = (*q, *k, *k, *q, *q, *q, *k, *k)
    for name, x in over.items():
        if name.startswith("stride"):
            c.strides[int(name[6:])] = x
        else:
            setattr(c, name, x)
    return c


INVALID, UNSUPPORTED = _lib.SA_ERR_INVALID, _lib.SA_ERR_UNSUPPORTED


@pytest.mark.parametrize("over, code", [
    (dict(dtype=3), INVALID), (dict(dtype=-1), INVALID), (dict(B=0), INVALID), (dict(H=0), INVALID), (dict(Hk=3), INVALID),
    (dict(Lq=0), INVALID), (dict(Lk=-1), INVALID), (dict(D=96), UNSUPPORTED), (dict(sm_scale=0.0), INVALID),
    (dict(sm_scale=math.nan), INVALID), (dict(sm_scale=math.inf), INVALID), (dict(cap=-1.0), INVALID),
    (dict(cap=math.inf), INVALID), (dict(cap=math.nan), INVALID), (dict(cap=1e-38), INVALID), (dict(q_start=1 << 29), INVALID),
    (dict(q_start=-(1 << 29)), INVALID), (dict(table=P, n_buckets=4), INVALID), (dict(table=P, buckets=P), INVALID),
    (dict(table=P, buckets=P, n_buckets=4, table_dtype=5), INVALID),
    (dict(table=P, buckets=P, n_buckets=4, radius=MOST_RADIUS + 1), UNSUPPORTED),
    (dict(table=P, buckets=P, n_buckets=4, radius=-1), UNSUPPORTED), (dict(follow=2), INVALID),
    (dict(Lq=1 << 28), UNSUPPORTED), (dict(B=1 << 23, Lq=1, Lk=1), UNSUPPORTED),
    (dict(H=1 << 21, Hk=1, B=1, Lq=1, Lk=1), UNSUPPORTED)], ids=str)
def test_scored_calls_refused_by_their_sizes(over, code):
    lib = _lib.load()
    n = (ctypes.c_int64 * 3)()
    call = scored(**over)
    assert lib.sa_attn_scored_sizes(call, n) == code
    assert lib.sa_attn_scored_fwd(call, None) == code
    assert lib.sa_attn_scored_bwd(call, None) == code


@pytest.mark.parametrize("over, fwd, bwd", [
    (dict(q=None), INVALID, INVALID), (dict(k=None), INVALID, INVALID), (dict(v=None), INVALID, INVALID),
    (dict(out=None), INVALID, INVALID), (dict(lse=None), INVALID, INVALID), (dict(dout=None), None, INVALID),
    (dict(q=P + 8), UNSUPPORTED, UNSUPPORTED), (dict(v=P + 2), UNSUPPORTED, UNSUPPORTED), (dict(dk=P + 8), None, UNSUPPORTED),
    (dict(stride0=4), UNSUPPORTED, UNSUPPORTED), (dict(stride5=68), UNSUPPORTED, UNSUPPORTED),
    (dict(stride5=-64), UNSUPPORTED, UNSUPPORTED), (dict(stride8=1 << 30), UNSUPPORTED, UNSUPPORTED),
    (dict(stride14=1 << 24), None, UNSUPPORTED), (dict(plan=None), INVALID, INVALID), (dict(plan=P + 16), INVALID, INVALID),
    (dict(plan_bytes=255), INVALID, INVALID), (dict(ranges=P + 4), INVALID, INVALID), (dict(out_lo=P + 8), INVALID, INVALID),
    (dict(workspace=None), None, INVALID), (dict(workspace=P + 128), None, INVALID), (dict(workspace_bytes=512), None, INVALID),
    (dict(follow=0), None, INVALID), (dict(dtable=P), None, INVALID)], ids=str)
def test_scored_calls_refused_by_their_tensors(over, fwd, bwd):
    lib = _lib.load()
    call = scored(**over)
    if fwd is not None:
        assert lib.sa_attn_scored_fwd(call, None) == fwd
    assert lib.sa_attn_scored_bwd(call, None) == bwd


def test_scored_null_calls():
    lib = _lib.load()
    assert lib.sa_attn_scored_sizes(None, (ctypes.c_int64 * 3)()) == INVALID
    assert lib.sa_attn_scored_sizes(scored(), None) == INVALID
    assert lib.sa_attn_scored_fwd(None, None) == INVALID
    assert lib.sa_attn_scored_bwd(None, None) == INVALID
    assert lib.sa_attn_cached_fwd(None, None) == INVALID
    assert lib.sa_attn_cached_workspace(None, ctypes.byref(ctypes.c_int64())) == INVALID


def sizes(**over):
    n = (ctypes.c_int64 * 3)()
    _lib.check(_lib.load().sa_attn_scored_sizes(scored(**over), n), "sizes")
    return list(n)


def test_scored_sizes():
    for over in (dict(), dict(dtype=2), dict(follow=0), dict(mask=P), dict(Lk=5000, Lq=5000), dict(ranges=None, Lq=64, Lk=64)):
        assert all(x % 256 == 0 for x in sizes(**over)), over
    # no lists: neither a mask nor ranges, or few rows and keys; nothing is split either
    assert sizes(ranges=None, Lq=256, Lk=256)[:2] == [0, 0] and sizes(Lq=256, Lk=256)[:2] == [0, 0]
    assert sizes(Lq=257, Lk=257)[0] > 0
    # with a mask a head's lists each: 4 bytes an entry, of keys and of rows
    few, many = sizes(Lq=6400, Lk=6400), sizes(Lq=6400, Lk=6400, mask=P)
    lists = lambda n: 2 * sum((x + 255) // 256 * 256 for x in (n * 100 * 100 * 4, n * 100 * 4))
    assert many[0] - few[0] == lists(2 * 4) - lists(2)
    assert sizes(follow=0)[0] < sizes()[0]


def cached(**over):
    B, H, Hk, Ln, L, Lp, D = 2, 4, 2, 3, 5000, 100, 64
    c = _lib.AttnCached(dtype=0, B=B, H=H, Hk=Hk, Ln=Ln, L=L, Lp=Lp, D=D, sm_scale=0.125, q=P, out=P, k=P, v=P, prefix_k=P,
                        prefix_v=P, lengths=P, workspace=P, workspace_bytes=1 << 40)
    q, k, p = (H * Ln * D, Ln * D, D), (Hk * L * D, L * D, D), (0, Lp * D, D)
    c.strides[:] = (*q, *q, *k, *k, *p, *p)
    for name, x in over.items():
        if name.startswith("stride"):
            c.strides[int(name[6:])] = x
        else:
            setattr(c, name, x)
    return c


@pytest.mark.parametrize("over, code", [
    (dict(dtype=7), INVALID), (dict(B=0), INVALID), (dict(Ln=0), INVALID), (dict(L=0), INVALID), (dict(Lp=-1), INVALID),
    (dict(H=5), INVALID), (dict(window=-1), INVALID), (dict(D=32), UNSUPPORTED), (dict(L=(1 << 29) + 1), UNSUPPORTED),
    (dict(Lp=(1 << 29) + 1), UNSUPPORTED), (dict(sm_scale=-1.0), INVALID), (dict(cap=math.inf), INVALID),
    (dict(table=P), INVALID), (dict(table=P, buckets=P, n_buckets=2, radius=4000), UNSUPPORTED),
    (dict(B=1 << 20), UNSUPPORTED)], ids=str)
def test_cached_calls_refused_by_their_sizes(over, code):
    lib = _lib.load()
    n = ctypes.c_int64()
    assert lib.sa_attn_cached_workspace(cached(**over), ctypes.byref(n)) == code
    assert lib.sa_attn_cached_fwd(cached(**over), None) == code


@pytest.mark.parametrize("over, code", [
    (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(k=None), INVALID), (dict(lengths=None), INVALID),
    (dict(prefix_v=None), INVALID), (dict(k=P + 8), UNSUPPORTED), (dict(prefix_k=P + 8), UNSUPPORTED),
    (dict(stride6=12), UNSUPPORTED), (dict(stride8=-64), UNSUPPORTED), (dict(stride11=1 << 25), UNSUPPORTED),
    (dict(workspace=None), INVALID), (dict(workspace=P + 64), INVALID), (dict(workspace_bytes=100), INVALID)], ids=str)
def test_cached_calls_refused_by_their_tensors(over, code):
    assert _lib.load().sa_attn_cached_fwd(cached(**over), None) == code


def test_cached_workspace():
    lib = _lib.load()
    n = ctypes.c_int64()
    _lib.check(lib.sa_attn_cached_workspace(cached(Lp=0, L=1024), ctypes.byref(n)), "workspace")
    assert n.value == 0  # up to 1024 keys without a prefix: nothing is split
    _lib.check(lib.sa_attn_cached_workspace(cached(Lp=0, L=1025), ctypes.byref(n)), "workspace")
    assert n.value > 0
    _lib.check(lib.sa_attn_cached_workspace(cached(Lp=500, L=500), ctypes.byref(n)), "workspace")
    assert n.value == 0  # nor with a short one, for as few sequences
    for over in (dict(Lp=1000, L=500), dict(Lp=50, L=50, B=1000)):
        _lib.check(lib.sa_attn_cached_workspace(cached(**over), ctypes.byref(n)), "workspace")
        assert n.value > 0
    assert lib.sa_attn_cached_workspace(cached(), None) == INVALID


def test_row_ranges_refused():
    lib = _lib.load()

    def call(lengths=P, B=1, n=1, L=10, causal=1, frame=1, window=0, out=P):
        return lib.sa_row_ranges(lengths, None, B, n, L, causal, frame, window, out, None)

    for over in (dict(lengths=None), dict(out=None), dict(B=0), dict(n=0), dict(L=0), dict(frame=0), dict(window=-1),
                 dict(causal=0, frame=2)):
        assert call(**over) == INVALID, over
    for over in (dict(n=8193), dict(B=65536), dict(L=(1 << 30) + 1)):
        assert call(**over) == UNSUPPORTED, over


def test_no_cpu_path():
    q = torch.zeros(1, 1, 4, 64)
    for f in (lambda: scored_attention(q, q, q, 1.0), lambda: scored_attention_forward(q, q, q, 1.0),
              lambda: cached_attention(q, q, q, torch.ones(1, dtype=torch.int32), 1.0),
              lambda: row_ranges(torch.ones(1, dtype=torch.int32), 4)):
        with pytest.raises(ValueError):
            f()


@pytest.mark.parametrize("n, radius, both", [(32, 128, True), (32, 128, False), (16, 64, True), (64, 800, True), (9, 7, True),
                                             (1, 5, True), (1, 5, False), (2, 0, True), (3, 1, False), (700, 100, False)])
def test_distance_buckets(n, radius, both):
    b = distance_buckets(n, radius, both, device="cpu").tolist()
    assert len(b) == 2 * radius + 1 and min(b) >= 0 and max(b) < n
    ahead = b[radius:]  # keys before the row, or itself
    assert ahead == sorted(ahead) and ahead[0] == 0
    behind = b[:radius][::-1]
    if both:
        side = (n - 1) // 2
        assert all((x == 0 and y == 0) or y == x + side for x, y in zip(ahead[1:], behind))
    else:
        assert not any(behind)
    for bad in (dict(n_buckets=0, radius=4), dict(n_buckets=4, radius=-1), dict(n_buckets=4, radius=MOST_RADIUS + 1)):
        with pytest.raises(ValueError):
            distance_buckets(**bad)


def test_reference_against_autograd():
    B, H, Hk, Lq, Lk, D = 2, 4, 2, 20, 37, 64
    q, k, v, do = (t.requires_grad_() for t in ref.inputs(1, B, H, Hk, Lq, Lk, D, torch.float64))
    table = torch.randn(9, H, dtype=torch.float64, requires_grad=True)
    buckets = distance_buckets(9, 7, device="cpu")
    slopes = torch.tensor([0.5, -0.25, 0.0, 0.1], dtype=torch.float64)
    ranges = torch.tensor([[[j // 3, j] for j in range(Lk)]] * B, dtype=torch.int32)
    far = torch.arange(Lq)[:, None] + 5 - torch.arange(Lk)
    s = 0.3 * (q @ k.repeat_interleave(2, 1).transpose(2, 3))
    s = 4 * torch.tanh(s / 4) - slopes[:, None, None] * far.abs() + table[buckets.long()[far.clamp(-7, 7) + 7]].permute(2, 0, 1)
    seen = ref.visible(B, H, Lq, Lk, ranges)
    p = torch.nan_to_num(torch.softmax(s.masked_fill(~seen, -math.inf), 3), nan=0.0)
    out = p @ v.repeat_interleave(2, 1)
    got = torch.autograd.grad(out, (q, k, v, table), do.detach())
    want = ref.train(q, k, v, do, 0.3, 4.0, slopes, table, buckets, ranges, None, 5)
    for name, x in zip(("out", "dq", "dk", "dv", "dtable"), (out, *got)):
        assert torch.allclose(x.detach(), want[name][0], rtol=1e-10, atol=1e-12), name
