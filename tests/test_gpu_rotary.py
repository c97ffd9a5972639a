"""Rotary positions against 64-bit rotations, within bounds that follow from the roundings: the two
products and their sum in fp32 (2^-24 of the second product and of the result), then the type's."""
import math

import pytest
import torch

from conftest import case
from sparseattnfunctions_amd.utils.rotary import (apply_rotary, apply_rotary_, rotary_frequencies, rotary_table,
                                                  video_positions)
from sparseattnfunctions_amd.workloads import Geometry

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _rotate(x, cos, sin, layout):
    """[B,H,L,D] in 64 bits, with what the fp32 arithmetic may add."""
    x = x.double()
    pairs = cos.shape[-1]
    i = torch.arange(pairs)
    ia, ib = (2 * i, 2 * i + 1) if layout == "interleaved" else (i, i + pairs)
    a, b = x[..., ia], x[..., ib]
    y, e = x.clone(), torch.zeros_like(x)
    y[..., ia], y[..., ib] = a * cos - b * sin, b * cos + a * sin
    e[..., ia], e[..., ib] = (b * sin).abs(), (a * sin).abs()
    return y, 2.0 ** -24 * (e + 2 * y.abs())


def _close(got, want, extra, dtype):
    u = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    tiny = {torch.float16: 2.0 ** -25}.get(dtype, 0.0)
    off = (got.detach().cpu().double() - want).abs()
    assert (off <= u * (want.abs() + extra) + extra + tiny).all(), off.max()


def _cos_sin(table, rows):
    """Per token; tokens without a row: (1, 0)."""
    ok = (rows >= 0) & (rows < table.shape[0])
    t = table.double()[rows.clamp(0, table.shape[0] - 1)]
    return torch.where(ok[..., None], t[..., 0], 1.0), torch.where(ok[..., None], t[..., 1], 0.0)


def _heads(g, B, H, L, D, dtype, memory="bhld"):
    x = torch.randn(B, H, L, D, generator=g).to(dtype)
    return x if memory == "bhld" else x.transpose(1, 2).contiguous().transpose(1, 2)


CASES = [
    # B, H, Hk, L, D, rot, skip
    (1, 1, 1, 1, 64, 64, 0),
    (2, 3, 3, 300, 64, 64, 26),
    (2, 30, 30, 45, 64, 32, 45),
    (1, 12, 3, 257, 128, 96, 7),
    (3, 5, 1, 33, 96, 96, 0),
    (2, 2, 2, 70, 64, 20, 3),  # pairs of which narrower accesses hold whole ones
    (2, 3, 2, 37, 64, 24, 5),
    (1, 4, 2, 19, 80, 2, 0),
    (1, 2, 2, 9, 7, 6, 1),
    (1, 1, 2, 5, 256, 256, 0),
    (1, 7, 0, 130, 64, 64, 2),  # queries alone
]


@pytest.mark.parametrize("memory", ["bhld", "blhd"])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", CASES, ids=str)
def test_rotation_and_gradient(dev, shape, dtype, layout, memory):
    B, H, Hk, L, D, rot, skip = shape
    case(f"rotary {shape} {dtype} {layout} {memory}")
    t = TYPES[dtype]
    g = torch.Generator().manual_seed(L + D)
    q, dq = (_heads(g, B, H, L, D, t, memory) for _ in range(2))
    k, dk = (_heads(g, B, Hk, L, D, t, memory) for _ in range(2)) if Hk else (None, None)
    table = rotary_table(torch.arange(max(1, L - skip), device=dev), rot)
    cos, sin = _cos_sin(table.cpu(), torch.arange(L) - skip)
    ql = q.to(dev).requires_grad_()
    kl = k.to(dev).requires_grad_() if Hk else None
    qo, ko = apply_rotary(ql, kl, table, layout=layout, skip=skip)
    assert qo.stride() == ql.stride() and qo.dtype == t and (ko is None) == (Hk == 0)
    _close(qo, *_rotate(q, cos, sin, layout), t)
    outs, leaves, grads = (qo,), (ql,), (dq.to(dev),)
    if Hk:
        _close(ko, *_rotate(k, cos, sin, layout), t)
        outs, leaves, grads = (qo, ko), (ql, kl), (dq.to(dev), dk.to(dev))
    back = torch.autograd.grad(outs, leaves, grads)
    for got, d in zip(back, (dq, dk)):
        _close(got, *_rotate(d, cos, -sin, layout), t)
    # text and the unturned values keep their bits
    assert torch.equal(qo[:, :, :skip].cpu(), q[:, :, :skip]) and torch.equal(qo[..., rot:].cpu(), q[..., rot:])
    # in place: the same bits
    q2, k2 = q.to(dev), k.to(dev) if Hk else None
    r = apply_rotary_(q2, k2, table, layout=layout, skip=skip)
    assert r[0] is q2 and torch.equal(q2, qo) and (not Hk or torch.equal(k2, ko))


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rot", [64, 20])
def test_rows(dev, rot, dtype, layout):
    # Tokens at rows of their own, shared or per sequence; entries outside the table leave a token alone,
    # not-a-numbers and infinities in it among the rest.
    case(f"rotary rows {rot} {dtype} {layout}")
    t = TYPES[dtype]
    g = torch.Generator().manual_seed(5)
    B, H, L = 3, 4, 90
    q, k = _heads(g, B, H, L, 64, t), _heads(g, B, 2, L, 64, t)
    table = rotary_table(torch.arange(200, device=dev) + 7, rot)
    for rows in (torch.randperm(L, generator=g), torch.randint(0, 200, (B, L), generator=g)):
        rows[..., 3], rows[..., 10], rows[..., 11], rows[..., 40] = -1, 200, 2 ** 31 - 1, -2 ** 31
        cos, sin = _cos_sin(table.cpu(), rows)
        if rows.dim() == 2:
            cos, sin = cos[:, None], sin[:, None]
        ql = q.to(dev).requires_grad_()
        qo, ko = apply_rotary(ql, k.to(dev), table, layout=layout, rows=rows.int().to(dev))
        _close(qo, *_rotate(q, cos, sin, layout), t)
        _close(ko, *_rotate(k, cos, sin, layout), t)
        d = _heads(g, B, H, L, 64, t)
        _close(torch.autograd.grad(qo, ql, d.to(dev))[0], *_rotate(d, cos, -sin, layout), t)
        odd = q.clone()
        odd[:, :, 3] = math.nan
        odd[:, :, 10, ::2] = math.inf
        got = apply_rotary(odd.to(dev), None, table, layout=layout, rows=rows.int().to(dev))[0].cpu()
        assert got[:, :, 3].isnan().all() and torch.equal(got[:, :, 10], odd[:, :, 10])
        # rows of another stride
        wide = torch.zeros(*rows.shape, 2, dtype=torch.int32, device=dev)
        wide[..., 0] = rows.int().to(dev)
        assert torch.equal(apply_rotary(q.to(dev), None, table, layout=layout, rows=wide[..., 0])[0], qo)


def test_one_token_of_each_sequence(dev):
    # A generating loop's call: the new token equals its place in the whole sequence.
    case("rotary single tokens")
    g = torch.Generator().manual_seed(6)
    table = rotary_table(torch.arange(1000, device=dev), 64)
    q = _heads(g, 4, 6, 1000, 64, torch.bfloat16, "blhd").to(dev)
    whole = apply_rotary(q, q[:, :2], table, layout="half")
    at = torch.tensor([0, 17, 999, 500], dtype=torch.int32, device=dev)
    one = torch.stack([q[b, :, i] for b, i in enumerate(at.tolist())])[:, :, None]
    got = apply_rotary(one, one[:, :2], table, layout="half", rows=at[:, None])
    for b, i in enumerate(at.tolist()):
        assert torch.equal(got[0][b, :, 0], whole[0][b, :, i]) and torch.equal(got[1][b, :, 0], whole[1][b, :, i])


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32, torch.float64])
@pytest.mark.parametrize("axes,theta,scaling", [
    (64, 10000.0, None), ((16, 24, 24), 10000.0, None), ((2, 4, 6, 8), 100.0, {"type": "linear", "factor": 3.0}),
    (128, 500000.0, {"type": "yarn", "factor": 8.0, "original_length": 4096}),
    (96, 10000.0, {"type": "ntk", "factor": 4.0}), (2, 10000.0, {"type": "ntk", "factor": 4.0}),
    (64, 10000.0, {"type": "yarn", "factor": 2.5, "original_length": 100, "beta_fast": 8, "beta_slow": 2}),
    (256, 10000.0, None)])
def test_table(dev, axes, theta, scaling, kind):
    # cos and sin: the reduced angle is off by 2^-24 of an eighth turn, the functions by two units in the
    # last place, the factor's product by one; the 64-bit angle by 2^-51 of itself.
    case(f"rotary table {axes} {scaling} {kind}")
    dims = (axes,) if isinstance(axes, int) else axes
    g = torch.Generator().manual_seed(7)
    for L, start in ((1, 0), (700, 0), (333, 4_000_000)):
        pos = start + torch.randint(0, 100000, (len(dims), L), generator=g)
        pos = pos.double() * (0.75 if kind.is_floating_point else 1)
        pos = pos.to(kind)
        if not kind.is_floating_point:
            pos[:, 0] = -pos[:, 0]
        got = rotary_table(pos.to(dev) if len(dims) > 1 else pos[0].to(dev), axes, theta=theta, scaling=scaling).cpu().double()
        want, bound = [], []
        for p, d in zip(pos.double(), dims):
            f, m = rotary_frequencies(d, theta, scaling)
            ang = p[:, None] * torch.tensor(f, dtype=torch.float64)
            want.append(torch.stack((ang.cos() * m, ang.sin() * m), -1))
            bound.append((m * (math.pi / 4 * 2.0 ** -24 + 5 * 2.0 ** -24 + ang.abs() * 2.0 ** -51))[..., None].expand(-1, -1, 2))
        want, bound = torch.cat(want, 1), torch.cat(bound, 1)
        assert got.shape == want.shape
        assert ((got - want).abs() <= bound).all(), ((got - want).abs() - bound).max()
    # a strided view of positions, and none at all
    wide = torch.zeros(len(dims), 50, 3, dtype=kind, device=dev)
    wide[..., 1] = 5
    assert torch.equal(rotary_table(wide[..., 1], axes, theta=theta, scaling=scaling),
                       rotary_table(wide[..., 1].contiguous(), axes, theta=theta, scaling=scaling))
    assert rotary_table(wide[:, :0, 0], axes).shape == (0, sum(dims) // 2, 2)


def test_video_positions(dev):
    case("video positions")
    geom = Geometry(text_len=5, T=3, Hp=4, Wp=6)
    pos = video_positions(geom, dev).cpu()
    assert pos.shape == (3, geom.n_video)
    n = torch.arange(geom.n_video)
    assert torch.equal(pos, torch.stack((n // 24, n // 6 % 4, n % 6)).int())


def test_relative_positions(dev):
    # What the rotation is for: turned scores depend on the distance of the tokens alone.
    case("rotary relative positions")
    g = torch.Generator().manual_seed(8)
    q, k = (torch.randn(1, 1, 1, 64, generator=g).to(dev).expand(1, 1, 300, 64) for _ in range(2))
    for layout in ("interleaved", "half"):
        a, b = apply_rotary(q, k, rotary_table(torch.arange(300, device=dev) + 1_000_000, 64), layout=layout)
        s = a[0, 0].double() @ b[0, 0].double().T
        for d in (0, 1, 100):
            x = s.diagonal(d)
            assert (x - x[0]).abs().max() <= 64 * 2.0 ** -22 * q.norm(dim=3).max() * k.norm(dim=3).max()


def test_steps_on_streams_and_in_graphs(dev):
    case("rotary streams and graphs")
    g = torch.Generator().manual_seed(9)
    q, k = (_heads(g, 2, 8, 500, 64, torch.bfloat16).to(dev) for _ in range(2))
    pos = torch.arange(500, device=dev)

    def step():
        t = rotary_table(pos, 64)
        return (t, *apply_rotary(q, k, t), *apply_rotary_(q.clone(), k.clone(), t, layout="half"))

    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev), torch.cuda.Stream(dev)]
    got = []
    for s in streams * 2:
        with torch.cuda.stream(s):
            got.append(step())
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        q.copy_(_heads(g, 2, 8, 500, 64, torch.bfloat16))
        pos.add_(i)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step()))


def test_second_derivatives_and_partial_gradients(dev):
    case("rotary second derivatives")
    table = rotary_table(torch.arange(20, device=dev), 64)
    q, k = (torch.randn(1, 2, 20, 64, device=dev, requires_grad=True) for _ in range(2))
    a, b = apply_rotary(q, k, table)
    (only,) = torch.autograd.grad(a.sum(), q, retain_graph=True)  # an expanded gradient, and none for k
    assert torch.equal(only, apply_rotary(torch.ones_like(q), None, table, inverse=True)[0])
    (first,) = torch.autograd.grad((a ** 3).sum(), q, create_graph=True)
    (second,) = torch.autograd.grad(first.sum(), q, retain_graph=True)
    # d/dq sum R^T 3 (Rq)^2 = R^T (6 Rq * (R 1))
    ones = apply_rotary(torch.ones_like(q), None, table)[0]
    want = apply_rotary(6 * a.detach() * ones, None, table, inverse=True)[0]
    assert torch.allclose(second, want, rtol=1e-5, atol=1e-5)
    (gk,) = torch.autograd.grad(b.sum(), k)
    assert torch.equal(gk, only)


def test_with_and_without_autograd(dev):
    # The same values with gradients, without, and where they are off; forward-mode tangents are refused.
    case("rotary without autograd")
    table = rotary_table(torch.arange(20, device=dev), 64)
    q, k = torch.randn(2, 1, 3, 20, 64, device=dev)
    want = apply_rotary(q, k, table)
    assert not want[0].requires_grad and not want[1].requires_grad
    for grads in ((True, False), (False, True)):
        x, y = (t.clone().requires_grad_(g) for t, g in zip((q, k), grads))
        got = apply_rotary(x, y, table)
        assert got[0].requires_grad and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        with torch.no_grad():
            got = apply_rotary(x, y, table)
        assert not got[0].requires_grad and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(k, torch.ones_like(k))
        with pytest.raises(RuntimeError):
            apply_rotary(q, dual, table)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_offsets_past_32_bits(dev, layout):
    # Batches 2^31 values apart, in wide accesses and one by one (20 turned values in halves); in place too.
    case(f"rotary far batches {layout}")
    base = torch.empty(2 ** 31 + 2 * 3840, dtype=torch.bfloat16, device=dev)
    for dims in (64, 20):
        table = rotary_table(torch.arange(20, device=dev), dims)
        q, k = torch.randn(2, 2, 3, 20, 64, device=dev).bfloat16()
        want = apply_rotary(q, k, table, layout=layout)
        far = [base.as_strided((2, 3, 20, 64), (2 ** 31, 1280, 64, 1), i * 3840).copy_(t) for i, t in enumerate((q, k))]
        assert all(torch.equal(x, y) for x, y in zip(apply_rotary(*far, table, layout=layout), want))
        apply_rotary_(*far, table, layout=layout)
        assert all(torch.equal(x, y) for x, y in zip(far, want))


def test_no_tokens_or_heads(dev):
    case("rotary empty")
    table = rotary_table(torch.arange(4, device=dev), 64)
    q = torch.randn(2, 3, 4, 64, device=dev)
    for a, b in ((q[:, :, :0], q[:, :, :0]), (q[:0], q[:0]), (q, q[:, :0]), (q[:, :0], q)):
        x, y = apply_rotary(a, b, table)
        assert x.shape == a.shape and y.shape == b.shape
        if a.numel():
            assert torch.equal(x, apply_rotary(a, None, table)[0])
        if b.numel():
            assert torch.equal(y, apply_rotary(b, None, table)[0])
    x, _ = apply_rotary(q, None, table[:0], skip=4)
    assert torch.equal(x, q)


def test_refusals(dev):
    case("rotary refusals")
    q = torch.zeros(2, 4, 10, 64, device=dev)
    table = rotary_table(torch.arange(10, device=dev), 64)
    rows = torch.zeros(10, dtype=torch.int32, device=dev)
    for bad in (dict(layout="pairs"), dict(skip=-1), dict(skip=11), dict(rows=rows, skip=1), dict(rows=rows.long()),
                dict(rows=rows[:9]), dict(rows=rows.cpu())):
        with pytest.raises(ValueError):
            apply_rotary(q, q, table, **bad)
    with pytest.raises(ValueError):
        apply_rotary(q, q, table[:9])  # ten tokens, nine rows
    with pytest.raises(ValueError):
        apply_rotary(q[..., :32], q[..., :32], table)
    with pytest.raises(ValueError):
        apply_rotary(q, q[:1], table)
    with pytest.raises(ValueError):
        apply_rotary(q, q[:, :, :5], table)
    with pytest.raises(TypeError):
        apply_rotary(q, q.half(), table)
    with pytest.raises(TypeError):
        apply_rotary(q.double(), None, table)
    with pytest.raises(ValueError):
        apply_rotary(q, q, table.half())
    with pytest.raises(ValueError):
        apply_rotary(q, q, table.clone().requires_grad_())
    with pytest.raises(ValueError):
        apply_rotary(q.cpu(), q, table)
    with pytest.raises(ValueError):
        apply_rotary_(q, q, table)  # one tensor twice
    with pytest.raises(ValueError):
        apply_rotary_(q[:, :1].expand(2, 4, 10, 64), None, table)
    with pytest.raises(ValueError):
        apply_rotary_(q.clone().requires_grad_(), None, table)
    with pytest.raises(TypeError):
        rotary_table(torch.zeros(3, dtype=torch.float16, device=dev), 64)
    for bad in ((torch.zeros(2, 3, device=dev), 64), (torch.zeros(3, device=dev), 63), (torch.zeros(3, device=dev), 258),
                (torch.zeros(5, 3, device=dev), (2, 2, 2, 2, 2))):
        with pytest.raises(ValueError):
            rotary_table(*bad)
    # a change in place is noticed where the table is still needed
    x = q.clone().requires_grad_()
    y, _ = apply_rotary(x, None, table)
    table.add_(0)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.sum(), x)
    # and apply_rotary_ counts as one
    z = x * 1
    w = z * z
    with torch.no_grad():
        apply_rotary_(z.detach(), None, table)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(w.sum(), x)
