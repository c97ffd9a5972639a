"""Attention with score rules on the GPU at the ends of what its arguments allow, against 64 bits."""
import math

import pytest
import torch

import scored_reference as ref
from conftest import case
from sparseattnfunctions_amd.utils.cached_attn import cached_attention
from sparseattnfunctions_amd.utils.scored_attn import distance_buckets, row_ranges, scored_attention

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
NAMES = ("out", "dq", "dk", "dv", "dtable")


@pytest.mark.parametrize("cut", ["longer", "every other", "one for all"])
def test_moved_ranges(dev, cut):
    case(f"ranges cut out of others ({cut}), moved by hooks")
    B, L = 3, 320
    lengths = torch.tensor([[100, 150], [320, 0], [7, 300]] * 2, device=dev)
    many = torch.full((2 * B, 500, 2), -2 ** 31, dtype=torch.int32, device=dev)
    many[:, :L] = row_ranges(lengths, L)
    ranges = {"longer": many[:B, :L], "every other": many[::2, :L], "one for all": many[:1, :L]}[cut]
    q, k, v, do = ref.inputs(12, B, 2, 1, L, L, 64, FP32, dev)
    for t in (q, k, v):
        t.requires_grad_()
    want = ref.train(q, k, v, do, 0.2, ranges=ranges)
    with torch.autograd.graph.save_on_cpu():
        out = scored_attention(q, k, v, 0.2, ranges=ranges)
        got = [out, *torch.autograd.grad(out, (q, k, v), do)]
    for n, x in zip(NAMES, got):
        ref.check(n, x, want[n])


def fine_cap(monkeypatch):
    """The reference's scores with an error that does not grow with the cap: tanh below 0.6 comes from a polynomial, off by 7e-8
    of the value and a handful of roundings, above it from 1 - 2 r, off by 2 (|y'| + 4) r 2^-24 <= 2^-22: less than 2^-20 of
    the score in all."""
    plain = ref.scores

    def scores(q, k, scale, far, cap=None, slopes=None, table=None, buckets=None):
        s, c, _, e_c, place = plain(q, k, scale, far, cap, slopes, table, buckets)
        e = plain(q, k, scale, far, None, slopes, table, buckets)[2]
        product = scale * (q @ k.transpose(-1, -2))
        return s, c, e + 2.0 ** -20 * product.abs(), e_c, place

    monkeypatch.setattr(ref, "scores", scores)


@pytest.mark.parametrize("cap", [257.0, 1e3, 1e4, 1e5, 1e7, 1e20])
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16], ids=str)
@pytest.mark.parametrize("kind", ["plain", "slopes", "table"])
def test_large_caps(dev, monkeypatch, cap, dtype, kind):
    case(f"cap {cap} {dtype} {kind}")
    fine_cap(monkeypatch)
    H, D = 2, 128 if kind == "slopes" else 64
    q, k, v, do = ref.inputs(13, 1, H, 1, 150, 330, D, dtype, dev)
    opts = dict(cap=cap, q_start=180)
    wanted = [q, k, v]
    if kind == "slopes":
        opts["slopes"] = torch.tensor([0.02, -0.01], device=dev)
    if kind == "table":
        opts["buckets"] = distance_buckets(32, 128, device=dev)
        opts["table"] = torch.randn(32, H, generator=torch.Generator().manual_seed(1)).to(dev)
        wanted.append(opts["table"])
    for t in wanted:
        t.requires_grad_()
    ranges = row_ranges(torch.tensor([330], device=dev), 330)
    want = ref.train(q, k, v, do, 0.3, ranges=ranges, **opts)
    out = scored_attention(q, k, v, 0.3, ranges=ranges, **opts)
    for n, x in zip(NAMES, (out, *torch.autograd.grad(out, wanted, do))):
        ref.check(n, x, want[n])


@pytest.mark.parametrize("cap", [257.0, 1e4, 1e7, 1e20])
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16], ids=str)
def test_large_caps_over_caches(dev, monkeypatch, cap, dtype):
    case(f"cap {cap} over caches {dtype}")
    fine_cap(monkeypatch)
    q, k, v, _ = ref.inputs(14, 2, 4, 2, 3, 1500, 64, dtype, dev)
    q = q[:, :, :3]
    n = torch.tensor([1500, 40], dtype=torch.int32, device=dev)
    ref.check("out", cached_attention(q, k, v, n, 0.3, cap=cap), ref.serve(q, k, v, n, 0.3, cap=cap))


@pytest.mark.parametrize("n", [300, 17776, 45104])
@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("dtype", [FP16, BF16], ids=str)
def test_many_weak_keys(dev, dtype, first, n):
    """A key that stands out, its value 0, and n of 2^-25.5 of its weight, their values 1."""
    case(f"{n} weak keys {dtype}, the strong one first: {first}")
    k = torch.zeros(1, 1, n + 1, 64, dtype=dtype, device=dev)
    v = torch.ones(1, 1, n + 1, 64, dtype=dtype, device=dev)
    at = 0 if first else n
    k[:, :, at, 0] = 16.0
    v[:, :, at] = 0
    q = torch.zeros(1, 1, 1, 64, dtype=dtype, device=dev)
    q[..., 0] = 1.0
    scale = 25.5 * math.log(2.0) / 16
    weak = n * 2.0 ** -25.5
    want = weak / (1 + weak)
    # P rounded to the type (fp16: also to steps of 2^-24, 2^-11 under the row's maximum) for all weak keys alike, out
    # rounded, the scores' 25.5 in fp32, and sums of n
    u = torch.finfo(dtype).eps / 2
    bound = want * (2 * u + 2.0 ** -18 + n * 2.0 ** -24) + (n * 2.0 ** -36 if dtype == FP16 else 0.0)
    assert bound < 0.02 * want
    lengths = torch.tensor([n + 1], dtype=torch.int32, device=dev)
    for out in (cached_attention(q, k, v, lengths, scale), scored_attention(q, k, v, scale)):
        assert (out.double() - want).abs().max().item() <= bound


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16], ids=str)
@pytest.mark.parametrize("L, Ln, Lp, window", [(400, 1, 0, 37), (400, 3, 0, 1), (2600, 2, 0, 700), (5000, 4, 0, 100), (60, 2, 100, 90),
                                               (60, 1, 100, 20), (60, 1, 300, 250), (90, 1, 3000, 2900), (90, 3, 3000, 30)])
def test_what_a_window_has_left_behind(dev, dtype, L, Ln, Lp, window):
    case(f"rows before a window: {L} {Ln} {Lp} {window} {dtype}")
    B, H, Hk = 3, 4, 2
    g = torch.Generator().manual_seed(15)
    q, k, v = (torch.randn(B, h, n, 64, generator=g).to(dtype).to(dev) for h, n in ((H, Ln), (Hk, L), (Hk, L)))
    prefix = tuple(torch.randn(Hk, Lp, 64, generator=g).to(dtype).to(dev) for _ in range(2)) if Lp else None
    n = torch.tensor([L, L // 2 + 5, Ln], dtype=torch.int32, device=dev)
    want = ref.serve(q, k, v, n, 0.3, window=window, prefix=prefix)
    first = n - Ln - window + 1  # of each sequence's own keys; of the prefix the first that any sequence sees
    at = torch.arange(L, device=dev)
    unseen = ((at < first[:, None]) | (at >= n[:, None]))[:, None, :, None]
    k, v = k.masked_fill(unseen, float("nan")), v.masked_fill(unseen, float("inf"))
    if Lp:
        unseen = (torch.arange(Lp, device=dev) < first.min() + Lp)[:, None]
        prefix = (prefix[0].masked_fill(unseen, float("-inf")), prefix[1].masked_fill(unseen, float("nan")))
    ref.check("out", cached_attention(q, k, v, n, 0.3, window=window, prefix=prefix), want)


def test_caches_are_not_differentiated(dev):
    case("a call over caches on tensors that autograd follows")
    q, k, v, _ = ref.inputs(16, 2, 2, 2, 1, 30, 64, BF16, dev)
    p = tuple(t[0].clone() for t in (k, v))
    n = torch.tensor([30, 4], dtype=torch.int32, device=dev)
    slopes, table = torch.ones(2, device=dev), torch.ones(3, 2, device=dev)
    buckets = distance_buckets(3, 1, device=dev)

    def call():
        return cached_attention(q, k, v, n, 0.3, slopes=slopes, table=table, buckets=buckets, prefix=p)

    want = call()
    assert not want.requires_grad
    for t in (q, k, v, slopes, table, *p):
        t.requires_grad_()
        out = call()
        assert torch.equal(out, want) and out.requires_grad
        with pytest.raises(NotImplementedError):
            out.sum().backward()
        with torch.no_grad():
            assert not call().requires_grad
        t.requires_grad_(False)


def shifted(monkeypatch, shift):
    """The reference with `shift` taken from each row's distances (which changes no probability) before the slopes: what the
    errors are relative to."""
    plain = ref.scores

    def scores(q, k, scale, far, cap=None, slopes=None, table=None, buckets=None):
        s, c, e, e_c, place = plain(q, k, scale, far, cap, None, table, buckets)
        add = slopes.double().cpu()[:, None, None] * (far.abs() - shift).double()
        return s - add, c, e + 2.0 ** -22 * (s.abs() + add.abs()), e_c, place

    monkeypatch.setattr(ref, "scores", scores)


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16], ids=str)
@pytest.mark.parametrize("kind", ["", "cap", "table"])
@pytest.mark.parametrize("where", ["behind", "ahead", "far behind", "far ahead", "across", "first keys"])
def test_slopes_of_distant_keys(dev, monkeypatch, where, kind, dtype):
    case(f"rows that see distant keys: {where} {kind} {dtype}")
    H, Lq, Lk, D, keys = 3, 70, 200, 64, 200
    start = {"behind": 100_000, "ahead": -100_000, "far behind": 2 ** 29 - 100, "far ahead": 100 - 2 ** 29, "across": 165,
             "first keys": 19_950}[where]
    if where == "first keys":
        Lq, Lk, D, keys = 40, 20_000, 128, 150
    q, k, v, do = ref.inputs(17, 1, H, 1, Lq, Lk, D, dtype, dev)
    slopes = torch.tensor([0.5, 0.02, -0.25], device=dev)
    ranges = torch.zeros(Lk, 2, dtype=torch.int32, device=dev)
    ranges[:keys, 1] = Lq
    place = torch.arange(Lq)[:, None] + start
    near, last = (place - place.clamp(0, keys - 1)).abs(), torch.maximum(place.abs(), (place - keys + 1).abs())
    shifted(monkeypatch, torch.stack([near, near, last]))  # (the row's heaviest keys: with a negative slope the far ones)
    opts = dict(slopes=slopes, ranges=ranges, q_start=start)
    wanted = [q, k, v]
    if kind == "cap":
        opts["cap"] = 5.0
    if kind == "table":
        opts["buckets"] = distance_buckets(32, 128, device=dev)
        opts["table"] = torch.randn(32, H, generator=torch.Generator().manual_seed(2)).to(dev)
        wanted.append(opts["table"])
    for t in wanted:
        t.requires_grad_()
    want = ref.train(q, k, v, do, 0.2, **opts)
    out = scored_attention(q, k, v, 0.2, **opts)
    for n, x in zip(NAMES, (out, *torch.autograd.grad(out, wanted, do))):
        ref.check(n, x, want[n])


def test_slopes_of_distant_keys_in_split_lists(dev, monkeypatch):
    case("rows that see distant keys, a document's lists split")
    H, L, start = 2, 2000, 300_000
    q, k, v, do = ref.inputs(18, 1, H, 1, L, L, 64, FP32, dev)
    slopes = torch.tensor([0.5, -0.01], device=dev)
    place = torch.arange(L)[:, None] + start
    shifted(monkeypatch, torch.stack([place - L + 1, place]))
    for t in (q, k, v):
        t.requires_grad_()
    want = ref.train(q, k, v, do, 0.2, slopes=slopes, q_start=start)
    out = scored_attention(q, k, v, 0.2, slopes=slopes, q_start=start)
    for n, x in zip(NAMES, (out, *torch.autograd.grad(out, (q, k, v), do))):
        ref.check(n, x, want[n])


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16], ids=str)
@pytest.mark.parametrize("Lp", [0, 100, 12_000])
def test_slopes_of_distant_keys_over_caches(dev, monkeypatch, Lp, dtype):
    case(f"the first keys of a long cache weigh most, a prefix of {Lp}, {dtype}")
    B, H, L = 2, 2, 20_000 if Lp == 0 else 500
    g = torch.Generator().manual_seed(19)
    q, k, v = (torch.randn(B, h, n, 64, generator=g).to(dtype).to(dev) for h, n in ((H, 2), (1, L), (1, L)))
    prefix = tuple(torch.randn(1, Lp, 64, generator=g).to(dtype).to(dev) for _ in range(2)) if Lp else None
    n = torch.tensor([L, L - 77], dtype=torch.int32, device=dev)
    slopes = torch.tensor([-0.5, -0.25], device=dev)
    shift = (Lp + n.cpu().long()[:, None] - 2 + torch.arange(2))[:, None, :, None]  # the distance of the first key
    shifted(monkeypatch, shift)
    ref.check("out", cached_attention(q, k, v, n, 0.2, slopes=slopes, prefix=prefix),
              ref.serve(q, k, v, n, 0.2, slopes=slopes, prefix=prefix))


@pytest.mark.parametrize("L", [768, 4000])  # bounds of key blocks taken where they are needed, and once for all
@pytest.mark.parametrize("kind", ["two", "three", "scattered"])
def test_ranges_with_gaps(dev, kind, L):
    """Keys of one block that rows far apart see, and rows between them that may hold anything."""
    case(f"ranges with gaps {kind} {L}")
    ranges = torch.zeros(L, 2, dtype=torch.int32)
    at = torch.arange(L)
    last = L // 64 * 64 - 64
    ranges[at % 2 == 0, 1] = 50
    ranges[at % 2 == 1] = torch.tensor([last, last + 40], dtype=torch.int32)
    if kind == "three":  # a bridge between two of them, and a key without rows
        ranges[at % 64 == 7] = torch.tensor([45, 64 * 5], dtype=torch.int32)
        ranges[at % 64 == 8] = torch.tensor([9, 9], dtype=torch.int32)
        ranges[at % 64 == 9] = torch.tensor([64 * 5, 64 * 6], dtype=torch.int32)
    if kind == "scattered":
        g = torch.Generator().manual_seed(3)
        begin = torch.randint(0, L // 64, (L,), generator=g) * 64
        ranges = torch.stack([begin, (begin + 3).clamp(max=L)], 1).int()
        ranges[(at // 64 > 1) | (at % 31 > 0)] = 0
    q, k, v, do = ref.inputs(20, 1, 2, 2, L, L, 64, FP32, dev)
    want = ref.train(q, k, v, do, 0.2, ranges=ranges)
    sees = torch.zeros(L // 64 + 2, dtype=torch.bool)  # blocks of rows
    for a, z in ranges.unique(dim=0).tolist():
        sees[a // 64:(z + 63) // 64 if z > a else 0] = True
    assert 2 <= sees.sum() < L // 64 - 1
    blind = (~sees[at // 64]).to(dev)
    q, do = q.masked_fill(blind[:, None], float("nan")), do.masked_fill(blind[:, None], float("inf"))
    for t in (q, k, v):
        t.requires_grad_()
    out = scored_attention(q, k, v, 0.2, ranges=ranges.to(dev))
    for n, x in zip(NAMES, (out, *torch.autograd.grad(out, (q, k, v), do))):
        ref.check(n, x, want[n])


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=str)
def test_most_distances_at_the_larger_head_dim(dev, dtype):
    case(f"1024 distances told apart on each side, head dim 128, {dtype}")
    q, k, v, do = ref.inputs(21, 1, 2, 1, 400, 1300, 128, dtype, dev)
    table = torch.randn(40, 2, generator=torch.Generator().manual_seed(4)).to(dev)
    buckets = distance_buckets(40, 1024, device=dev)
    for t in (q, k, v, table):
        t.requires_grad_()
    opts = dict(table=table, buckets=buckets, q_start=500, cap=20.0)
    want = ref.train(q, k, v, do, 0.1, **opts)
    out = scored_attention(q, k, v, 0.1, **opts)
    for n, x in zip(NAMES, (out, *torch.autograd.grad(out, (q, k, v, table), do))):
        ref.check(n, x, want[n])


def test_inference_mode(dev):
    case("calls in inference mode, and tensors made in it")
    q, k, v, do = ref.inputs(22, 2, 2, 2, 300, 300, 64, BF16, dev)
    lengths = torch.tensor([[200, 50], [300, 0]], device=dev)
    n = torch.tensor([300, 7], dtype=torch.int32, device=dev)
    table = torch.randn(9, 2, device=dev)
    buckets = distance_buckets(9, 7, device=dev)
    opts = dict(table=table, buckets=buckets)
    want = scored_attention(q, k, v, 0.2, ranges=row_ranges(lengths, 300), **opts)
    served = cached_attention(q[:, :, :2], k, v, n, 0.2, **opts)
    table.requires_grad_()
    with torch.inference_mode():
        opts["buckets"] = distance_buckets(9, 7, device=dev)
        ranges = row_ranges(lengths, 300)
        assert torch.equal(scored_attention(q, k, v, 0.2, ranges=ranges, **opts), want)
        assert torch.equal(cached_attention(q[:, :, :2], k, v, n, 0.2, **opts), served)
    # and in training, what was made there
    q.requires_grad_()
    for made in (opts["buckets"], ranges):
        assert made.is_inference()
    grads = torch.autograd.grad(scored_attention(q, k, v, 0.2, ranges=ranges, **opts), (q, table), do)
    opts["buckets"] = distance_buckets(9, 7, device=dev)
    for a, b in zip(grads, torch.autograd.grad(scored_attention(q, k, v, 0.2, ranges=row_ranges(lengths, 300), **opts), (q, table), do)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", ["", "slopes"])
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16], ids=str)
def test_gradients_of_saturated_caps(dev, monkeypatch, dtype, kind, D):
    """Scores of six to eleven caps, all of one sign: what is left of the cap's derivative has its bits."""
    case(f"saturated caps {dtype} {kind} {D}")
    plain = ref.scores

    def scores(q, k, scale, far, cap=None, slopes=None, table=None, buckets=None):
        # r = 1 / (exp2(y') + 1), y' up to 32: the argument's rounding 2^-24 |y'| log(2), exp2's, the sum's and the reciprocal's
        # 2^-22, and 4 (r - r^2) with it: 2^-19 of itself in all, besides twice the score's error over the cap
        s, c, e, _, place = plain(q, k, scale, far, cap, slopes, table, buckets)
        product = plain(q, k, scale, far, None, slopes, table, buckets)[2]
        return s, c, e, c * (2.0 ** -19 + 2 * product / cap), place

    monkeypatch.setattr(ref, "scores", scores)
    q, k, v, do = ref.inputs(23, 1, 2, 1, 200, 330, D, dtype, dev)
    q[..., 0], k[..., 0] = 8, 8  # scores of 43 +- 4 at a cap of 5
    q[..., 1:] *= 0.7 * (64 / D) ** 0.5
    k[..., 1:] *= 0.7
    scale = 43.0 / 64
    q[..., 1:] /= 8 * scale
    do = do * 2.0 ** 12  # (fp16: dS of 1e-7 and less times this; with 2^14 some were infinite)
    assert torch.isfinite(do).all()
    s = scale * (q.double() @ k.double().transpose(2, 3).repeat_interleave(2, 1))
    assert 30 < s.min() and s.max() < 55
    opts = dict(cap=5.0, q_start=130, ranges=row_ranges(torch.tensor([330], device=dev), 330))
    if kind == "slopes":
        opts["slopes"] = torch.tensor([0.02, -0.01], device=dev)
    for t in (q, k, v):
        t.requires_grad_()
    want = ref.train(q, k, v, do, scale, **opts)
    out = scored_attention(q, k, v, scale, **opts)
    for n, x in zip(NAMES, (out, *torch.autograd.grad(out, (q, k, v), do))):
        ref.check(n, x, want[n])


@pytest.mark.parametrize("cap", [1e-2, 2e-12, 1e-13, 1e-25])
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16], ids=str)
def test_small_caps(dev, dtype, cap):
    case(f"cap {cap} {dtype}")
    q, k, v, do = ref.inputs(24, 1, 2, 1, 150, 330, 64, dtype, dev)
    opts = dict(cap=cap, ranges=row_ranges(torch.tensor([100, 180], device=dev), 330))
    for t in (q, k, v):
        t.requires_grad_()
    want = ref.train(q, k, v, do, 0.3, **opts)
    out = scored_attention(q, k, v, 0.3, **opts)
    for n, x in zip(NAMES, (out, *torch.autograd.grad(out, (q, k, v), do))):
        ref.check(n, x, want[n])
    n = torch.tensor([330], dtype=torch.int32, device=dev)
    ref.check("served", cached_attention(q.detach()[:, :, :3], k, v, n, 0.3, cap=cap), ref.serve(q[:, :, :3], k, v, n, 0.3, cap=cap))


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16], ids=str)
@pytest.mark.parametrize("cap", [None, 5.0, 1e4])
def test_a_bias_that_hides_beside_slopes(dev, dtype, cap):
    case(f"a bias of -inf beside slopes, cap {cap}, {dtype}")
    q, k, v, do = ref.inputs(25, 1, 2, 2, 300, 300, 64, dtype, dev)
    slopes = torch.tensor([0.5, -0.02], device=dev)
    for t in (q, k, v):
        t.requires_grad_()
    buckets = distance_buckets(5, 2, device=dev)  # -2 and less, -1, 0, 1, 2 and more: 4, 3, 0, 1, 2
    table = torch.zeros(5, 2, device=dev)
    hiding = table.clone()
    hiding[3:] = float("-inf")  # keys behind the row
    opts = dict(cap=cap, slopes=slopes, buckets=buckets)
    want = ref.train(q, k, v, do, 0.2, table=table, ranges=row_ranges(torch.tensor([300], device=dev), 300), **opts)
    hiding.requires_grad_()
    out = scored_attention(q, k, v, 0.2, table=hiding, **opts)
    for n, x in zip(NAMES, (out, *torch.autograd.grad(out, (q, k, v, hiding), do))):
        ref.check(n, x, want[n])
    # all keys: rows of zeros, and no gradients
    nothing = torch.full_like(table, float("-inf")).requires_grad_()
    out = scored_attention(q, k, v, 0.2, table=nothing, **opts)
    assert not out.any()
    for x in torch.autograd.grad(out, (q, k, v, nothing), do):
        assert not x.any()
    # over caches, keys two and more away
    far = torch.zeros(5, 2, device=dev)
    far[2] = float("-inf")
    n = torch.tensor([300], dtype=torch.int32, device=dev)
    want = ref.serve(q[:, :, :2], k, v, n, 0.2, cap=cap, slopes=slopes, window=2)
    ref.check("served", cached_attention(q.detach()[:, :, :2], k.detach(), v.detach(), n, 0.2, table=far, **opts), want)
    assert not cached_attention(q.detach()[:, :, :2], k.detach(), v.detach(), n, 0.2, table=nothing.detach(), **opts).any()
