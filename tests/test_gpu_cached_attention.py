"""Attention of new tokens over cached keys on the GPU against 64 bits, alone and behind what a training call gives."""
import pytest
import torch

import scored_reference as ref
from conftest import case
from sparseattnfunctions_amd.utils.cached_attn import cached_attention
from sparseattnfunctions_amd.utils.scored_attn import distance_buckets, row_ranges, scored_attention

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def rule(H, dev, kind):
    r = {"cap": 4.0 if "cap" in kind else None, "slopes": None, "table": None, "buckets": None}
    if "slopes" in kind:
        r["slopes"] = torch.exp2(-torch.arange(1, H + 1).float()) * torch.tensor([1.0, -0.05]).repeat(H)[:H]
        r["slopes"] = r["slopes"].to(dev)
    if "table" in kind:
        r["buckets"] = distance_buckets(32, 128, bidirectional=False, device=dev)
        r["table"] = torch.randn(32, H, generator=torch.Generator().manual_seed(H)).to(BF16).to(dev)
    return r


def make(seed, B, H, Hk, Ln, L, D, dtype, dev, Lp=0):
    g = torch.Generator().manual_seed(seed)
    x = [torch.randn(s, generator=g).to(dtype).to(dev) for s in ((B, H, Ln, D), (B, Hk, L, D), (B, Hk, L, D))]
    prefix = None
    if Lp:
        prefix = tuple(torch.randn(Hk, Lp, D, generator=g).to(dtype).to(dev) for _ in range(2))
    return (*x, prefix)


CASES = {
    "one": (dict(B=1, H=1, Hk=1, Ln=1, L=1), [1], dict()),
    "ends": (dict(B=6, H=2, Hk=2, Ln=1, L=33), [0, 1, 31, 32, 33, 17], dict()),
    "before_the_first": (dict(B=5, H=4, Hk=2, Ln=5, L=40), [0, 1, 4, 5, 40], dict(kind="slopes")),
    "clamped": (dict(B=3, H=2, Hk=1, Ln=2, L=50), [-7, 51, 2 ** 30], dict(kind="cap")),
    "tiles": (dict(B=2, H=12, Hk=2, Ln=8, L=300, D=128), [300, 111], dict(kind="table")),
    "odd_tiles": (dict(B=3, H=5, Hk=1, Ln=7, L=64), [64, 7, 30], dict(kind="cap slopes table")),
    "split": (dict(B=2, H=3, Hk=3, Ln=1, L=3000), [3000, 1029], dict(kind="table cap")),
    "split_far": (dict(B=1, H=6, Hk=1, Ln=4, L=9000, D=128), [8999], dict(kind="slopes")),
    "split_short": (dict(B=4, H=2, Hk=2, Ln=2, L=2500), [0, 1, 64, 2500], dict()),
    "window_one": (dict(B=2, H=2, Hk=2, Ln=3, L=90), [90, 2], dict(window=1)),
    "window": (dict(B=3, H=4, Hk=2, Ln=4, L=2000, D=128), [2000, 40, 3], dict(window=37, kind="table")),
    "longer_than_the_cache": (dict(B=2, H=2, Hk=1, Ln=9, L=4), [4, 2], dict(Lp=40, window=7)),
    "many": (dict(B=70, H=2, Hk=1, Ln=1, L=20), list(range(-25, 45)), dict(kind="slopes")),
    "prefix_one": (dict(B=2, H=2, Hk=2, Ln=1, L=8), [1, 8], dict(Lp=1)),
    "prefix": (dict(B=5, H=6, Hk=2, Ln=3, L=77, D=128), [0, 2, 3, 77, 50], dict(Lp=226, kind="cap slopes")),
    "prefix_long": (dict(B=40, H=2, Hk=2, Ln=1, L=30), [i % 31 for i in range(40)], dict(Lp=5000, kind="table")),
    "prefix_of_many": (dict(B=60, H=10, Hk=10, Ln=1, L=40), [i % 41 for i in range(60)], dict(Lp=90, kind="slopes")),
    "prefix_of_long": (dict(B=2, H=4, Hk=2, Ln=20, L=1500), [1500, 7], dict(Lp=700, window=900, kind="cap")),
    "prefix_window": (dict(B=4, H=3, Hk=3, Ln=2, L=600), [0, 1, 100, 600], dict(Lp=300, window=150, kind="table cap")),
}


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16], ids=str)
@pytest.mark.parametrize("name", list(CASES))
def test_values(dev, name, dtype):
    case(f"cached {name} {dtype}")
    sizes, lengths, opts = CASES[name]
    opts = dict(opts)
    q, k, v, prefix = make(sorted(CASES).index(name), dtype=dtype, dev=dev, Lp=opts.pop("Lp", 0), **{"D": 64, **sizes})
    opts = dict(window=opts.get("window", 0), prefix=prefix, **rule(q.shape[1], dev, opts.get("kind", "")))
    lengths = torch.tensor(lengths, dtype=torch.int32, device=dev)
    past = torch.arange(k.shape[2], device=dev) >= lengths[:, None, None]
    for t, x in ((k, float("nan")), (v, float("inf"))):  # rows that are not there yet
        t.masked_fill_(past[..., None], x)
    want = ref.serve(q, k, v, lengths, 0.3, **opts)
    kept = [t.clone() for t in (q, k, v, lengths)]
    got = cached_attention(q, k, v, lengths, 0.3, **opts)
    ref.check(name, got, want)
    assert torch.equal(cached_attention(q, k, v, lengths, 0.3, **opts), got)
    nothing = (lengths.clamp(0, k.shape[2])[:, None] - q.shape[2] + torch.arange(q.shape[2], device=dev) < 0)[:, None, :, None]
    assert not got.masked_select(nothing).any()
    for a, b in zip((q, k, v, lengths), kept):
        assert torch.equal(a.nan_to_num(), b.nan_to_num())
    # caches whose heads lie side by side, in a larger buffer
    B, Hk, L, D = k.shape
    wide = torch.full((B, L + 5, 2 * Hk, D), float("nan"), dtype=dtype, device=dev)
    wide[:, 3:L + 3, :Hk], wide[:, 3:L + 3, Hk:] = k.transpose(1, 2), v.transpose(1, 2)
    wide = wide[:, 3:L + 3].transpose(1, 2)
    if prefix is not None:
        side = torch.stack(prefix, 2).transpose(0, 1).contiguous()  # [Lp, Hk, 2, D]
        opts["prefix"] = tuple(side[:, :, i].transpose(0, 1)[None] for i in range(2))
    assert torch.equal(cached_attention(q.transpose(1, 2).contiguous().transpose(1, 2), wide[:, :Hk], wide[:, Hk:], lengths, 0.3,
                                        **opts), got)


def test_odd_strides(dev):
    case("one sequence of a tensor, queries that are not aligned, one key head for all")
    q, k, v, _ = make(3, 3, 2, 2, 1, 100, 64, BF16, dev)
    n = torch.tensor([70, 100, 3], dtype=torch.int32, device=dev)
    want = cached_attention(q, k, v, n, 0.3)
    odd = torch.zeros(3, 2, 1, 67, dtype=BF16, device=dev)[..., 1:65]
    odd.copy_(q)
    assert torch.equal(cached_attention(odd, k, v, n, 0.3), want)
    for b in range(3):
        one = torch.empty(100 * 64 * 2 + 8, dtype=BF16, device=dev)
        kb = one[8:].as_strided((1, 2, 100, 64), (3, 6400, 64, 1), 8)  # (a stride of no consequence)
        kb.copy_(k[b:b + 1])
        assert torch.equal(cached_attention(q[b:b + 1], kb, v[b:b + 1], n[b:b + 1], 0.3), want[b:b + 1])
    same = cached_attention(q, k[:, :1].expand(3, 2, 100, 64), v[:1].expand(3, 2, 100, 64), n, 0.3)
    assert torch.equal(same, cached_attention(q, k[:, :1].repeat(1, 2, 1, 1), v[:1].repeat(3, 1, 1, 1), n, 0.3))


def test_long_cache(dev):
    case("a cache whose offsets pass 32 bits")
    L = 2 ** 24 + 1000  # 2^31 bytes and more a tensor; the sequences 2^32 apart
    k = torch.zeros(2, 1, L, 64, dtype=BF16, device=dev)
    v = torch.zeros(2, 1, L, 64, dtype=BF16, device=dev)
    q, row, _, _ = make(4, 2, 1, 1, 1, 1, 64, BF16, dev)
    n = torch.tensor([L - 5, L], dtype=torch.int32, device=dev)
    for b, j in ((0, L - 7), (1, L - 1)):  # one key stands out by far
        k[b, 0, j] = 8 * q[b, 0, 0]
        v[b, 0, j] = row[b, 0, 0]
    out = cached_attention(q, k, v, n, 1.0)
    # of the others a weight of at most L exp(-8 |q|^2) is left, |q|^2 about 64: nothing of bf16's
    assert (q.float() ** 2).sum(3).min() > 10
    assert torch.equal(out[:, :, 0], row[:, :, 0])


@pytest.mark.parametrize("B, H, Ln, L", [(0, 2, 1, 5), (2, 0, 1, 5), (2, 2, 0, 5), (2, 2, 1, 0)])
def test_nothing(dev, B, H, Ln, L):
    case(f"empty {B} {H} {Ln} {L}")
    q, k, v, _ = make(0, B, H, H, Ln, L, 64, BF16, dev)
    out = cached_attention(q, k, v, torch.zeros(B, dtype=torch.int32, device=dev), 0.3)
    assert out.shape == q.shape and not out.any()


def test_empty_prefix(dev):
    case("a prefix of no tokens")
    q, k, v, _ = make(1, 2, 2, 1, 1, 9, 64, FP16, dev)
    n = torch.tensor([4, 9], dtype=torch.int32, device=dev)
    assert torch.equal(cached_attention(q, k, v, n, 0.3, prefix=(k[0, :, :0], v[0, :, :0])), cached_attention(q, k, v, n, 0.3))


@pytest.mark.parametrize("L, Lp", [(200, 0), (3000, 0), (60, 400)])
def test_captured_calls_as_sequences_grow(dev, L, Lp):
    case(f"captured {L} {Lp}")
    q, k, v, prefix = make(5, 3, 4, 2, 1, L, 64, BF16, dev, Lp)
    n = torch.tensor([1, L // 2, L - 5], dtype=torch.int32, device=dev)
    opts = dict(prefix=prefix, **rule(4, dev, "table cap"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cached_attention(q, k, v, n, 0.3, **opts)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = cached_attention(q, k, v, n, 0.3, **opts)
    with torch.cuda.graph(graph2, pool=graph.pool()):  # (the graphs' workspaces are in one pool)
        held2 = cached_attention(q, k, v, n, 0.3, **opts)
    for turn in range(5):
        q.copy_(make(20 + turn, 3, 4, 2, 1, 1, 64, BF16, dev)[0])
        want = cached_attention(q, k, v, n, 0.3, **opts).clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want), turn
        graph2.replay()
        torch.cuda.synchronize()
        assert torch.equal(held2, want), turn
        n.add_(1)


def test_two_streams(dev):
    case("two calls at once")
    a = make(6, 4, 4, 2, 1, 4000, 64, BF16, dev)
    b = make(7, 4, 4, 2, 1, 4000, 64, BF16, dev)
    n = torch.tensor([4000, 3, 2222, 1025], dtype=torch.int32, device=dev)
    want = [cached_attention(*x[:3], n, 0.3) for x in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for s, x, to in zip(streams, (a, b), got):
            with torch.cuda.stream(s):
                to.append(cached_attention(*x[:3], n, 0.3))
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        assert all(torch.equal(o, w) for o in outs)


def test_refusals(dev):
    case("refusals")
    q, k, v, prefix = make(8, 2, 4, 2, 1, 30, 64, BF16, dev, 10)
    n = torch.tensor([3, 30], dtype=torch.int32, device=dev)

    def refused(error, q=q, k=k, v=v, n=n, scale=0.3, **opts):
        with pytest.raises(error):
            cached_attention(q, k, v, n, scale, **opts)

    for scale in (0.0, float("nan"), float("inf")):
        refused(ValueError, scale=scale)
    refused(ValueError, n=n.long())
    refused(ValueError, n=n[:1])
    refused(ValueError, n=n.cpu())
    refused(ValueError, window=-1)
    refused(ValueError, window=2 ** 31)
    refused(ValueError, k=k[:, :1])
    refused(TypeError, v=v.float())
    refused(ValueError, k=k[..., ::2].repeat(1, 1, 1, 2).transpose(2, 3).contiguous().transpose(2, 3))
    refused(ValueError, k=torch.zeros(2, 2, 30, 65, dtype=BF16, device=dev)[..., 1:])
    refused(NotImplementedError, q=q[..., :16], k=k[..., :16], v=v[..., :16])
    refused(ValueError, prefix=(prefix[0], prefix[1][:, :5]))
    refused(ValueError, prefix=(prefix[0][:1], prefix[1][:1]))
    refused(ValueError, prefix=(prefix[0].cpu(), prefix[1].cpu()))
    refused(TypeError, prefix=(prefix[0].float(), prefix[1].float()))
    refused(ValueError, prefix=tuple(t[None].expand(2, -1, -1, -1) for t in prefix))
    refused(ValueError, prefix=tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in prefix))
    refused(ValueError, cap=-1.0)
    refused(ValueError, table=torch.zeros(4, 4, device=dev))
    refused(ValueError, slopes=torch.ones(3, device=dev))


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16], ids=str)
@pytest.mark.parametrize("kind", ["cap", "slopes", "table cap"])
def test_a_layer_is_served_as_it_was_trained(dev, dtype, kind):
    """Two documents that begin alike, packed into one row as in training; then the first part held once as a prefix and the
    rest token by token, some at a time, over caches: the outputs of training, and one step of it on the way."""
    case(f"train, then serve: {kind} {dtype}")
    H, Hk, D, Lp, own, window = 4, 2, 64, 70, (50, 33), 60 if kind == "slopes" else 0
    g = torch.Generator().manual_seed(11)
    first = [torch.randn(1, h, Lp, D, generator=g) for h in (H, Hk, Hk)]
    rest = [[torch.randn(1, h, n, D, generator=g) for h in (H, Hk, Hk)] for n in own]
    q, k, v = (torch.cat([first[i], rest[0][i], first[i], rest[1][i]], 2).to(dtype).to(dev).requires_grad_() for i in range(3))
    r = rule(H, dev, kind)
    if r["table"] is not None:
        r["table"].requires_grad_()
    lengths = torch.tensor([[Lp + n for n in own]], device=dev)
    ranges = row_ranges(lengths, q.shape[2], window=window)
    out = scored_attention(q, k, v, 0.3, ranges=ranges, **r)
    want = ref.train(q, k, v, torch.ones_like(q), 0.3, ranges=ranges, **r)
    leaves = [q, k, v] + ([r["table"]] if r["table"] is not None else [])
    names = ("out", "dq", "dk", "dv", "dtable")
    for name, x in zip(names, (out, *torch.autograd.grad(out, leaves, torch.ones_like(q)))):
        ref.check(name, x, want[name])

    out = out.detach()
    prefix = tuple(t.detach()[0, :, :Lp] for t in (k, v))
    begins = [Lp, 2 * Lp + own[0]]
    kc, vc = (torch.full((2, Hk, max(own), D), float("nan"), dtype=dtype, device=dev) for _ in range(2))
    n = torch.zeros(2, dtype=torch.int32, device=dev)
    r["table"] = None if r["table"] is None else r["table"].detach()
    at = 0
    while at < min(own):
        new = min(1 + at % 3, min(own) - at)
        rows = [slice(b + at, b + at + new) for b in begins]
        for i, x in enumerate(rows):
            kc[i, :, at:at + new], vc[i, :, at:at + new] = k.detach()[0, :, x], v.detach()[0, :, x]
        n += new
        got = cached_attention(torch.cat([q.detach()[:, :, x] for x in rows]), kc, vc, n, 0.3, prefix=prefix, window=window, **r)
        for i, x in enumerate(rows):  # each within its bound of the same values
            value, bound = want["out"][0][0, :, x], want["out"][1][0, :, x]
            # the serving call rounds P, and its sum (fp16: up to 128 of them to steps of 2^-24)
            u = {FP32: 0.0, BF16: 2 * 2.0 ** -8, FP16: 2 * 2.0 ** -11 + 2 * 128 * 2.0 ** -25}[dtype]
            most = torch.cat([v.detach()[0, :, begins[i] - Lp:begins[i]], v.detach()[0, :, begins[i]:x.stop]], 1)
            most = most.abs().amax(1).double().cpu().repeat_interleave(H // Hk, 0)[:, None]
            ref.check("served", got[i], (value, bound + (1.05 * u + 2.0 ** -20) * most))
        at += new
