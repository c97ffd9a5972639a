"""Attention with score rules and its gradients on the GPU against 64 bits, within bounds that scored_reference.py derives."""
import pytest
import torch
import torch.utils.checkpoint

import scored_reference as ref
from conftest import case
from sparseattnfunctions_amd.utils.scored_attn import (distance_buckets, row_ranges, scored_attention,
                                                       scored_attention_backward, scored_attention_forward)

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
NAMES = ("out", "dq", "dk", "dv", "dtable")


def interval(lengths, L, causal=True, prefix=None, frame=1, window=0):
    """Each key's first row and the one behind its last, [L, 2], document by document."""
    rows, begin = [[0, 0]] * L, 0
    for n, size in enumerate(lengths):
        size = max(0, min(size, L - begin))
        end, head = begin + size, begin + min(size, max(0, prefix[n]) if prefix else 0)
        for j in range(begin, end):
            a, z = begin, end
            if j >= head:
                if causal:
                    a = j - (j - head) % frame
                elif window:
                    a = max(begin, j + 1 - window)
                if window:
                    z = min(end, j + window)
            rows[j] = [a, z]
        begin = end
    return torch.tensor(rows, dtype=torch.int32).view(L, 2)


def seen_alike(a, b):
    """Intervals with the same rows: empty ones are alike wherever they lie."""
    empty = lambda r: r[..., 0] >= r[..., 1]
    return bool(((a == b).all(-1) | (empty(a) & empty(b))).all())


@pytest.mark.parametrize("lengths, L, opts", [
    ([[1]], 1, dict()), ([[0]], 3, dict()), ([[5, 0, 7]], 20, dict()), ([[5, 9], [0, 3]], 12, dict(causal=False)),
    ([[300, 1, 777, 4], [4, 4, 4, 2000]], 1500, dict(prefix=[[3, 5, 700, 9], [0, 0, 100, 226]], frame=45)),
    ([[400, 900, 3000]], 2500, dict(window=37)), ([[400, 900, 3000]], 2500, dict(window=37, causal=False, prefix=[[50, 0, 4]])),
    ([[2047, 2], [1024, 1024]], 2048, dict(causal=False, window=1)), ([[100, -5, 30]], 140, dict()),
    ([[3] * 700], 2000, dict(frame=2)), ([[64, 64]], 128, dict(frame=1350, prefix=[[10, 10]])),
    ([[90]], 70, dict(frame=8, window=5))], ids=str)
def test_row_ranges(dev, lengths, L, opts):
    case(f"row ranges {lengths} {L} {opts}")
    prefix = opts.get("prefix")
    t = torch.tensor(lengths, dtype=torch.int32, device=dev)
    got = row_ranges(t, L, **{**opts, "prefix": None if prefix is None else torch.tensor(prefix, device=dev)})
    want = torch.stack([interval(x, L, **{**opts, "prefix": None if prefix is None else prefix[b]}) for b, x in enumerate(lengths)])
    assert got.dtype == torch.int32 and got.shape == want.shape and seen_alike(got.cpu(), want)
    if not prefix:
        assert torch.equal(row_ranges(t.long().t().contiguous().t(), L, **opts), got)
        if len(lengths) == 1:
            assert torch.equal(row_ranges(t[0], L, **opts), got)


def rule(seed, H, dev, cap=None, slopes=False, table=None):
    g = torch.Generator().manual_seed(seed)
    r = {"cap": cap, "slopes": None, "table": None, "buckets": None}
    if slopes:  # of both signs, and zero
        x = torch.exp2(-torch.arange(1, H + 1).float())
        x[1::3] *= -0.1
        x[2::3] = 0.0
        r["slopes"] = x.to(dev)
    if table:
        n, radius, dtype = table
        r["buckets"] = distance_buckets(n, radius, device=dev)
        r["table"] = torch.randn(n, H, generator=g).to(dtype).to(dev).requires_grad_()
    return r


CASES = {
    "one": dict(L=1),
    "one_key": dict(Lq=70, Lk=1, cap=5.0),
    "half_block": dict(L=33, D=128, cap=5.0),
    "causal_slopes": dict(L=64, lengths=[[64]], slopes=True),
    "both_ways": dict(L=65, table=(9, 7, FP32), q_start=-3),
    "documents": dict(H=6, Hk=2, L=200, lengths=[[90, 0, 70]], prefix=[[10, 5, 100]], cap=5.0),
    "frames": dict(B=2, L=321, lengths=[[321], [300]], prefix=[[30], [30]], frame=45),
    "window": dict(H=3, L=400, lengths=[[400]], causal=False, window=37, slopes=True, D=128),
    "causal_table": dict(B=2, L=700, lengths=[[700], [500]], table=(32, 128, BF16)),
    "last_rows": dict(Lq=70, Lk=500, q_start=430, table=(3, 0, FP16)),
    "every_rule": dict(H=3, Lq=300, Lk=97, q_start=-100, cap=5.0, slopes=True, table=(64, 800, FP32)),
    "mask": dict(B=2, H=4, Hk=2, L=450, keep=0.4),
    "mask_and_ranges": dict(H=2, L=450, keep=0.6, lengths=[[100, 320]], D=128, cap=5.0, slopes=True),
    "split_rows": dict(L=2600, lengths=[[2600]]),
    "split_keys": dict(H=3, Hk=1, L=1100, lengths=[[1000]], D=128, table=(32, 128, FP32)),
    "far": dict(H=2, L=1300, table=(33, 1024, FP32), slopes=True, cap=5.0),
}


def make(name, dtype, dev):
    c = {"B": 1, "H": 2, "D": 64, "q_start": 0, "keep": 1.0, "lengths": None, **CASES[name]}
    B, H = c["B"], c["H"]
    Hk, Lq, Lk = c.get("Hk", H), c.get("Lq", c.get("L")), c.get("Lk", c.get("L"))
    seed = sorted(CASES).index(name)
    q, k, v, do = ref.inputs(seed, B, H, Hk, Lq, Lk, c["D"], dtype, dev)
    r = rule(seed, H, dev, c.get("cap"), c.get("slopes", False), c.get("table"))
    ranges = mask = None
    if c["lengths"] is not None:
        prefix = c.get("prefix")
        ranges = row_ranges(torch.tensor(c["lengths"], device=dev), Lk, causal=c.get("causal", True), frame=c.get("frame", 1),
                            prefix=None if prefix is None else torch.tensor(prefix, device=dev), window=c.get("window", 0))
    if c["keep"] < 1:
        mask = torch.rand(B, H, -(-Lq // 64), -(-Lk // 64), generator=torch.Generator().manual_seed(seed)) < c["keep"]
        mask[:, 0, 1], mask[:, -1, :, 2] = False, False  # rows that see nothing, keys that nobody sees
        mask = mask.to(dev)
    for t in (q, k, v):
        t.requires_grad_()
    return (q, k, v, do), dict(r, ranges=ranges, block_mask=mask, q_start=c["q_start"])


def reference(q, k, v, do, scale, opts):
    o = dict(opts)
    o["mask"] = o.pop("block_mask", None)
    return ref.train(q, k, v, do, scale, **o)


def results(q, k, v, do, scale, opts):
    out = scored_attention(q, k, v, scale, **opts)
    wanted = [q, k, v] + ([opts["table"]] if opts.get("table") is not None else [])
    return [out, *torch.autograd.grad(out, wanted, do)]


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16], ids=str)
@pytest.mark.parametrize("name", list(CASES))
def test_values_and_gradients(dev, name, dtype):
    case(f"scored {name} {dtype}")
    (q, k, v, do), opts = make(name, dtype, dev)
    scale = 0.25
    got = results(q, k, v, do, scale, opts)
    want = reference(q, k, v, do, scale, opts)
    for n, x in zip(NAMES, got):
        ref.check(n, x, want[n])
    again = results(q, k, v, do, scale, opts)
    for n, x, y in zip(NAMES, got, again):
        assert torch.equal(x, y), n
    out, state = scored_attention_forward(q, k, v, scale, **opts)
    assert torch.equal(out, got[0])
    halves = scored_attention_backward(do, state)
    for n, x, y in zip(NAMES, got[1:], halves):
        assert torch.equal(x, y), n
    assert opts["table"] is not None or halves[3] is None
    with torch.no_grad():  # nothing is kept: the forward pass is the same
        assert torch.equal(scored_attention(q, k, v, scale, **opts), got[0])


@pytest.mark.parametrize("L", [130, 290])  # without and with lists
@pytest.mark.parametrize("one", [False, True])
def test_own_ranges(dev, L, one):
    case(f"own ranges {L} {one}")
    B = 2
    g = torch.Generator().manual_seed(L)
    ranges = torch.randint(-20, L + 20, (1 if one else B, L, 2), generator=g, dtype=torch.int32)
    ranges[:, 5:12] = 7  # nobody
    ranges[:, 20] = torch.tensor([-2 ** 31, 2 ** 31 - 1])
    ranges[:, 64:128, 1] = 40  # only the first rows
    q, k, v, do = ref.inputs(L, B, 2, 2, L, L, 64, FP32, dev)
    opts = dict(ranges=ranges.to(dev))
    for t in (q, k, v):
        t.requires_grad_()
    want = reference(q, k, v, do, 0.2, opts)
    shapes = [ranges.to(dev)] + ([ranges[0].to(dev)] if one else [])
    wide = torch.zeros(*ranges.shape[:2], 3, dtype=torch.int32, device=dev)
    wide[..., 1:] = ranges.to(dev)
    for r in shapes + [wide[..., 1:]]:
        for n, x in zip(NAMES, results(q, k, v, do, 0.2, dict(ranges=r))):
            ref.check(n, x, want[n])


def test_masks_of_other_shapes_and_types(dev):
    case("block masks")
    B, H, L = 2, 3, 300
    q, k, v, do = ref.inputs(3, B, H, H, L, L, 64, BF16, dev)
    for t in (q, k, v):
        t.requires_grad_()
    for shape, dtype in (((1, 1, 5, 5), torch.bool), ((B, 1, 7, 9), torch.int32), ((1, H, 5, 6), torch.uint8), ((B, H, 6, 5), torch.float32)):
        mask = torch.randint(0, 3, shape, generator=torch.Generator().manual_seed(4)).to(dtype).to(dev)
        for m in (mask, mask.transpose(2, 3).contiguous().transpose(2, 3)):
            want = reference(q, k, v, do, 0.125, dict(block_mask=m))
            for n, x in zip(NAMES, results(q, k, v, do, 0.125, dict(block_mask=m))):
                ref.check(n, x, want[n])


def test_strides(dev):
    case("strides")
    B, H, Hk, L, D = 2, 4, 2, 150, 64
    want = None
    q, k, v, do = ref.inputs(5, B, H, Hk, L, L, D, BF16, dev)
    for t in (q, k, v):
        t.requires_grad_()
    plain = results(q, k, v, do, 0.2, dict(cap=3.0))

    def blhd(t):
        return t.detach().transpose(1, 2).contiguous().transpose(1, 2)

    def odd(t):  # rows that are not 16-byte aligned
        x = torch.zeros(*t.shape[:3], D + 3, dtype=t.dtype, device=dev)
        x[..., 1:D + 1] = t.detach()
        return x[..., 1:D + 1]

    def wide(t):
        x = torch.full((*t.shape[:2], L + 7, D + 8), float("nan"), dtype=t.dtype, device=dev)
        x[:, :, 2:L + 2, 8:] = t.detach()
        return x[:, :, 2:L + 2, 8:]

    for change in (blhd, odd, wide):
        x = [change(t).requires_grad_() for t in (q, k, v)]
        for n, a, b in zip(NAMES, results(*x, change(do), 0.2, dict(cap=3.0)), plain):
            assert torch.equal(a, b), (change.__name__, n)
    # one tensor three times; one row, head and sequence for all; a broadcast gradient
    x = q.detach()[:, :, :100].clone().requires_grad_()
    out = scored_attention(x, x, x, 0.2)
    want = ref.train(x, x, x, do[:, :, :100], 0.2)
    bound = sum(want[n][1] for n in ("dq", "dk", "dv"))
    value = sum(want[n][0] for n in ("dq", "dk", "dv"))
    got, = torch.autograd.grad(out, x, do[:, :, :100])
    ref.check("sum", got, (value, bound * (1 + 2 ** -7) + 2 ** -7 * value.abs() + 2 ** -7 * sum(want[n][0].abs() for n in ("dq", "dk", "dv"))))
    row = q.detach()[:1, :1, :1].clone()
    y = [row.expand(B, H, L, D), k.detach()[:, :, :1].expand(B, Hk, L, D), v.detach()[:1].expand(B, Hk, L, D)]
    y = [t.requires_grad_() for t in y]
    want = ref.train(*y, do, 0.2)
    for n, a in zip(NAMES, results(*y, do, 0.2, {})):
        ref.check(n, a, want[n])
    ones = torch.ones((), dtype=BF16, device=dev).expand_as(q)
    for a, b in zip(results(q, k, v, ones, 0.2, {}), results(q, k, v, ones.contiguous(), 0.2, {})):
        assert torch.equal(a, b)


def test_sequences_far_apart(dev):
    case("32-bit offsets between sequences")
    B, H, L, D = 2, 1, 100, 64
    apart = 2 ** 31 + 64 * 100  # elements
    buf = torch.empty(apart + 64 * 200, dtype=BF16, device=dev)
    x = ref.inputs(6, B, H, H, L, L, D, BF16, dev)
    views = []
    for i, t in enumerate(x[:2]):
        w = torch.as_strided(buf, (B, H, L, D), (apart, D, D, 1), i * 64 * 100)
        w.copy_(t)
        views.append(w.requires_grad_())
    q, k = views
    v = x[2].requires_grad_()
    want = ref.train(q, k, v, x[3], 0.2)
    for n, a in zip(NAMES, results(q, k, v, x[3], 0.2, {})):
        ref.check(n, a, want[n])


def test_hidden_values_may_be_anything(dev):
    case("NaN and infinities in blocks that nobody sees")
    L = 700
    q, k, v, do = ref.inputs(7, 1, 2, 2, L, L, 64, BF16, dev)
    ranges = row_ranges(torch.tensor([300, 84], device=dev), L)  # blocks from 384 on: nobody's
    want = ref.train(q, k, v, do, 0.2, ranges=ranges)
    for t, x in ((q, float("nan")), (k, float("inf")), (v, float("nan")), (do, float("-inf"))):
        t[:, :, 384:] = x
    for t in (q, k, v):
        t.requires_grad_()
    for n, a in zip(NAMES, results(q, k, v, do, 0.2, dict(ranges=ranges))):
        ref.check(n, a, want[n])


def test_large_scores(dev):
    case("scores that leave the exponential's range")
    q, k, v, do = ref.inputs(8, 1, 1, 1, 90, 90, 64, FP32, dev)
    for t in (q, k, v):
        t.requires_grad_()
    for opts in (dict(), dict(cap=500.0), dict(slopes=torch.tensor([3.0], device=dev))):
        want = ref.train(q, k, v, do, 40.0, **opts)
        for n, a in zip(NAMES, results(q, k, v, do, 40.0, opts)):
            ref.check(n, a, want[n])


@pytest.mark.parametrize("dtype", [FP32, BF16], ids=str)
@pytest.mark.parametrize("low", [torch.finfo(BF16).min, torch.finfo(FP32).min, float("-inf")])
def test_a_bias_that_hides(dev, dtype, low):
    case(f"a bias of {low}")
    q, k, v, do = ref.inputs(8, 1, 2, 2, 300, 300, 64, dtype, dev)
    for t in (q, k, v):
        t.requires_grad_()
    table = torch.zeros(3, 2, dtype=FP32, device=dev)
    table[1] = 0.5
    buckets = distance_buckets(3, 1, device=dev)  # bucket 2: keys behind the row
    want = ref.train(q, k, v, do, 0.2, table=table, buckets=buckets, ranges=row_ranges(torch.tensor([300], device=dev), 300))
    hiding = table.clone()
    hiding[2] = low
    got = results(q, k, v, do, 0.2, dict(table=hiding.requires_grad_(), buckets=buckets))
    for n, a in zip(NAMES, got):
        ref.check(n, a, want[n])
    assert not got[4][2].any()


def test_gradient_against_differences(dev):
    case("differences")
    (q, k, v, do), opts = make("every_rule", FP32, dev)
    names = ("dq", "dk", "dv", "dtable")
    want = reference(q, k, v, do, 0.25, opts)
    got = dict(zip(NAMES, results(q, k, v, do, 0.25, opts)))
    x = dict(zip(names, (q, k, v, opts["table"])))
    g = torch.Generator().manual_seed(9)
    for n in names:
        way = torch.randn(x[n].shape, generator=g, dtype=torch.float64)
        loss = []
        for h in (1e-4, -1e-4):
            y = {m: t.detach().double().cpu() for m, t in x.items()}
            y[n] = y[n] + h * way
            o = dict(opts, table=y["dtable"])
            loss.append((reference(y["dq"], y["dk"], y["dv"], do, 0.25, o)["out"][0] * do.double().cpu()).sum())
        slope = ((loss[0] - loss[1]) / 2e-4).item()
        mine = (got[n].double().cpu() * way).sum().item()
        # the differences' own error: h^2 times a third derivative, which is of the order of the slope's terms
        assert abs(mine - slope) <= (want[n][1] * way.abs()).sum().item() + 1e-6 * (want[n][0] * way).abs().sum().item(), n


def test_needs_and_hooks(dev):
    case("subsets of gradients, moved and recomputed tensors, one derivative")
    (q, k, v, do), opts = make("causal_table", BF16, dev)
    table = opts["table"]
    full = results(q, k, v, do, 0.25, opts)
    leaves = (q, k, v, table)
    for bits in range(1, 16):
        some = [t.detach().requires_grad_(bool(bits >> i & 1)) for i, t in enumerate(leaves)]
        out = scored_attention(*some[:3], 0.25, **dict(opts, table=some[3]))
        wanted = [t for t in some if t.requires_grad]
        for a, b in zip(torch.autograd.grad(out, wanted, do), [x for i, x in enumerate(full[1:]) if bits >> i & 1]):
            assert torch.equal(a, b), bits
        need = [bool(bits >> i & 1) for i in range(4)]
        _, state = scored_attention_forward(*some[:3], 0.25, **dict(opts, table=some[3]))
        for i, (a, b) in enumerate(zip(scored_attention_backward(do, state, need), full[1:])):
            assert (a is None) == (not need[i]) and (a is None or torch.equal(a, b)), (bits, i)
    with torch.autograd.graph.save_on_cpu():
        for a, b in zip(results(q, k, v, do, 0.25, opts), full):
            assert torch.equal(a, b)
    out = torch.utils.checkpoint.checkpoint(lambda *t: scored_attention(*t[:3], 0.25, **dict(opts, table=t[3])), *leaves,
                                            use_reentrant=False)
    for a, b in zip(torch.autograd.grad(out, leaves, do), full[1:]):
        assert torch.equal(a, b)
    out = scored_attention(q, k, v, 0.25, **opts)
    for _ in range(2):
        for a, b in zip(torch.autograd.grad(out, leaves, do, retain_graph=True), full[1:]):
            assert torch.equal(a, b)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, leaves, do, create_graph=True)
    with pytest.raises(RuntimeError):  # a saved tensor that has been written to
        out = scored_attention(q, k, v, 0.25, **opts)
        with torch.no_grad():
            k.add_(0)
        torch.autograd.grad(out, leaves, do)


@pytest.mark.parametrize("B, H, Lq, Lk", [(0, 2, 5, 5), (1, 0, 5, 5), (1, 2, 0, 5), (1, 2, 5, 0)])
def test_nothing(dev, B, H, Lq, Lk):
    case(f"empty {B} {H} {Lq} {Lk}")
    q, k, v, do = ref.inputs(0, B, H, H, Lq, Lk, 64, BF16, dev)
    for t in (q, k, v):
        t.requires_grad_()
    out = scored_attention(q, k, v, 0.2, cap=2.0)
    assert out.shape == q.shape and not out.any()
    for a, t in zip(torch.autograd.grad(out, (q, k, v), do), (q, k, v)):
        assert a.shape == t.shape and not a.any()
    with pytest.raises(ValueError):
        scored_attention_forward(q, k, v, 0.2)
    lengths = torch.zeros(B, 1, dtype=torch.int32, device=dev)
    assert row_ranges(lengths, Lk).shape == (B, Lk, 2)


def test_other_stream(dev):
    case("another stream")
    (q, k, v, do), opts = make("documents", BF16, dev)
    want = results(q, k, v, do, 0.25, opts)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x = [t.detach().clone().requires_grad_() for t in (q, k, v)]
        got = results(*x, do, 0.25, opts)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_two_steps_at_once(dev):
    case("two streams")
    calls = [make(n, BF16, dev) for n in ("split_keys", "causal_table")]
    want = [results(*x, 0.25, opts) for x, opts in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(4):
        for s, (x, opts), to in zip(streams, calls, got):
            with torch.cuda.stream(s):
                to.append(results(*[t.detach().requires_grad_() for t in x[:3]], x[3], 0.25,
                                  dict(opts, table=opts["table"].detach().requires_grad_())))
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        assert all(torch.equal(a, b) for o in outs for a, b in zip(o, w))


@pytest.mark.parametrize("name", ["documents", "split_keys", "mask_and_ranges"])
def test_captured_step(dev, name):
    case(f"captured {name}")
    (q, k, v, do), opts = make(name, BF16, dev)
    L = k.shape[2]
    q, k, v = (t.detach() for t in (q, k, v))
    lengths = torch.tensor([[L // 2, L // 3]], dtype=torch.int32, device=dev)
    if opts["table"] is not None:
        opts["table"] = opts["table"].detach()

    def step():
        o = dict(opts, ranges=row_ranges(lengths, L))
        out, state = scored_attention_forward(q, k, v, 0.25, **o)
        return (out, *(t for t in scored_attention_backward(do, state) if t is not None))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for turn, cut in enumerate((1, L // 5, 2 * L, L - 1)):
        for t, new in zip((q, k, v, do), ref.inputs(50 + turn, *q.shape[:2], k.shape[1], q.shape[2], L, q.shape[3], BF16, dev)):
            t.copy_(new)
        lengths.copy_(torch.tensor([[cut, L // 2]]))
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(held, want)):
            assert torch.equal(a, b), (turn, i)


def test_refusals(dev):
    case("refusals")
    q, k, v, do = ref.inputs(0, 2, 4, 2, 70, 90, 64, BF16, dev)
    table, buckets = torch.zeros(4, 4, device=dev), torch.zeros(9, dtype=torch.int32, device=dev)
    ranges = torch.zeros(2, 90, 2, dtype=torch.int32, device=dev)
    mask = torch.ones(2, 4, 2, 2, dtype=torch.bool, device=dev)
    slopes = torch.ones(4, device=dev)

    def refused(error, *qkv, scale=0.1, **opts):
        for f in (scored_attention, scored_attention_forward):
            with pytest.raises(error):
                f(*(qkv or (q, k, v)), scale, **opts)

    for scale in (0.0, -1.0, float("nan"), float("inf")):
        refused(ValueError, scale=scale)
    for cap in (0.0, -1.0, float("inf"), float("nan"), 1e-36):
        refused(ValueError, cap=cap)
    refused(ValueError, q.cpu(), k, v)
    refused(ValueError, q, k.cpu(), v)
    refused(ValueError, q[0], k, v)
    refused(ValueError, q, k, v[:, :, :50])
    refused(ValueError, q, k[:1], v[:1])
    refused(ValueError, q[:, :3], k, v)
    refused(TypeError, q, k.float(), v)
    refused(TypeError, q.double(), k.double(), v.double())
    refused(NotImplementedError, q[..., :32], k[..., :32], v[..., :32])
    refused(ValueError, slopes=slopes.double())
    refused(ValueError, slopes=slopes[:3])
    refused(ValueError, slopes=slopes.cpu())
    refused(ValueError, slopes=slopes.clone().requires_grad_())
    refused(ValueError, table=table)
    refused(ValueError, buckets=buckets)
    refused(ValueError, table=table[:, :3], buckets=buckets)
    refused(ValueError, table=table[:0], buckets=buckets)
    refused(TypeError, table=table.double(), buckets=buckets)
    refused(ValueError, table=table, buckets=buckets.long())
    refused(ValueError, table=table, buckets=buckets[:8])
    refused(ValueError, table=table, buckets=buckets.cpu())
    refused(NotImplementedError, table=table, buckets=torch.zeros(2 * 1025 + 1, dtype=torch.int32, device=dev))
    refused(ValueError, ranges=ranges.long())
    refused(ValueError, ranges=ranges[:, :80])
    refused(ValueError, ranges=ranges.cpu())
    refused(ValueError, ranges=ranges[:1].expand(3, -1, -1))
    refused(ValueError, block_mask=mask[0])
    refused(ValueError, block_mask=mask[..., :1])
    refused(ValueError, block_mask=mask.cpu())
    refused(ValueError, block_mask=mask[:, :3])
    refused(ValueError, q_start=2 ** 29)
    _, state = scored_attention_forward(q, k, v, 0.1)
    for bad in (do.cpu(), do.float(), do[:, :, :50]):
        with pytest.raises(ValueError):
            scored_attention_backward(bad, state)
    lengths = torch.tensor([[5, 6]], device=dev)
    for bad in (lambda: row_ranges(lengths.float(), 9), lambda: row_ranges(lengths[None], 9), lambda: row_ranges(lengths, -1),
                lambda: row_ranges(lengths[:, :0], 9), lambda: row_ranges(lengths, 2 ** 31), lambda: row_ranges(lengths, 9, frame=0),
                lambda: row_ranges(lengths, 9, window=-1), lambda: row_ranges(lengths, 9, causal=False, frame=2),
                lambda: row_ranges(lengths, 9, prefix=lengths.float()), lambda: row_ranges(lengths, 9, prefix=lengths.cpu()),
                lambda: row_ranges(lengths, 9, prefix=torch.zeros(3, dtype=torch.int32, device=dev))):
        with pytest.raises(ValueError):
            bad()
