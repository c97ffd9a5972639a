"""Operators of attention whose scores follow a rule besides the dot product, in training and over a
cache of keys: caps, distances, learned position biases, documents, prefixes.

A case names an operator:

  attend   `scored_attention` over `row_ranges` and its backward pass: softmax attention whose scores
           are capped by a tanh or lose a slope times the distance, where each key is seen by an
           interval of rows (documents packed in a row, causal by token or by frame, prefixes that
           all rows see, windows) and by the blocks of a mask; then the gradients of q, k and v
  relate   the same with a learned bias by buckets of the distance, and the gradient of its table
  cached   `cached_attention`: new tokens of each sequence over its cache of keys and values
  shared   the same where all sequences begin with one prefix, whose keys and values are held once

Sizes are the package's own geometries (226 text + 13 x 30 x 45 video tokens with 30 heads, 224 +
11 x 48 x 85 with 48), its kernel sweep's shortest length and its small test clip; `draw` spreads them
from one token to those, over odd lengths, head layouts, rules and types.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
MOST_PAIRS = 15 * 17776 ** 2  # query-key pairs of the largest training case, seen or not
MOST_FLOPS = 2.2e12  # and its operations on the seen ones
MOST_VALUES = 2 * 8 * 30 * 17776 * 64  # cached keys and values of the largest serving case

TRAIN = {"B": 1, "H": 2, "Hk": 2, "D": 64, "cap": 0.0, "slopes": False, "buckets": 0, "radius": 0, "causal": True,
         "docs": 1, "pad": 0, "prefix": 0, "frame": 1, "window": 0, "keep": 1.0, "q_start": 0}
SERVE = {"cap": 0.0, "slopes": False, "buckets": 0, "radius": 0, "window": 0, "prefix": 0, "least": 0.5}


def listed():
    return [
        # A small layer trained in fp32 with capped scores, causally: latency counts.
        {"name": "attend_fp32_2k", "op": "attend", **TRAIN, "dtype": "fp32", "Lq": 2048, "Lk": 2048, "cap": 30.0},
        # Half the heads of a full-size video layer that is generated frame by frame: every token sees the
        # text, its own frame and those before.
        {"name": "attend_bf16_frames", "op": "attend", **TRAIN, "dtype": "bf16", "H": 15, "Hk": 15, "Lq": 17776, "Lk": 17776,
         "prefix": 226, "frame": 1350},
        # Seven clips of unlike length packed into one row, 128-wide heads that share keys in threes.
        {"name": "attend_fp16_packed", "op": "attend", **TRAIN, "dtype": "fp16", "H": 15, "Hk": 5, "D": 128, "Lq": 8229,
         "Lk": 8229, "docs": 7, "pad": 100, "cap": 50.0},
        # Distances instead of positions, over a window and the blocks of a mask.
        {"name": "attend_bf16_slopes", "op": "attend", **TRAIN, "dtype": "bf16", "B": 2, "H": 12, "Hk": 12, "Lq": 4546,
         "Lk": 4546, "slopes": True, "window": 1350, "prefix": 226, "keep": 0.5},
        # The shortest sequence of the kernel sweep, every token seeing every other.
        {"name": "relate_bf16_dense", "op": "relate", **TRAIN, "dtype": "bf16", "B": 2, "H": 30, "Hk": 30, "Lq": 2560,
         "Lk": 2560, "buckets": 32, "radius": 128, "causal": False},
        # A small clip in fp32, causally.
        {"name": "relate_fp32_clip", "op": "relate", **TRAIN, "dtype": "fp32", "B": 1, "H": 4, "Hk": 4, "Lq": 526, "Lk": 526,
         "buckets": 32, "radius": 128},
        # Queries of the last frame against four frames and their caption.
        {"name": "relate_fp16_cross", "op": "relate", **TRAIN, "dtype": "fp16", "B": 2, "H": 12, "Hk": 6, "D": 128,
         "Lq": 1350, "Lk": 5626, "q_start": 4276, "buckets": 64, "radius": 800, "causal": False},
        # One new token behind a small clip: latency counts.
        {"name": "cached_bf16_clip", "op": "cached", **SERVE, "dtype": "bf16", "B": 1, "H": 30, "Hk": 30, "Ln": 1, "L": 526,
         "D": 64, "slopes": True},
        # One new token of each of eight sequences at the smaller video size.
        {"name": "cached_bf16_video", "op": "cached", **SERVE, "dtype": "bf16", "B": 8, "H": 30, "Hk": 30, "Ln": 1, "L": 17776,
         "D": 64, "cap": 30.0},
        # Four proposed tokens of each of four long sequences, six query heads to a key head.
        {"name": "cached_fp16_few", "op": "cached", **SERVE, "dtype": "fp16", "B": 4, "H": 48, "Hk": 8, "Ln": 4, "L": 45104,
         "D": 128, "buckets": 32, "radius": 128},
        # Thirty-two continuations of one video: a token of each.
        {"name": "shared_bf16_video", "op": "shared", **SERVE, "dtype": "bf16", "B": 32, "H": 30, "Hk": 30, "Ln": 1, "L": 1350,
         "D": 64, "prefix": 17776, "least": 0.0, "cap": 30.0},
        # Three new tokens of four answers to one caption.
        {"name": "shared_fp16_caption", "op": "shared", **SERVE, "dtype": "fp16", "B": 4, "H": 12, "Hk": 4, "Ln": 3, "L": 77,
         "D": 128, "prefix": 226, "least": 0.0, "slopes": True},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "relate", "cached", "cached", "shared"])
    if op in ("attend", "relate"):
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        c = {"op": op, **TRAIN, "dtype": dtype, "B": rng.randint(1, 2), "Hk": rng.randint(1, 10), "D": rng.choice([64, 64, 128])}
        c["H"] = c["Hk"] * rng.choice([1, 1, 2, 3])
        most = 4000 if dtype == "fp32" else 17776
        c["Lq"] = c["Lk"] = _log_uniform(rng, 8, most)
        c["cap"] = rng.choice([0.0, 0.0, 20.0, 50.0])
        if op == "relate":
            c["buckets"], c["radius"] = rng.choice([(32, 128), (32, 128), (16, 64), (64, 800), (9, 7)])
            c["causal"] = rng.random() < 0.3
            if rng.random() < 0.4:  # all keys of another, longer sequence: every pair is seen
                c["causal"] = False
                c["Lk"] = _log_uniform(rng, c["Lq"], most)
                c["q_start"] = c["Lk"] - c["Lq"]
        else:
            c["slopes"] = rng.random() < 0.4
            c["causal"] = rng.random() < 0.8
        if c["Lk"] == c["Lq"]:
            c["docs"] = min(rng.choice([1, 1, 2, 5, 9]), c["Lq"] // 4)
            c["pad"] = rng.choice([0, 0, c["Lq"] // 9])
            c["prefix"] = rng.choice([0, 77, 226])
            c["frame"] = rng.choice([1, 1, 45, 1350]) if c["causal"] else 1
            c["window"] = rng.choice([0, 0, 100, 1350]) if c["frame"] == 1 else 0
        c["keep"] = rng.choice([1.0, 1.0, round(rng.uniform(0.1, 0.9), 2)])
        while c["B"] * c["H"] * c["Lq"] * c["Lk"] > MOST_PAIRS or work(c)["flops"] > MOST_FLOPS:
            rep = c["H"] // c["Hk"]
            c["B"], c["Hk"] = 1, max(1, c["Hk"] // 2)
            c["H"] = c["Hk"] * (rep if c["Hk"] > 1 else 1)
        return c
    c = {"op": op, **SERVE, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "B": _log_uniform(rng, 1, 32),
         "Hk": rng.randint(1, 16), "Ln": rng.choice([1, 1, 1, 2, 5, 8]), "L": _log_uniform(rng, 16, 45104),
         "D": rng.choice([64, 64, 128])}
    c["H"] = c["Hk"] * rng.choice([1, 1, 3, 6])
    c["cap"] = rng.choice([0.0, 0.0, 20.0, 50.0])
    rule = rng.choice(["none", "slopes", "table"])
    c["slopes"] = rule == "slopes"
    if rule == "table":
        c["buckets"], c["radius"] = rng.choice([(32, 128), (16, 64), (64, 800)])
    c["window"] = rng.choice([0, 0, 0, 1350])
    c["least"] = rng.choice([0.0, 0.5, 1.0])
    if op == "shared":
        c["prefix"] = _log_uniform(rng, 1, 17776)
    size = {"fp32": 2}.get(c["dtype"], 1)
    while (2 * c["B"] * c["Hk"] * c["L"] * c["D"] * size > MOST_VALUES
           or c["B"] * c["H"] * c["Ln"] * (c["L"] + c["prefix"]) > 3e8):
        c["B"], c["L"] = max(1, c["B"] // 2), c["L"] // 2 + 1
    return c


# ---- inputs ----------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _wave(L, D):
    """[L, D]: unit-norm sinusoids of the token's index, by which tokens find their neighbours."""
    n = torch.arange(L, device="cuda", dtype=torch.float64)[:, None]
    ang = n * 10000.0 ** (-2.0 * torch.arange(D // 2, device="cuda", dtype=torch.float64) / D)
    return torch.stack((ang.sin(), ang.cos()), dim=-1).reshape(L, D).float() / math.sqrt(D / 2)


def _lengths(case, turn=0):
    """The documents' lengths, in proportion to 1, 2, 3 .. and turned by `turn` places."""
    n, L = case["docs"], case["Lq"] - case["pad"]
    ends = [L * i * (i + 1) // (n * (n + 1)) for i in range(n + 1)]
    sizes = [b - a for a, b in zip(ends, ends[1:])]
    turn %= n
    return sizes[turn:] + sizes[:turn]


def _slopes(H):
    """One for each head, from 2^-1 to 2^-8."""
    return torch.exp2(-8.0 * torch.arange(1, H + 1, device="cuda", dtype=torch.float64) / H).float()


def _distance_buckets(n, radius, bidirectional):
    """The bucket of each distance i - j from -radius to radius: the nearest half of them (of each
    side's) hold one distance each, the others grow in proportion to it."""
    side = (n - 1) // 2 if bidirectional else n - 1
    exact = max(1, side // 2)
    places = []
    for d in range(-radius, radius + 1):
        a = abs(d) if bidirectional else max(d, 0)
        if a > exact:
            a = min(side, exact + int((side - exact) * math.log(a / exact) / math.log(radius / exact)) + 1)
        places.append(a if d >= 0 or not bidirectional else side + a)
    return torch.tensor(places, dtype=torch.int32, device="cuda")


def _rule(case, state, g, bidirectional):
    """The score rule's parameters: the same in training and serving."""
    H, dtype = case["H"], DTYPES[case["dtype"]]
    state["cap"] = case["cap"] or None
    state["slopes"] = _slopes(H) if case["slopes"] else None
    state["table"] = state["buckets"] = None
    if case["buckets"]:
        state["buckets"] = _distance_buckets(case["buckets"], case["radius"], bidirectional)
        state["table"] = _normal(g, case["buckets"], H).to(dtype)
    state["scale"] = 1.0 / math.sqrt(case["D"])
    if case["cap"]:  # scores that the cap bends
        state["scale"] *= 3.0


def _prepare_train(case, seed):
    g = _generator(seed)
    B, H, Hk, Lq, Lk, D = (case[x] for x in ("B", "H", "Hk", "Lq", "Lk", "D"))
    dtype = DTYPES[case["dtype"]]
    wave = 2 * _wave(Lk, D)
    state = {"q": _normal(g, B, H, Lq, D) + wave[Lk - Lq:], "k": _normal(g, B, Hk, Lk, D) + wave, "v": _normal(g, B, Hk, Lk, D)}
    state = {n: x.to(dtype).requires_grad_() for n, x in state.items()}
    state["dout"] = _normal(g, B, H, Lq, D).to(dtype)
    _rule(case, state, g, not case["causal"])
    if state["table"] is not None:
        state["table"].requires_grad_()
    state["lengths"] = None
    if Lq == Lk:
        turn = random.Random(seed)
        state["lengths"] = torch.tensor([_lengths(case, turn.randrange(case["docs"])) for _ in range(B)], dtype=torch.int32,
                                        device="cuda")
    state["prefix"] = None
    if case["prefix"]:
        state["prefix"] = torch.full_like(state["lengths"], case["prefix"])
    state["mask"] = None
    if case["keep"] < 1.0:
        nq, nk, nt = math.ceil(Lq / 64), math.ceil(Lk / 64), math.ceil(case["prefix"] / 64)
        mask = torch.rand(B, H, nq, nk, device="cuda", generator=g) < case["keep"]
        mask |= torch.eye(nq, nk, dtype=torch.bool, device="cuda")
        mask[..., :nt] = True
        state["mask"] = mask
    for x in ("causal", "frame", "window", "q_start"):
        state[x] = case[x]
    return state


def _prepare_serve(case, seed):
    g = _generator(seed)
    B, H, Hk, Ln, L, D = (case[x] for x in ("B", "H", "Hk", "Ln", "L", "D"))
    dtype = DTYPES[case["dtype"]]
    state = {"q": _normal(g, B, H, Ln, D).to(dtype), "k": _normal(g, B, Hk, L, D).to(dtype), "v": _normal(g, B, Hk, L, D).to(dtype)}
    _rule(case, state, g, False)
    least = min(L, max(Ln, int(case["least"] * L)))
    state["lengths"] = torch.randint(least, L + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
    state["window"], state["prefix"] = case["window"], None
    if case["prefix"]:
        state["prefix"] = tuple(_normal(g, Hk, case["prefix"], D).to(dtype) for _ in range(2))
    return state


def prepare(case, seed):
    make = _prepare_train if case["op"] in ("attend", "relate") else _prepare_serve
    return dict(make(case, seed), op=case["op"])


# ---- the operators -----------------------------------------------------------------------------


def _train(s):
    from sparseattnfunctions_amd.utils.scored_attn import row_ranges, scored_attention

    ranges = None
    if s["lengths"] is not None:
        ranges = row_ranges(s["lengths"], s["q"].shape[2], causal=s["causal"], prefix=s["prefix"], frame=s["frame"],
                            window=s["window"])
    out = scored_attention(s["q"], s["k"], s["v"], s["scale"], cap=s["cap"], slopes=s["slopes"], table=s["table"],
                           buckets=s["buckets"], ranges=ranges, block_mask=s["mask"], q_start=s["q_start"])
    wanted = (s["q"], s["k"], s["v"]) + (() if s["table"] is None else (s["table"],))
    return (out.detach(), *torch.autograd.grad(out, wanted, s["dout"]))


def _plain_ranges(s, L):
    """(from, until) [B, L] of each key's rows."""
    sizes = s["lengths"].long()
    ends = sizes.cumsum(1)
    at = torch.arange(L, device="cuda")
    doc = (at >= ends[:, :, None]).sum(1)  # behind the last document: their number
    inside = doc < sizes.shape[1]
    doc = doc.clamp_max(sizes.shape[1] - 1)
    end = ends.gather(1, doc)
    begin = end - sizes.gather(1, doc)
    body = begin if s["prefix"] is None else torch.minimum(begin + s["prefix"].long().gather(1, doc), end)
    head = at < body
    first, until = begin, end
    if s["causal"]:
        first = torch.where(head, begin, body + (at - body) // s["frame"] * s["frame"])
    if s["window"]:
        until = torch.where(head, end, torch.minimum(end, at + s["window"]))
        if not s["causal"]:
            first = torch.where(head, begin, torch.maximum(begin, at - s["window"] + 1))
    return torch.where(inside, first, 0), torch.where(inside, until, 0)


def _distances(s, Lq, Lk):
    return torch.arange(Lq, device="cuda")[:, None] + s["q_start"] - torch.arange(Lk, device="cuda")


def _plain_train(s):
    with torch.no_grad():
        q, do = s["q"].float(), s["dout"].float()
        B, H, Lq, D = q.shape
        Hk, Lk = s["k"].shape[1:3]
        k, v = (s[n].float().repeat_interleave(H // Hk, dim=1) for n in ("k", "v"))
        x = (q @ k.transpose(2, 3)).mul_(s["scale"])
        bent = None
        if s["cap"] is not None:
            x.div_(s["cap"]).tanh_()
            bent = 1 - x * x
            x.mul_(s["cap"])
        far = _distances(s, Lq, Lk)
        if s["slopes"] is not None:
            x.sub_(s["slopes"][:, None, None] * far.abs())
        if s["table"] is not None:
            radius = s["buckets"].numel() // 2
            place = s["buckets"].long()[far.clamp(-radius, radius) + radius]
            x.add_(s["table"].float()[place].permute(2, 0, 1))
        if s["lengths"] is not None:
            first, until = _plain_ranges(s, Lk)
            at = torch.arange(Lq, device="cuda")[:, None]
            x.masked_fill_(~((at >= first[:, None]) & (at < until[:, None]))[:, None], float("-inf"))
        if s["mask"] is not None:
            seen = s["mask"].repeat_interleave(64, dim=2)[:, :, :Lq].repeat_interleave(64, dim=3)[..., :Lk]
            x.masked_fill_(~seen, float("-inf"))
            del seen
        top = x.amax(dim=3, keepdim=True)
        x.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
        total = x.sum(dim=3, keepdim=True)
        p = x.div_(torch.where(total == 0, 1.0, total))  # a row without a key: zeros
        out = p @ v
        dv = p.transpose(2, 3) @ do
        ds = (do @ v.transpose(2, 3)).sub_((do * out).sum(dim=3, keepdim=True)).mul_(p)
        del p, x
        extra = ()
        if s["table"] is not None:
            # by distance first: each row one place further left than the row above it
            by_far = torch.nn.functional.pad(ds.sum(dim=0).flip(1), (0, Lq)).flatten(1)[:, :Lq * (Lk + Lq - 1)]
            by_far = by_far.view(H, Lq, -1).sum(dim=1, dtype=torch.float64)
            far = s["q_start"] + Lq - 1 - torch.arange(Lk + Lq - 1, device="cuda")
            place = s["buckets"].long()[far.clamp(-radius, radius) + radius]
            extra = (torch.zeros(s["table"].shape, dtype=torch.float64, device="cuda").index_add_(0, place, by_far.T)
                     .to(s["table"].dtype),)
        if bent is not None:
            ds.mul_(bent)
            del bent
        dq, dk = (ds @ k).mul_(s["scale"]), (ds.transpose(2, 3) @ q).mul_(s["scale"])
        dk, dv = (t.view(B, Hk, H // Hk, Lk, D).sum(dim=2) for t in (dk, dv))
        return tuple(t.to(s["q"].dtype) for t in (out, dq, dk, dv)) + extra


def _serve(s):
    from sparseattnfunctions_amd.utils.cached_attn import cached_attention

    return cached_attention(s["q"], s["k"], s["v"], s["lengths"], s["scale"], cap=s["cap"], slopes=s["slopes"],
                            table=s["table"], buckets=s["buckets"], window=s["window"], prefix=s["prefix"])


def _plain_serve(s):
    q, k, v = (s[n].float() for n in ("q", "k", "v"))
    B, H, Ln, D = q.shape
    Hk, L = k.shape[1:3]
    Lp = 0 if s["prefix"] is None else s["prefix"][0].shape[1]
    rows = q.view(B, Hk, H // Hk * Ln, D)
    x = (rows @ k.transpose(2, 3)).view(B, H, Ln, L)
    if Lp:  # all sequences' rows against the one prefix
        kp, vp = (t.float() for t in s["prefix"])
        rows = rows.transpose(0, 1).reshape(Hk, -1, D)
        first = (rows @ kp.transpose(1, 2)).view(Hk, B, H // Hk * Ln, Lp).transpose(0, 1).reshape(B, H, Ln, Lp)
        x = torch.cat((first, x), dim=3)
    x = x * s["scale"]
    if s["cap"] is not None:
        x = s["cap"] * (x / s["cap"]).tanh()
    own_place = s["lengths"].long()[:, None] - Ln + torch.arange(Ln, device="cuda")  # [B, Ln]
    far = (Lp + own_place)[:, :, None] - torch.arange(Lp + L, device="cuda")
    if s["slopes"] is not None:
        x = x - s["slopes"][:, None, None] * far.abs()[:, None]
    if s["table"] is not None:
        radius = s["buckets"].numel() // 2
        place = s["buckets"].long()[far.clamp(-radius, radius) + radius]
        x = x + s["table"].float()[place].permute(0, 3, 1, 2)
    seen = (far >= 0) & (own_place >= 0)[:, :, None]
    if s["window"]:
        seen &= far < s["window"]
    x = x.masked_fill(~seen[:, None], float("-inf"))
    top = x.amax(dim=3, keepdim=True)
    x = (x - torch.where(top == float("-inf"), 0.0, top)).exp()
    total = x.sum(dim=3, keepdim=True)
    x = x / torch.where(total == 0, 1.0, total)
    out = (x[..., Lp:].reshape(B, Hk, -1, L) @ v).view(B, H, Ln, D)
    if Lp:
        mass = x[..., :Lp].reshape(B, Hk, -1, Lp).transpose(0, 1).reshape(Hk, -1, Lp)
        out = out + (mass @ vp).view(Hk, B, -1, D).transpose(0, 1).reshape(B, H, Ln, D)
    return out.to(s["q"].dtype)


def run(state):
    if state["op"] in ("attend", "relate"):
        return _train(state) if own else _plain_train(state)
    return _serve(state) if own else _plain_serve(state)


# ---- what each operator cannot do without --------------------------------------------------------


def _seen_pairs(case):
    """Query-key pairs of one head that the ranges leave."""
    if case["Lq"] != case["Lk"]:
        return case["Lq"] * case["Lk"]
    pairs = 0
    for n in _lengths(case):
        head = min(case["prefix"], n)
        pairs += head * n
        if not case["causal"] and not case["window"]:
            pairs += (n - head) * n
            continue
        for first in range(0, n - head, case["frame"]):
            keys = min(case["frame"], n - head - first)
            if not case["causal"]:
                pairs += min(n, head + first + case["window"]) - max(0, head + first - case["window"] + 1)
            elif case["window"]:  # (frames of one token)
                pairs += min(n - head - first, case["window"])
            else:
                pairs += keys * (n - head - first)
    return pairs


def work(case):
    B, H, Hk, D, size = case["B"], case["H"], case["Hk"], case["D"], BYTES[case["dtype"]]
    if case["op"] in ("attend", "relate"):
        Lq, Lk = case["Lq"], case["Lk"]
        moved = B * D * size * 4 * (H * Lq + Hk * Lk)  # q, out, dout, dq; k, v, dk, dv
        if case["keep"] < 1.0:
            moved += B * H * math.ceil(Lq / 64) * math.ceil(Lk / 64)
        kept = case["keep"] + (1 - case["keep"]) * min(1.0, (64 + 2 * case["prefix"]) / Lk)  # the diagonal and the prefix
        return {"bytes": moved, "flops": int(14 * D * B * H * _seen_pairs(case) * kept)}
    least = min(case["L"], max(case["Ln"], int(case["least"] * case["L"])))
    keys = (least + case["L"]) / 2
    first = case["prefix"]
    if case["window"]:
        keys, first = min(keys, case["window"]), max(0, min(first, case["window"] - keys))
    moved = 2 * D * size * (B * H * case["Ln"] + Hk * (B * keys + first))
    return {"bytes": int(moved), "flops": int(4 * D * B * H * case["Ln"] * (keys + first))}


# ---- 64-bit values -------------------------------------------------------------------------------


def _exact_scores(s, x, far, h):
    """(the rule's scores of head h, and their derivative by the product) for x = q k^T and the distances."""
    x = x * s["scale"]
    slope = torch.ones((), dtype=torch.float64, device="cuda")
    if s["cap"] is not None:
        e = torch.exp(-2.0 * (x / s["cap"]).abs())
        t = torch.sign(x) * (1 - e) / (1 + e)
        x, slope = s["cap"] * t, 4 * e / (1 + e) ** 2
    if s["slopes"] is not None:
        x = x - s["slopes"][h].double() * far.abs()
    place = None
    if s["table"] is not None:
        radius = (s["buckets"].numel() - 1) // 2
        place = s["buckets"][torch.clamp(far, -radius, radius) + radius].long()
        x = x + s["table"].detach()[:, h].double()[place]
    return x, slope * s["scale"], place


def _exact_interval(case, lengths, prefix, L):
    """Python's lists of each key's first row and the one behind its last, document by document."""
    first, until = [0] * L, [0] * L
    begin = 0
    for n, size in enumerate(lengths):
        end = begin + size
        text = min(end, begin + (prefix[n] if prefix is not None else 0))
        for j in range(begin, end):
            first[j], until[j] = begin, end
            if j < text:
                continue
            if case["causal"]:
                first[j] = j - (j - text) % case["frame"]
            elif case["window"]:
                first[j] = max(begin, j + 1 - case["window"])
            if case["window"]:
                until[j] = min(end, j + case["window"])
        begin = end
    return torch.tensor([first, until], device="cuda")


def _exact_train(case, s):
    """Head by head and some query rows at a time: probabilities, then the chain rule."""
    q, k, v, do = (s[n].detach().double() for n in ("q", "k", "v", "dout"))
    B, H, Lq, D = q.shape
    Hk, Lk = k.shape[1:3]
    out, dq = torch.zeros_like(q), torch.zeros_like(q)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    dtable = None if s["table"] is None else torch.zeros(s["table"].shape, dtype=torch.float64, device="cuda")
    column = torch.arange(Lk, device="cuda")
    for b in range(B):
        spans = None
        if s["lengths"] is not None:
            prefix = None if s["prefix"] is None else s["prefix"][b].tolist()
            spans = _exact_interval(case, s["lengths"][b].tolist(), prefix, Lk)
        for h in range(H):
            g = h * Hk // H
            for r0 in range(0, Lq, 4096):
                r = slice(r0, min(r0 + 4096, Lq))
                row = torch.arange(r.start, r.stop, device="cuda")[:, None]
                x, slope, place = _exact_scores(s, torch.mm(q[b, h, r], k[b, g].T), row + s["q_start"] - column, h)
                if spans is not None:
                    x = torch.where((spans[0] <= row) & (row < spans[1]), x, float("-inf"))
                if s["mask"] is not None:
                    x = torch.where(s["mask"][b, h][row[:, 0] // 64][:, column // 64], x, float("-inf"))
                prob = torch.nan_to_num(torch.softmax(x, dim=1), nan=0.0)
                o = torch.mm(prob, v[b, g])
                dprob = torch.mm(do[b, h, r], v[b, g].T)
                dx = prob * (dprob - (prob * dprob).sum(dim=1, keepdim=True))
                if dtable is not None:
                    for n in range(dtable.shape[0]):
                        dtable[n, h] += torch.where(place == n, dx, 0.0).sum()
                dx = dx * slope
                out[b, h, r] = o
                dq[b, h, r] = torch.mm(dx, k[b, g])
                dk[b, g] += torch.mm(dx.T, q[b, h, r])
                dv[b, g] += torch.mm(prob.T, do[b, h, r])
    return (out, dq, dk, dv) + (() if dtable is None else (dtable,))


def _exact_serve(s):
    """Sequence by sequence and head by head, over the keys that there are."""
    q = s["q"].double()
    B, H, Ln, D = q.shape
    Hk = s["k"].shape[1]
    out = torch.zeros_like(q)
    for b, n in enumerate(s["lengths"].tolist()):
        for h in range(H):
            g = h * Hk // H
            keys, values = s["k"][b, g, :n].double(), s["v"][b, g, :n].double()
            if s["prefix"] is not None:
                keys, values = (torch.cat((t[g].double(), x)) for t, x in zip(s["prefix"], (keys, values)))
            place = keys.shape[0] - Ln + torch.arange(Ln, device="cuda")[:, None]
            far = place - torch.arange(keys.shape[0], device="cuda")
            x = _exact_scores(s, torch.mm(q[b, h], keys.T), far, h)[0]
            seen = (far >= 0) & (place >= keys.shape[0] - n)
            if s["window"]:
                seen &= far < s["window"]
            x = torch.where(seen, x, float("-inf"))
            out[b, h] = torch.mm(torch.nan_to_num(torch.softmax(x, dim=1), nan=0.0), values)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_train(case, s) if case["op"] in ("attend", "relate") else _exact_serve(s)
