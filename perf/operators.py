"""Operators of a training or generating loop around the package's attention: block-sparse
attention with its gradients, and rotary positions of its queries and keys.

A case names an operator:

  attention  `block_sparse_train_fn` and its backward pass: softmax attention over the 64 x 64
             blocks that a mask keeps, then the gradients of q, k and v
  rotate     `apply_rotary`: queries and keys turned by the angles of their positions
  turn       `apply_rotary` and its backward pass
  table      `rotary_table`: the cosines and sines of a sequence's positions

Sizes are the package's own geometries (226 text + 13 x 30 x 45 video tokens with 30 heads, 224 +
11 x 48 x 85 with 48), its small fp32 configuration and its kernel sweep's shortest length;
`draw` spreads them from one token to those, over odd lengths, other densities and types.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
MOST_PAIRS = 15 * 17776 ** 2  # query-key pairs of the largest attention case, kept or not
MOST_FLOPS = 9.4e11  # and its operations on the kept ones
MOST_VALUES = 2 * 48 * 45104 * 64  # query and key values of the largest rotary case


def listed():
    return [
        # A small layer trained in fp32, the package's CPU-runnable configuration: latency counts.
        {"name": "attention_fp32_2k", "op": "attention", "dtype": "fp32", "B": 1, "H": 2, "Lq": 2048, "Lk": 2048, "D": 64,
         "keep": 0.25, "text": 0, "bias": False, "empty": 0.0},
        # The shortest sequence of the kernel sweep with every block kept, as in the dense warm-up steps.
        {"name": "attention_bf16_dense", "op": "attention", "dtype": "bf16", "B": 2, "H": 30, "Lq": 2560, "Lk": 2560,
         "D": 64, "keep": 1.0, "text": 0, "bias": False, "empty": 0.0},
        # fp16 training with 128-wide heads, at a length that fills no whole block.
        {"name": "attention_fp16_d128", "op": "attention", "dtype": "fp16", "B": 1, "H": 15, "Lq": 8229, "Lk": 8229,
         "D": 128, "keep": 0.35, "text": 0, "bias": False, "empty": 0.0},
        # Half the heads of a full-size video layer, a fifth of the blocks and all text rows and columns.
        {"name": "attention_bf16_18k", "op": "attention", "dtype": "bf16", "B": 1, "H": 15, "Lq": 17776, "Lk": 17776,
         "D": 64, "keep": 0.2, "text": 226, "bias": False, "empty": 0.0},
        # Queries of one frame against four and their captions, whose padding a key bias masks; some
        # query blocks keep no block at all.
        {"name": "attention_bias_cross", "op": "attention", "dtype": "bf16", "B": 2, "H": 12, "Lq": 1350, "Lk": 5626,
         "D": 64, "keep": 0.3, "text": 226, "bias": True, "empty": 0.1},
        # One new token of each of eight sequences, each at a position of its own.
        {"name": "rotate_one_token", "op": "rotate", "dtype": "bf16", "B": 8, "H": 30, "Hk": 30, "L": 1, "D": 64,
         "rot": 64, "layout": "half", "skip": 0, "rows": "batch", "memory": "blhd"},
        # A layer of a denoising step at the smaller video size: text tokens stay as they are.
        {"name": "rotate_2b", "op": "rotate", "dtype": "bf16", "B": 2, "H": 30, "Hk": 30, "L": 17776, "D": 64, "rot": 64,
         "layout": "interleaved", "skip": 226, "rows": "none", "memory": "bhld"},
        # fp32 heads of which three quarters turn, keys with fewer heads, tokens in another order.
        {"name": "rotate_fp32_part", "op": "rotate", "dtype": "fp32", "B": 1, "H": 15, "Hk": 5, "L": 8229, "D": 128,
         "rot": 96, "layout": "half", "skip": 0, "rows": "shared", "memory": "bhld"},
        # A training step's layer at the larger video size, and back.
        {"name": "turn_15_5b", "op": "turn", "dtype": "bf16", "B": 1, "H": 48, "Hk": 48, "L": 45104, "D": 64, "rot": 64,
         "layout": "interleaved", "skip": 224, "rows": "none", "memory": "blhd"},
        # A short fp16 clip in training.
        {"name": "turn_fp16_short", "op": "turn", "dtype": "fp16", "B": 2, "H": 30, "Hk": 30, "L": 1576, "D": 64,
         "rot": 32, "layout": "half", "skip": 226, "rows": "none", "memory": "bhld"},
        # The table of one frame's grid, and of a text context eight times the trained one.
        {"name": "table_frame", "op": "table", "axes": "16,24,24", "L": 1350, "theta": 10000.0, "scaling": "none",
         "factor": 1.0, "start": 0, "kind": "float"},
        {"name": "table_long", "op": "table", "axes": "128", "L": 45104, "theta": 500000.0, "scaling": "yarn",
         "factor": 8.0, "start": 1000000, "kind": "int"},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "rotate", "turn", "table"])
    if op == "attention":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        c = {"op": op, "dtype": dtype, "B": rng.randint(1, 2), "H": rng.randint(1, 30), "D": rng.choice([64, 64, 128])}
        most = 4000 if dtype == "fp32" else 17776
        # (with a single key every weight is 1, and the gradients of q and k are rounding errors around 0)
        c["Lq"] = _log_uniform(rng, 2, most)
        c["Lk"] = c["Lq"] if rng.random() < 0.6 else _log_uniform(rng, 2, most)
        if rng.random() < 0.1:
            c["Lq"] = 1
        c["keep"] = round(rng.uniform(0.05, 1.0), 3)
        c["text"] = rng.choice([0, 0, 77, 226])
        c["bias"] = dtype != "fp32" and rng.random() < 0.3
        c["empty"] = rng.choice([0.0, 0.0, 0.1, 0.5])
        while c["B"] * c["H"] * c["Lq"] * c["Lk"] > MOST_PAIRS or work(c)["flops"] > MOST_FLOPS:
            if c["B"] == c["H"] == 1:
                c["keep"] /= 2
            c["B"], c["H"] = 1, max(1, c["H"] // 2)
        return c
    if op == "table":
        axes = rng.choice(["16,24,24", "64", "128", "96", "32,48,48", "22,22,20"])
        return {"op": op, "axes": axes, "L": _log_uniform(rng, 1, 65536), "theta": rng.choice([100.0, 10000.0, 500000.0]),
                "scaling": rng.choice(["none", "linear", "ntk", "yarn"]), "factor": round(rng.uniform(1.0, 16.0), 2),
                "start": rng.choice([0, 0, _log_uniform(rng, 1, 4000000)]), "kind": rng.choice(["int", "float"])}
    D = rng.choice([64, 64, 96, 128])
    c = {"op": op, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "B": rng.randint(1, 4), "D": D,
         "L": _log_uniform(rng, 1, 45104), "rot": rng.choice([D, D, D // 2, D - 16, 20])}
    c["Hk"] = rng.randint(1, 16)
    c["H"] = c["Hk"] * rng.randint(1, 48 // c["Hk"])
    size = {"fp32": 2}.get(c["dtype"], 1)
    while c["B"] * (c["H"] + c["Hk"]) * c["L"] * D * size > MOST_VALUES:
        c["B"], c["L"] = max(1, c["B"] // 2), c["L"] // 2 + 1
    c["layout"] = rng.choice(["interleaved", "half"])
    c["rows"] = rng.choice(["none", "none", "shared", "batch"])
    c["skip"] = rng.choice([0, min(226, c["L"] // 3)]) if c["rows"] == "none" else 0
    c["memory"] = rng.choice(["bhld", "blhd"])
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


def _block_mask(case, g):
    """Random blocks, the diagonal, the text's block rows and columns; some rows with nothing."""
    nq, nk, tb = math.ceil(case["Lq"] / 64), math.ceil(case["Lk"] / 64), math.ceil(case["text"] / 64)
    mask = torch.rand(case["B"], case["H"], nq, nk, device="cuda", generator=g) < case["keep"]
    mask |= torch.eye(nq, nk, dtype=torch.bool, device="cuda")
    mask[:, :, :tb] = True
    mask[..., :tb] = True
    mask &= torch.rand(case["B"], case["H"], nq, 1, device="cuda", generator=g) >= case["empty"]
    return mask


def _prepare_attention(case, seed):
    g = _generator(seed)
    B, H, Lq, Lk, D, dtype = (case[x] for x in ("B", "H", "Lq", "Lk", "D", "dtype"))
    state = {"q": _normal(g, B, H, Lq, D) + 2 * _wave(Lq, D), "k": _normal(g, B, H, Lk, D) + 2 * _wave(Lk, D),
             "v": _normal(g, B, H, Lk, D)}
    state = {n: x.to(DTYPES[dtype]).requires_grad_() for n, x in state.items()}
    state["bias"] = None
    if case["bias"]:  # keys weighted by the tokens they stand for, and each batch's padding masked out
        bias = torch.randint(1, 5, (B, 1, Lk), device="cuda", generator=g).float().log()
        padded = torch.randint(1, case["text"] + 2, (B, 1, 1), device="cuda", generator=g)
        at = torch.arange(Lk, device="cuda")
        state["bias"] = bias.masked_fill_((at < case["text"]) & (at >= padded), float("-inf"))
    state["mask"] = _block_mask(case, g)
    state["dout"] = _normal(g, B, H, Lq, D).to(DTYPES[dtype])
    state["scale"] = 1.0 / math.sqrt(D)
    state["text_blocks"] = math.ceil(case["text"] / 64)
    return state


def _inverse_frequencies(dims, theta, scaling, factor, trained):
    """Radians per position of an axis of `dims` values, and the tables' common factor."""
    freq = theta ** (-torch.arange(0, dims, 2, dtype=torch.float64) / dims)
    if scaling == "linear":
        return freq / factor, 1.0
    if scaling == "ntk":
        return (theta * factor ** (dims / max(dims - 2, 1))) ** (-torch.arange(0, dims, 2, dtype=torch.float64) / dims), 1.0
    if scaling == "yarn":  # turns over the trained length decide between the two
        turns = trained * freq / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return freq * keep + freq / factor * (1 - keep), 0.1 * math.log(factor) + 1.0
    return freq, 1.0


def _axes(case):
    return [int(d) for d in case["axes"].split(",")]


def _scaling(case):
    if case["scaling"] == "none":
        return None
    s = {"type": case["scaling"], "factor": case["factor"]}
    if case["scaling"] == "yarn":
        s["original_length"] = 4096
    return s


def _cos_sin(positions, axes, theta, scaling="none", factor=1.0):
    """[L, pairs, 2] in 64 bits; positions [axes, L]."""
    parts = []
    for pos, dims in zip(positions, axes):
        freq, m = _inverse_frequencies(dims, theta, scaling, factor, 4096)
        ang = pos.double()[:, None] * freq.to(pos.device)
        parts.append(torch.stack((ang.cos() * m, ang.sin() * m), dim=-1))
    return torch.cat(parts, dim=1)


def _prepare_table(case, seed):
    g = _generator(seed)
    axes, L = _axes(case), case["L"]
    pos = case["start"] + int(torch.randint(0, 1000, (1,), device="cuda", generator=g)) + torch.arange(L, device="cuda")
    if len(axes) == 3:  # a grid of frames, rows and columns; float grids are rescaled ones
        w, h = max(1, math.isqrt(L)), max(1, math.isqrt(math.isqrt(L)))
        pos = torch.stack((pos // (w * h), (pos // w) % h, pos % w))
    else:
        pos = pos[None]
    if case["kind"] == "float":
        pos = (pos.double() * 0.75).float()
    return {"positions": pos if len(axes) == 3 else pos[0], "axes": tuple(axes), "theta": case["theta"],
            "scaling": _scaling(case), "factor": case["factor"], "kind": case["scaling"]}


def _prepare_rotary(case, seed):
    g = _generator(seed)
    B, H, Hk, L, D, dtype = (case[x] for x in ("B", "H", "Hk", "L", "D", "dtype"))

    def heads(n):
        x = _normal(g, B, n, L, D) if case["memory"] == "bhld" else _normal(g, B, L, n, D).transpose(1, 2)
        return x.to(DTYPES[dtype])

    state = {"q": heads(H), "k": heads(Hk), "layout": case["layout"], "skip": case["skip"], "rows": None}
    if case["op"] == "turn":
        state["q"].requires_grad_()
        state["k"].requires_grad_()
        state["dq"], state["dk"] = heads(H), heads(Hk)
    n = L - case["skip"]
    start = int(torch.randint(0, 1000, (1,), device="cuda", generator=g))
    if case["rows"] == "shared":  # another order of the tokens, some of them without a position
        state["rows"] = torch.randperm(L, device="cuda", generator=g, dtype=torch.int32)
        state["rows"][::7] = -1
    elif case["rows"] == "batch":  # each sequence at a place of its own in a longer table
        n = L + 4096
        first = torch.randint(0, 4096, (B, 1), device="cuda", generator=g, dtype=torch.int32)
        state["rows"] = first + torch.arange(L, device="cuda", dtype=torch.int32)
    pos = start + torch.arange(n, device="cuda")
    state["table"] = _cos_sin(pos[None], [case["rot"]], 10000.0).float().contiguous()
    return state


def prepare(case, seed):
    make = {"attention": _prepare_attention, "table": _prepare_table}.get(case["op"], _prepare_rotary)
    return dict(make(case, seed), op=case["op"])


# ---- the operators -----------------------------------------------------------------------------


def _attention(s):
    from sparseattnfunctions_amd.utils.block_sparse_attn_grad import block_sparse_train_fn

    out = block_sparse_train_fn(s["q"], s["k"], s["v"], s["mask"], s["scale"], key_bias=s["bias"],
                                n_text_blocks=s["text_blocks"])
    return (out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"]))


def _plain_attention(s):
    with torch.no_grad():
        q, k, v, do = (s[n].float() for n in ("q", "k", "v", "dout"))
        mask = s["mask"].repeat_interleave(64, dim=2)[:, :, :q.shape[2]].repeat_interleave(64, dim=3)[..., :k.shape[2]]
        p = (q @ k.transpose(2, 3)).mul_(s["scale"])
        if s["bias"] is not None:
            p += s["bias"][:, :, None]
        p.masked_fill_(~mask, float("-inf"))
        del mask
        top = p.amax(dim=3, keepdim=True)
        p.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
        total = p.sum(dim=3, keepdim=True)
        p.div_(torch.where(total == 0, 1.0, total))  # a row without a key: zeros
        out = p @ v
        dv = p.transpose(2, 3) @ do
        ds = (do @ v.transpose(2, 3)).sub_((do * out).sum(dim=3, keepdim=True)).mul_(p)
        del p
        dq, dk = (ds @ k).mul_(s["scale"]), (ds.transpose(2, 3) @ q).mul_(s["scale"])
        return tuple(x.to(s["q"].dtype) for x in (out, dq, dk, dv))


def _plain_turn(x, s, back=False):
    """The rotation of x [B, H, L, D] (its transpose, `back`), in 32 bits."""
    rot = 2 * s["table"].shape[1]
    L, skip, rows = x.shape[2], s["skip"], s["rows"]
    table = s["table"]
    if rows is None:
        table = table[:L - skip]
    else:
        table = table[rows.clamp_min(0).long()]
        still = (rows < 0)[..., None]
        table = torch.stack((table[..., 0].masked_fill(still, 1.0), table[..., 1].masked_fill(still, 0.0)), dim=-1)
    cos, sin = table[..., 0], -table[..., 1] if back else table[..., 1]
    if rows is not None and rows.dim() == 2:
        cos, sin = cos[:, None], sin[:, None]
    y = x.float()
    part = y[:, :, skip:, :rot]
    if s["layout"] == "interleaved":
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(3)
    else:
        a, b = part[..., :rot // 2], part[..., rot // 2:]
        part = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=3)
    part = torch.cat((part, y[:, :, skip:, rot:]), dim=3)
    return torch.cat((y[:, :, :skip], part), dim=2).to(x.dtype)


def run(state):
    s = state
    if s["op"] == "attention":
        return _attention(s) if own else _plain_attention(s)
    if s["op"] == "table":
        if own:
            from sparseattnfunctions_amd.utils.rotary import rotary_table

            return rotary_table(s["positions"], s["axes"], theta=s["theta"], scaling=s["scaling"])
        pos = s["positions"] if s["positions"].dim() == 2 else s["positions"][None]
        return _cos_sin(pos, s["axes"], s["theta"], s["kind"], s["factor"]).float()
    if not own:
        with torch.no_grad():
            out = _plain_turn(s["q"], s), _plain_turn(s["k"], s)
            if s["op"] == "turn":
                out += _plain_turn(s["dq"], s, back=True), _plain_turn(s["dk"], s, back=True)
            return out
    from sparseattnfunctions_amd.utils.rotary import apply_rotary

    q, k = apply_rotary(s["q"], s["k"], s["table"], layout=s["layout"], skip=s["skip"], rows=s["rows"])
    if s["op"] == "turn":
        return (q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"])))
    return q, k


# ---- what each operator cannot do without --------------------------------------------------------


def _pairs(case):
    """Query-key pairs of one head, on average."""
    nq, nk, tb = math.ceil(case["Lq"] / 64), math.ceil(case["Lk"] / 64), math.ceil(case["text"] / 64)
    tq, tk = min(tb, nq) / nq, min(tb, nk) / nk
    kept = tq + (1 - tq) * (tk + (1 - tk) * case["keep"])
    return case["Lq"] * case["Lk"] * max(kept, 1 / nk) * (1 - case["empty"])


def work(case):
    if case["op"] == "attention":
        B, H, Lq, Lk, D, size = case["B"], case["H"], case["Lq"], case["Lk"], case["D"], BYTES[case["dtype"]]
        moved = B * H * D * size * 4 * (Lq + Lk)  # q, out, dout, dq; k, v, dk, dv
        moved += B * H * math.ceil(Lq / 64) * math.ceil(Lk / 64) + (4 * B * Lk if case["bias"] else 0)
        return {"bytes": moved, "flops": int(14 * D * B * H * _pairs(case))}
    if case["op"] == "table":
        axes = _axes(case)
        each = 8 if case["kind"] == "int" else 4
        return {"bytes": case["L"] * (len(axes) * each + 4 * sum(axes)), "flops": case["L"] * sum(axes) * 20}
    values = case["B"] * (case["H"] + case["Hk"]) * case["L"] * case["D"] * (2 if case["op"] == "turn" else 1)
    rows = {"none": case["L"] - case["skip"], "shared": case["L"], "batch": case["B"] * case["L"]}[case["rows"]]
    return {"bytes": 2 * values * BYTES[case["dtype"]] + rows * 4 * case["rot"], "flops": 3 * values * case["rot"] // case["D"]}


# ---- 64-bit values -------------------------------------------------------------------------------


def _exact_attention(s):
    """Head by head and some query rows at a time: probabilities, then the chain rule."""
    q, k, v, do = (s[n].detach().double() for n in ("q", "k", "v", "dout"))
    B, H, Lq, D = q.shape
    Lk, scale = k.shape[2], s["scale"]
    out, dq = torch.zeros_like(q), torch.zeros_like(q)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    blocks = torch.arange(Lk, device="cuda") // 64
    for b in range(B):
        for h in range(H):
            for r0 in range(0, Lq, 4096):
                r = slice(r0, min(r0 + 4096, Lq))
                seen = s["mask"][b, h][torch.arange(r.start, r.stop, device="cuda") // 64][:, blocks]
                x = scale * torch.mm(q[b, h, r], k[b, h].T)
                if s["bias"] is not None:
                    x = x + s["bias"][b, 0].double()
                x = torch.where(seen, x, float("-inf"))
                prob = torch.nan_to_num(torch.softmax(x, dim=1), nan=0.0)
                o = torch.mm(prob, v[b, h])
                dprob = torch.mm(do[b, h, r], v[b, h].T)
                dx = prob * (dprob - (prob * dprob).sum(dim=1, keepdim=True))
                out[b, h, r] = o
                dq[b, h, r] = scale * torch.mm(dx, k[b, h])
                dk[b, h] += scale * torch.mm(dx.T, q[b, h, r])
                dv[b, h] += torch.mm(prob.T, do[b, h, r])
    return out, dq, dk, dv


def _exact_turn(x, s, back):
    """Each pair as a complex number times cos + i sin."""
    x, table, L = x.detach().double(), s["table"].double(), x.shape[2]
    pairs = table.shape[1]
    turn = torch.complex(table[..., 0], table[..., 1])
    if back:
        turn = turn.conj()
    rows = s["rows"]
    if rows is None:
        rows = torch.arange(L, device="cuda") - s["skip"]
    one = torch.ones((), dtype=turn.dtype, device="cuda")
    turn = torch.where((rows >= 0)[..., None], turn[rows.clamp_min(0).long()], one)
    turn = turn[:, None] if rows.dim() == 2 else turn
    i = torch.arange(pairs, device="cuda")
    at, bt = (2 * i, 2 * i + 1) if s["layout"] == "interleaved" else (i, i + pairs)
    z = torch.complex(x[..., at], x[..., bt]) * turn
    y = x.clone()
    y[..., at], y[..., bt] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(s)
    if case["op"] == "table":
        pos = s["positions"].double().reshape(len(s["axes"]), -1)
        columns = []
        for p, dims in zip(pos, s["axes"]):
            for j in range(dims // 2):
                f, m = case["theta"] ** (-2.0 * j / dims), 1.0
                if case["scaling"] == "linear":
                    f /= case["factor"]
                elif case["scaling"] == "ntk":
                    f = (case["theta"] * case["factor"] ** (dims / max(dims - 2, 1))) ** (-2.0 * j / dims)
                elif case["scaling"] == "yarn":
                    g = min(1.0, max(0.0, (4096 * f / (2 * math.pi) - 1) / 31))
                    f, m = g * f + (1 - g) * f / case["factor"], 0.1 * math.log(case["factor"]) + 1
                columns.append(torch.polar(torch.full_like(p, m), p * f))
        return torch.view_as_real(torch.stack(columns, dim=1)).contiguous()
    pairs = [("q", False), ("k", False)] + ([("dq", True), ("dk", True)] if case["op"] == "turn" else [])
    return tuple(_exact_turn(s[n], s, back) for n, back in pairs)
