"""64-bit attention with score rules and its gradients, with a bound of what the kernels may be off, element by element.
Test code only."""
import math

import torch

from grad_reference import unit


def visible(B, H, Lq, Lk, ranges=None, mask=None):
    """bool [B,H,Lq,Lk]."""
    rows = torch.arange(Lq)[:, None]
    seen = torch.ones(B, H, Lq, Lk, dtype=torch.bool)
    if ranges is not None:
        r = ranges.cpu()
        r = (r[None] if r.dim() == 2 else r).expand(B, Lk, 2)
        seen &= ((r[:, None, :, 0] <= rows) & (rows < r[:, None, :, 1]))[:, None]
    if mask is not None:
        m = (mask.cpu() != 0).expand(B, H, *mask.shape[2:])
        seen &= m.repeat_interleave(64, 2)[:, :, :Lq].repeat_interleave(64, 3)[..., :Lk]
    return seen


def scores(q, k, scale, far, cap=None, slopes=None, table=None, buckets=None):
    """(s, derivative of s by scale q.k, error of s, error of the derivative, place): q [B,H,Lq,D], k [B,H,Lk,D] in 64 bits,
    far: distances [Lq, Lk] or [B, 1, Lq, Lk].

    Errors: a dot product of D terms in fp32, e = (D + 8) 2^-24 scale sum |q||k|. tanh comes out of exp2 (1 ulp), an
    addition, a reciprocal (1 ulp) and a subtraction, each at most 2^-23 of numbers up to 2: 6 * 2^-23, and its derivative
    4 (r - r^2) is off by four times r's error, 2.5 * 2^-23, and the roundings: 2^-19, and by 2 e / cap. Each of the other
    terms goes through a product with log2(e) (rounded, as the term is) and an addition to the sum so far: 2^-22 of it."""
    D = q.shape[-1]
    s = scale * (q @ k.transpose(-1, -2))
    e = (D + 8) * 2.0 ** -24 * scale * (q.abs() @ k.abs().transpose(-1, -2))
    c, e_c = torch.ones_like(s), torch.zeros_like(s)
    if cap is not None:
        t = torch.tanh(s / cap)
        c = 1.0 / torch.cosh((s / cap).clamp(-300, 300)) ** 2
        e_c = 2.0 ** -19 + 2 * e / cap
        s = cap * t
        e = e + 6 * 2.0 ** -23 * cap
    size = s.abs()
    place = None
    if slopes is not None:
        add = slopes.double().cpu()[:, None, None] * far.abs().double()
        s, size = s - add, size + add.abs()
    if table is not None:
        R = buckets.numel() // 2
        place = buckets.cpu().long().clamp(0, table.shape[0] - 1)[far.clamp(-R, R) + R]
        add = table.detach().double().cpu()[place]
        add = add.permute(2, 0, 1) if add.dim() == 3 else add.squeeze(1).permute(0, 3, 1, 2)
        s, size = s + add, size + add.abs()
    return s, c, e + 2.0 ** -22 * size, e_c, place


def softmax(s, seen):
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = top.masked_fill(top == -math.inf, 0.0)
    x = torch.exp(s - top)
    total = x.sum(-1, keepdim=True)
    lse = top + total.log().masked_fill(total == 0, 0.0)
    return x / total.masked_fill(total == 0, 1.0), s - top, lse


def finite(x):
    return torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0)


def train(q, k, v, do, scale, cap=None, slopes=None, table=None, buckets=None, ranges=None, mask=None, q_start=0):
    """{name: (value, bound)} of out, dq, dk, dv (and dtable).

    u is the type's rounding (0 inside fp32 calls, whose roundings count in the sums), g = (n + 16) 2^-24 the fp32 sums of
    n terms. P = exp(s - max) is off by the scores' error (its own and, over the row's sum, at most the largest one's), by the
    exponent's rounding 2^-24 |s - max| and by exp2's and the sum's 2^-20; the backward pass has the row's log-sum besides,
    2^-23 of it. The forward pass takes P as two terms of the type: 2 u^2, or half the smallest step of fp16.
      out: sum P |v| (that + 2 g), rounded
      delta = sum do (out + rest): out's error before its rounding, the rest's rounding u^2 |out|, the sum's
      dS = P (dP - delta), its product with the cap's derivative rounded to the type: u
      dq, dk: scale sum |error of dS| |k| and g of the sum, rounded; dv: P rounded; dtable: dS in fp32, rounded once.
    Where P or its product with dP - delta is below fp32's normal range it may be taken as 0: off by 2^-126 (|dP - delta| + 1),
    which a bucket of distant keys, of probability 2^-120, is made of. Second-order terms: 5 %."""
    dtype = q.dtype
    f32 = dtype == torch.float32
    u = 0.0 if f32 else unit(dtype)
    last = unit(dtype)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    B, H, Lq, D = q.shape
    Hk, Lk = k.shape[1:3]
    rep = H // Hk
    table_type = None if table is None else table.dtype
    q, k, v, do = (t.detach().double().cpu() for t in (q, k, v, do))
    k, v = (t.repeat_interleave(rep, 1) for t in (k, v))
    far = torch.arange(Lq)[:, None] + q_start - torch.arange(Lk)
    seen = visible(B, H, Lq, Lk, ranges, mask)
    s, c, e, e_c, place = scores(q, k, scale, far, cap, slopes, table, buckets)
    p, below, lse = softmax(s, seen)
    e = e.masked_fill(~seen, 0.0)
    at = seen.double()
    e = e + 2.0 ** -24 * finite(below).abs()
    rel = e + e.amax(3, keepdim=True) + 2.0 ** -20
    n = max(Lq, Lk, D) * rep
    g = (n + 16) * 2.0 ** -24
    out = p @ v
    e_out = 1.05 * ((p * (rel + 2 * u * u + 2 * g)) @ v.abs() + tiny * (at @ v.abs()))
    dp = do @ v.transpose(2, 3)
    delta = (do * out).sum(3, keepdim=True)
    ds = p * (dp - delta)
    e_delta = (do.abs() * (e_out + (u * u + (D + 8) * 2.0 ** -24) * out.abs() + tiny)).sum(3, keepdim=True)
    rel = rel + 2.0 ** -23 * lse.abs()
    e_ds = p * ((dp - delta).abs() * rel + e_delta + (D + 8) * 2.0 ** -24 * (do.abs() @ v.abs().transpose(2, 3)))
    e_ds = e_ds + 2.0 ** -126 * at * ((dp - delta).abs() + 1)
    dc = ds * c
    e_dc = e_ds * c + ds.abs() * e_c + (u + 2.0 ** -22) * dc.abs() + tiny * at
    dq, e_dq = scale * (dc @ k), scale * ((e_dc + g * dc.abs()) @ k.abs())
    dk, e_dk = scale * (dc.transpose(2, 3) @ q), scale * ((e_dc + g * dc.abs()).transpose(2, 3) @ q.abs())
    dv, e_dv = p.transpose(2, 3) @ do, (p * (rel + u + g) + tiny * at).transpose(2, 3) @ do.abs()
    dk, e_dk, dv, e_dv = (t.view(B, Hk, rep, Lk, D).sum(2) for t in (dk, e_dk, dv, e_dv))
    want = {"out": (out, e_out + last * out.abs() + tiny), "dq": (dq, 1.05 * e_dq + last * dq.abs() + tiny),
            "dk": (dk, 1.05 * e_dk + last * dk.abs() + tiny), "dv": (dv, 1.05 * e_dv + last * dv.abs() + tiny)}
    if table is not None:
        g = (Lq + Lk + 64 * B + 64) * 2.0 ** -24
        value, bound = torch.zeros(table.shape, dtype=torch.float64), torch.zeros(table.shape, dtype=torch.float64)
        where = place.flatten()
        value.index_add_(0, where, ds.sum(0).flatten(1).T)
        bound.index_add_(0, where, (e_ds + (g + 2.0 ** -22) * ds.abs()).sum(0).flatten(1).T)
        last = unit(table_type)
        want["dtable"] = (value, 1.05 * bound + last * value.abs() + (2.0 ** -25 if table_type == torch.float16 else 2.0 ** -126))
    return want


def serve(q, k, v, lengths, scale, cap=None, slopes=None, table=None, buckets=None, window=0, prefix=None):
    """(value, bound) of the new tokens' output: errors as in `train`, with P rounded to the type (its sum, too)."""
    dtype = q.dtype
    u = 0.0 if dtype == torch.float32 else unit(dtype)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    B, H, Ln, D = q.shape
    Hk, L = k.shape[1:3]
    lengths = lengths.cpu().long().clamp(0, L)
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    past = torch.arange(L) >= lengths[:, None, None]  # [B,1,L]
    k, v = (t.masked_fill(past[..., None], 0.0) for t in (k, v))  # (whatever they hold)
    Lp = 0
    if prefix is not None:
        pk, pv = (t.detach().double().cpu().reshape(1, Hk, -1, D).expand(B, -1, -1, -1) for t in prefix)
        Lp = pk.shape[2]
        k, v = torch.cat((pk, k), 2), torch.cat((pv, v), 2)
    k, v = (t.repeat_interleave(H // Hk, 1) for t in (k, v))
    own = lengths[:, None] - Ln + torch.arange(Ln)
    far = (Lp + own)[:, None, :, None] - torch.arange(Lp + L)  # [B,1,Ln,Lp+L]
    seen = (far >= 0) & (own >= 0)[:, None, :, None]
    if window:
        seen = seen & (far < window)
    s, _, e, _, _ = scores(q, k, scale, far, cap, slopes, table, buckets)
    seen = seen.expand_as(s)
    p, below, _ = softmax(s, seen)
    e = e.masked_fill(~seen, 0.0) + 2.0 ** -24 * finite(below).abs()
    rel = e + e.amax(3, keepdim=True) + 2.0 ** -20
    g = (Lp + L + 16) * 2.0 ** -24
    out = p @ v
    bound = (p * (rel + 2 * u + 2 * g) + 2 * tiny * seen) @ v.abs()
    return out, 1.05 * bound + unit(dtype) * out.abs() + tiny


def check(name, got, want):
    value, bound = want
    x = got.detach().double().cpu()
    assert x.shape == value.shape, (name, x.shape, value.shape)
    assert torch.isfinite(x).all(), name
    off = (x - value).abs()
    if off.numel():
        i = (off - bound).argmax()
        assert (off - bound).flatten()[i] <= 0, (name, off.flatten()[i].item(), bound.flatten()[i].item(), value.flatten()[i].item())


def inputs(seed, B, H, Hk, Lq, Lk, D, dtype, dev="cpu"):
    g = torch.Generator().manual_seed(seed)
    shapes = ((B, H, Lq, D), (B, Hk, Lk, D), (B, Hk, Lk, D), (B, H, Lq, D))
    return [torch.randn(s, generator=g).to(dtype).to(dev) for s in shapes]
