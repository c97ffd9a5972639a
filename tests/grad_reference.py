"""64-bit gradients of block-sparse attention, with a bound of what a kernel that rounds P, dS and its
results to a type may be off, element by element. Test code only."""
import math

import torch

from oracle.attention import expand_block_mask


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def reference(q, k, v, do, mask, scale, bias=None, allowed=None):
    """{name: (value, bound)} of out, dq, dk, dv in 64 bits. `allowed` (bool [B,H,Lq,Lk]) replaces the
    block mask's tokens; it may also hold whole numbers: how often a key is listed.

    Bounds, with u the type's rounding (0 inside an fp32 call, where it counts in the sums), and g the
    fp32 sums' (n + 16) 2^-24 for the longest sum n. A score is off by at most e = (D + 8) 2^-24 scale
    sum |q||k|, so P = exp(s - lse) by a factor of 1 + 2 e (its own and the row sum's) and u for a row
    sum of rounded terms: p. Then
      out: sum_j P |v| (p + u + g), rounded;  dv: sum_i P |do| (p + u + g), rounded;
      delta = sum_d do out: D = sum_d |do| (error of out) + g sum |do||out|
      dS = P (dP - delta): P (|dP - delta| p + D + g sum |do||v|) + u |dS|
      dq: scale sum (error of dS + g |dS|) |k|, rounded; dk alike.
    Below fp16's normal range a rounding is off by 2^-25 instead; bf16 and fp32 have fp32's exponents,
    below whose normal range exp2 and a product may give 0: off by less than 2^-126. Second-order terms:
    5 %."""
    dtype = q.dtype
    f32 = dtype == torch.float32
    u = 0.0 if f32 else unit(dtype)
    last = unit(dtype)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    B, H, Lq, D = q.shape
    Lk = k.shape[2]
    q, k, v, do = (t.detach().double() for t in (q, k, v, do))
    if allowed is None:
        allowed = expand_block_mask(mask.expand(B, H, *mask.shape[2:]), Lq, Lk)
    times = allowed.double()
    s = scale * (q @ k.transpose(2, 3))
    if bias is not None:
        s = s + bias.double()[:, :, None]
    s = s.masked_fill(times == 0, -math.inf)
    top = s.amax(3, keepdim=True)
    x = times * torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
    total = x.sum(3, keepdim=True)
    p = x / total.masked_fill(total == 0, 1.0)
    out, dp = p @ v, do @ v.transpose(2, 3)
    delta = (do * out).sum(3, keepdim=True)
    ds = p * (dp - delta)
    dq, dk, dv = scale * (ds @ k), scale * (ds.transpose(2, 3) @ q), p.transpose(2, 3) @ do

    n = max(Lq, Lk, D)
    g = (n + 16) * 2.0 ** -24
    e = (D + 8) * 2.0 ** -24 * scale * (q.abs() @ k.abs().transpose(2, 3))
    if bias is not None:
        e = e + 2.0 ** -22 * bias.double()[:, :, None].abs().masked_fill(bias[:, :, None].isinf(), 0.0)
    e = e.masked_fill(p == 0, 0.0)
    rel = e + e.amax(3, keepdim=True) + u + 2.0 ** -20
    at = (p > 0).double()
    e_out = (p * (rel + u + g)) @ v.abs() + tiny * (at @ v.abs())
    e_dv = (p * (rel + u + g)).transpose(2, 3) @ do.abs() + tiny * (at.transpose(2, 3) @ do.abs())
    e_out = 1.05 * e_out + last * out.abs() + tiny
    d = (do.abs() * (e_out + (D + 8) * 2.0 ** -24 * out.abs())).sum(3, keepdim=True)
    e_ds = p * ((dp - delta).abs() * rel + d + (D + 8) * 2.0 ** -24 * (do.abs() @ v.abs().transpose(2, 3)))
    e_ds = e_ds + (u + g) * ds.abs() + tiny * at
    e_dq = scale * (e_ds @ k.abs())
    e_dk = scale * (e_ds.transpose(2, 3) @ q.abs())
    return {"out": (out, e_out), "dq": (dq, 1.05 * e_dq + last * dq.abs() + tiny),
            "dk": (dk, 1.05 * e_dk + last * dk.abs() + tiny), "dv": (dv, 1.05 * e_dv + last * dv.abs() + tiny)}


def check(got, want, names=("out", "dq", "dk", "dv"), norm=None):
    """Every element within its bound; with `norm`, each tensor's 2-norm error within norm times its own."""
    for name, x in zip(names, got):
        value, bound = want[name]
        x = x.detach().double().cpu()
        assert torch.isfinite(x).all(), name
        off = (x - value).abs()
        worst = (off - bound).max().item()
        assert worst <= 0, (name, worst, off.max().item(), bound.flatten()[(off - bound).argmax()].item())
        if norm is not None:
            assert off.norm() <= norm * value.norm(), (name, (off.norm() / value.norm()).item(), norm)
