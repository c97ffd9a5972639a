"""Gradients where a row's keys all have a large finite bias, as a block row that lists nothing but padding has: the
bias is added in fp32 like any additive mask's, and the backward pass has to take the probabilities that the forward
pass took, whatever the bias's size."""
import math

import numpy as np
import pytest
import torch

from conftest import case
from grad_reference import check, reference, unit
from oracle.attention import expand_block_mask
from sparseattnfunctions_amd._kv import kv_list_from_mask
from sparseattnfunctions_amd.utils.block_sparse_attn_grad import (block_sparse_attention_backward,
                                                                  block_sparse_attention_lse,
                                                                  block_sparse_attention_train, block_sparse_train_fn)

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
LOG2E = np.float32(math.log2(math.e))


def _reference(q, k, v, do, mask, scale, bias):
    """{name: (value, bound)} of out, dq, dk, dv in 64 bits from the scores that fp32 holds: bias * log2(e) rounded, then
    its sum with the scaled product rounded. q and k are small whole numbers, whose products are exact.

    Bounds as in grad_reference.reference, but for the scores' error: the difference of a score and the row's offset
    is one fp32 subtraction, off by 2^-24 of at most 2^7 (below that P is 0), the row sum's logarithm, at most 2^7 as well,
    another two: 3 * 2^-17. Rows whose offset is at most 64 have it and that logarithm in one number below 2^7, from which
    the sums of D / 16 products start: off by half a step, 2^-18, for each of at most 8 + 3 roundings. e = 2^-14."""
    dtype = q.dtype
    u = unit(dtype)
    tiny = 2.0 ** -25 if dtype == FP16 else 2.0 ** -126
    Lq, Lk, D = q.shape[2], k.shape[2], q.shape[3]
    q, k, v, do = (t.double() for t in (q, k, v, do))
    allowed = expand_block_mask(mask, Lq, Lk)
    s2 = float(np.float32(np.float32(scale) * LOG2E))
    b2 = torch.from_numpy(bias.numpy() * LOG2E)
    assert b2.dtype == torch.float32
    x = ((q @ k.transpose(2, 3)) * s2 + b2.double()[:, :, None]).float().double().masked_fill(~allowed, -math.inf)
    top = x.amax(3, keepdim=True)
    p = torch.exp2(x - top.masked_fill(top == -math.inf, 0.0))
    total = p.sum(3, keepdim=True)
    p = p / total.masked_fill(total == 0, 1.0)
    out, dp = p @ v, do @ v.transpose(2, 3)
    delta = (do * out).sum(3, keepdim=True)
    ds = p * (dp - delta)
    dq, dk, dv = scale * (ds @ k), scale * (ds.transpose(2, 3) @ q), p.transpose(2, 3) @ do

    g = (max(Lq, Lk, D) + 16) * 2.0 ** -24
    rel = 2.0 ** -14 + u + 2.0 ** -20
    at = (p > 0).double()
    e_out = 1.05 * ((p * (rel + u + g)) @ v.abs() + tiny * (at @ v.abs())) + u * out.abs() + tiny
    e_dv = (p * (rel + u + g)).transpose(2, 3) @ do.abs() + tiny * (at.transpose(2, 3) @ do.abs())
    sums = (D + 8) * 2.0 ** -24
    d = (do.abs() * (e_out + sums * out.abs())).sum(3, keepdim=True)
    e_ds = p * ((dp - delta).abs() * rel + d + sums * (do.abs() @ v.abs().transpose(2, 3))) + (u + g) * ds.abs() + tiny * at
    e_dq, e_dk = scale * (e_ds @ k.abs()), scale * (e_ds.transpose(2, 3) @ q.abs())
    return {"out": (out, e_out), "dq": (dq, 1.05 * e_dq + u * dq.abs() + tiny),
            "dk": (dk, 1.05 * e_dk + u * dk.abs() + tiny), "dv": (dv, 1.05 * e_dv + u * dv.abs() + tiny)}


def _inputs(dtype, B, H, Lq, Lk, D, value):
    """Keys of the last third at `value`, of the second batch all of them; the second row block lists only such keys."""
    g = torch.Generator().manual_seed(3)
    q, k = (torch.randint(-2, 3, (B, H, L, D), generator=g).to(dtype) for L in (Lq, Lk))
    v, do = (torch.randn(B, H, L, D, generator=g).to(dtype) for L in (Lk, Lq))
    nq, nk = math.ceil(Lq / 64), math.ceil(Lk / 64)
    mask = torch.rand(B, H, nq, nk, generator=g) < 0.6
    mask[..., 0] = True
    first = 64 * (2 * nk // 3)
    mask[:, :, 1] = torch.arange(nk) >= first // 64
    bias = torch.randint(1, 5, (B, 1, Lk), generator=g).float().log()
    bias[..., first:] = value
    bias[1:] = value
    return (q, k, v, do), mask, bias


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shape,value,scale", [
    ((2, 3, 200, 330), -40.0, 0.125), ((2, 3, 200, 330), -300.0, 0.125), ((2, 3, 200, 330), -1e4, 0.125), ((2, 3, 200, 330), -1e6, 0.125),
    ((2, 3, 200, 330), -1e9, 0.125), ((2, 3, 200, 330), -1e30, 0.125),
    ((2, 3, 200, 330), -1e9, 8.0),  # scores that differ by more than an fp32 step at 1e9
    ((2, 70, 400, 330), -1e9, 0.125),  # one pair of waves per block
    ((2, 1, 150, 4400), -1e9, 0.125),  # few query blocks over long lists: split over workgroups
    ((2, 1, 4400, 150), -1e9, 0.125)])
def test_rows_of_biased_keys(dev, dtype, D, shape, value, scale):
    case(f"rows of keys biased by {value} {shape} {dtype} D={D}")
    inputs, mask, bias = _inputs(dtype, *shape, D, value)
    leaves = [t.to(dev).requires_grad_() for t in inputs[:3]]
    out = block_sparse_train_fn(*leaves, mask.to(dev), scale, key_bias=bias.to(dev))
    got = (out, *torch.autograd.grad(out, leaves, inputs[3].to(dev)))
    check(got, _reference(*inputs, mask, scale, bias))


def test_probabilities_sum_to_one(dev):
    # do = 1: the columns of dv hold each key's probabilities, which sum to the number of rows: off by a rounding of
    # each probability and of each sum, 2^-8 each.
    case("sums of the recomputed probabilities")
    for value in (-1e4, -1e7, -1e9, -1e30):
        (q, k, v, _), mask, bias = _inputs(BF16, 2, 2, 200, 330, 64, value)
        q = (q.float() * 1.37).bfloat16()
        x = [t.to(dev) for t in (q, k, v)]
        kv = kv_list_from_mask(mask.to(dev), 2, 2, 4, 6)
        out, lse = block_sparse_attention_lse(*x, kv, 0.125, key_bias=bias.to(dev))
        dv = block_sparse_attention_backward(torch.ones_like(out), *x, out, lse, kv, 0.125, key_bias=bias.to(dev))[2]
        off = dv.double().sum(2) / 200 - 1
        assert off.abs().max() <= 2 * 2.0 ** -8, (value, off.abs().max().item())


def test_bias_of_each_head_and_of_all(dev):
    # A bias with values of its own for every head, in a tensor with odd strides, and one for all heads.
    case("bias per head")
    g = torch.Generator().manual_seed(8)
    B, H, Lq, Lk = 2, 3, 150, 200
    q, k, v, do = (torch.randn(B, H, L, 64, generator=g).bfloat16() for L in (Lq, Lk, Lk, Lq))
    mask = torch.rand(B, H, 3, 4, generator=g) < 0.7
    mask[..., 0] = True
    wide = torch.randn(H, B, Lk + 3, generator=g)
    for bias in (wide[..., 1:Lk + 1].transpose(0, 1), wide[0, 0, :Lk]):
        leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
        b = wide.to(dev)[..., 1:Lk + 1].transpose(0, 1) if bias.dim() == 3 else bias.to(dev)
        out = block_sparse_train_fn(*leaves, mask.to(dev), 0.125, key_bias=b)
        got = (out, *torch.autograd.grad(out, leaves, do.to(dev)))
        check(got, reference(q, k, v, do, mask, 0.125, bias=bias.expand(B, H, Lk)), norm=1.5 * unit(BF16))


@pytest.mark.parametrize("lists", ["mask", "lists"])
def test_saved_tensors_of_a_biased_call_may_move(dev, lists):
    case(f"saved tensor hooks with a bias, {lists}")
    inputs, mask, bias = _inputs(BF16, 2, 3, 200, 330, 64, -1e9)
    x, mask, bias = [t.to(dev) for t in inputs], mask.to(dev), bias.to(dev)
    kv = kv_list_from_mask(mask, 2, 3, 4, 6)

    def grads():
        # (q in rows of 72 values, which come back from the host in rows of 64)
        wide = torch.zeros(2, 3, 200, 72, dtype=BF16, device=dev)
        wide[..., :64] = x[0]
        leaves = [wide[..., :64].requires_grad_(), *(t.detach().requires_grad_() for t in x[1:3])]
        if lists == "mask":
            out = block_sparse_train_fn(*leaves, mask, 0.125, key_bias=bias)
        else:
            out = block_sparse_attention_train(*leaves, kv, 0.125, key_bias=bias)
        return out, lambda: torch.autograd.grad(out, leaves, x[3])

    want = grads()[1]()
    with torch.autograd.graph.save_on_cpu():
        out, back = grads()
        got = back()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    check((out, *got), _reference(*inputs, mask.cpu(), 0.125, bias.cpu()))
