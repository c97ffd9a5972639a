"""Gradients of block-sparse attention against 64-bit ones, within bounds that follow from the roundings
(tests/grad_reference.py)."""
import math

import pytest
import torch
import torch.utils.checkpoint

from conftest import case
from grad_reference import check, reference, unit
from sparseattnfunctions_amd._kv import KVList, kv_list_from_mask
from sparseattnfunctions_amd.block_mask_attn import dense_kv_list
from sparseattnfunctions_amd.utils.block_sparse_attn_grad import (
    block_sparse_attention_backward, block_sparse_attention_lse, block_sparse_attention_train, block_sparse_train_fn,
    transpose_kv_list)
from sparseattnfunctions_amd.utils.block_sparse_attn_kernel import block_sparse_attention, block_sparse_triton_fn

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _rand(g, *shape, dtype=FP32):
    return torch.randn(*shape, generator=g).to(dtype)


def _inputs(seed, dtype, B, H, Lq, Lk, D):
    g = torch.Generator().manual_seed(seed)
    return [_rand(g, B, H, L, D, dtype=dtype) for L in (Lq, Lk, Lk, Lq)], g


def _mask(g, B, H, Lq, Lk, density, empty=0.0):
    nq, nk = math.ceil(Lq / 64), math.ceil(Lk / 64)
    mask = torch.rand(B, H, nq, nk, generator=g) < density
    mask |= torch.eye(nq, nk, dtype=torch.bool)
    return mask & (torch.rand(B, H, nq, 1, generator=g) >= empty)


def _grads(fn, q, k, v, do):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = fn(*leaves)
    return (out, *torch.autograd.grad(out, leaves, do))


SHAPES = [
    # B, H, Lq, Lk, density, empty rows
    (1, 1, 1, 1, 1.0, 0.0),
    (1, 2, 1, 200, 1.0, 0.0),
    (1, 2, 64, 64, 1.0, 0.0),
    (2, 3, 65, 33, 1.0, 0.0),
    (2, 3, 130, 257, 0.5, 0.0),
    (1, 2, 300, 1, 1.0, 0.3),
    (2, 2, 400, 210, 0.4, 0.4),
    (1, 2, 700, 700, 0.3, 0.2),
    (2, 30, 640, 600, 0.3, 0.1),  # one pair of waves per block at head dim 128
    (2, 45, 580, 640, 0.4, 0.0),  # and at 64
    (1, 3, 70, 4500, 0.4, 0.0),  # few query blocks over long lists: split over workgroups
    (1, 3, 4500, 70, 0.6, 0.1),  # few key blocks
    (1, 2, 2300, 2200, 1.0, 0.0),
]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gradients(dev, shape, dtype, D):
    B, H, Lq, Lk, density, empty = shape
    case(f"gradients {shape} {dtype} D={D}")
    (q, k, v, do), g = _inputs(1, dtype, B, H, Lq, Lk, D)
    mask = _mask(g, B, H, Lq, Lk, density, empty)
    scale = 1 / math.sqrt(D)
    got = _grads(lambda *x: block_sparse_train_fn(*x, mask.to(dev), scale), *(t.to(dev) for t in (q, k, v, do)))
    assert all(x.dtype == dtype for x in got)
    # Roundings are independent: one is off by u / sqrt(3) at most in the mean square, and a result has
    # seen four (row sum, P or dS, out in delta, itself): 1.2 u. (One key: dq and dk are 0.) fp32: sums
    # of n terms, each a product of rounded ones, about sqrt(n) 2^-24, n up to 700.
    norm = None if Lk == 1 else 1.5 * unit(dtype) if dtype != FP32 else 32 * 2.0 ** -24
    check(got, reference(q, k, v, do, mask, scale), norm=norm)
    dead = ~mask.any(2)  # key blocks in no list
    for x in got[2:]:
        blocks = torch.nn.functional.pad(x.cpu().float(), (0, 0, 0, -Lk % 64)).unflatten(2, (-1, 64))
        assert not blocks[dead].any()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
def test_forward_keeps_the_bits_of_block_sparse_triton_fn(dev, dtype):
    # (fp32 with fewer than eight query blocks: split operands here, not there)
    for D, L, H in ((64, 640, 30), (128, 333 if dtype != FP32 else 530, 2), (64, 9000, 1), (64, 4300, 1)):
        case(f"forward bits D={D} L={L} {dtype}")
        (q, k, v, _), g = _inputs(2, dtype, 1, H, L, L, D)
        mask = _mask(g, 1, H, L, L, 1.0 if L > 4000 else 0.3).to(dev)
        q, k, v = q.to(dev), k.to(dev), v.to(dev)
        want = block_sparse_triton_fn(q, k, v, mask, 0.1)
        assert torch.equal(block_sparse_train_fn(q, k, v, mask, 0.1), want)


# The blocks behind the last full round of workgroups are split: by two in short lists, by three in long ones,
# all of them where there is less than a round.
@pytest.mark.parametrize("H,L,D,text", [(9, 1100, 64, 0), (17, 2100, 64, 2), (9, 2100, 128, 0)])
def test_fp32_remainders(dev, H, L, D, text):
    case(f"fp32 remainders H={H} L={L} D={D}")
    Lk = L - 20
    (q, k, v, do), g = _inputs(17, FP32, 1, H, L, Lk, D)
    mask = _mask(g, 1, H, L, Lk, 0.3, 0.1)
    mask[:, :, :text] = True
    mask[..., :text] = True
    fn = lambda *x: block_sparse_train_fn(*x, mask.to(dev), 0.125, n_text_blocks=text)
    got = _grads(fn, *(t.to(dev) for t in (q, k, v, do)))
    # (as in test_gradients, sums of up to 2 100 terms)
    check(got, reference(q, k, v, do, mask, 0.125), norm=64 * 2.0 ** -24)
    assert all(torch.equal(a, b) for a, b in zip(got, _grads(fn, *(t.to(dev) for t in (q, k, v, do)))))


# Launches of more than a round, whose last items run longest list first: the bits of launches of some heads
# each, which take the order of the items.
@pytest.mark.parametrize("dtype,H,group,L,D", [(BF16, 12, 6, 4170, 64), (FP16, 33, 11, 2090, 128)])
def test_last_round_by_length(dev, dtype, H, group, L, D):
    case(f"last round H={H} L={L} D={D}")
    (q, k, v, do), g = _inputs(19, dtype, 1, H, L, L, D)
    mask = _mask(g, 1, H, L, L, 0.1, 0.2)
    mask &= torch.rand(1, H, *mask.shape[2:], generator=g) < torch.rand(1, H, mask.shape[2], 1, generator=g)
    q, k, v, do, mask = (t.to(dev) for t in (q, k, v, do, mask))
    got = _grads(lambda *x: block_sparse_train_fn(*x, mask, 0.125), q, k, v, do)
    for h in range(0, H, group):
        some = slice(h, h + group)
        want = _grads(lambda *x: block_sparse_train_fn(*x, mask[:, some], 0.125), *(t[:, some] for t in (q, k, v, do)))
        assert all(torch.equal(x[:, some], y) for x, y in zip(got[1:], want[1:]))
    check([x[:, :1] for x in got], reference(*(t[:, :1].cpu() for t in (q, k, v, do, mask)), 0.125),
          norm=1.5 * unit(dtype))


@pytest.mark.parametrize("D", [64, 128])
def test_fp32_small_and_large_gradients(dev, D):
    # Powers of two come out of every product: 2^-60 and 2^60 times the gradient give as much of the results, but for
    # terms 2^-60 of the others.
    case(f"fp32 gradients far from one D={D}")
    (q, k, v, do), g = _inputs(20, FP32, 1, 2, 200, 150, D)
    mask = _mask(g, 1, 2, 200, 150, 0.6).to(dev)
    q, k, v, do = (t.to(dev) for t in (q, k, v, do))
    want = _grads(lambda *x: block_sparse_train_fn(*x, mask, 0.125), q, k, v, do)[1:]
    for f in (2.0 ** -60, 2.0 ** 60):
        got = _grads(lambda *x: block_sparse_train_fn(*x, mask, 0.125), q, k, v, do * f)[1:]
        for x, y in zip(got, want):
            assert torch.allclose(x / f, y, rtol=2.0 ** -22, atol=2.0 ** -22 * y.abs().max().item())


# Text blocks whose long lists are split: of the query pass, of the key pass (and more text blocks than a head has
# blocks), of both, unlike many of them on each XCD.
@pytest.mark.parametrize("H,Lq,Lk,D,text,bias", [(12, 330, 2700, 64, 4, True), (24, 2700, 200, 128, 9, False),
                                                 (3, 6200, 6150, 64, 1, False)])
def test_split_text_blocks(dev, H, Lq, Lk, D, text, bias):
    case(f"split text blocks H={H} {Lq} x {Lk} D={D}")
    (q, k, v, do), g = _inputs(18, BF16, 2 if bias else 1, H, Lq, Lk, D)
    B = q.shape[0]
    mask = _mask(g, B, H, Lq, Lk, 0.2, 0.1)
    mask[:, :, :text] = True
    mask[..., :text] = True
    b = _rand(g, B, 1, Lk) if bias else None
    fn = lambda *x: block_sparse_train_fn(*x, mask.to(dev), 0.125, n_text_blocks=text,
                                          key_bias=b.to(dev) if bias else None)
    got = _grads(fn, *(t.to(dev) for t in (q, k, v, do)))
    check(got, reference(q, k, v, do, mask, 0.125, bias=b), norm=1.5 * unit(BF16))
    assert all(torch.equal(x, y) for x, y in zip(got, _grads(fn, *(t.to(dev) for t in (q, k, v, do)))))


@pytest.mark.parametrize("D", [64, 128])
def test_text_blocks(dev, D):
    # The hint of long first rows changes the schedule (shared rows in the forward pass) and no value.
    case(f"text blocks D={D}")
    (q, k, v, do), g = _inputs(16, BF16, 2, 75, 320, 300, D)
    mask = _mask(g, 2, 75, 320, 300, 0.3)
    mask[:, :, :2] = True
    mask[..., :2] = True
    got = _grads(lambda *x: block_sparse_train_fn(*x, mask.to(dev), 0.125, n_text_blocks=2), *(t.to(dev) for t in (q, k, v, do)))
    check(got, reference(q, k, v, do, mask, 0.125), norm=1.5 * unit(BF16))


def test_saved_tensor_hooks_and_two_backward_passes(dev):
    case("saved tensor hooks")
    (q, k, v, do), g = _inputs(17, BF16, 1, 2, 200, 200, 64)
    mask = _mask(g, 1, 2, 200, 200, 0.6).to(dev)
    x = [t.to(dev) for t in (q, k, v, do)]
    want = _grads(lambda *y: block_sparse_train_fn(*y, mask, 0.125), *x)
    with torch.autograd.graph.save_on_cpu():
        got = _grads(lambda *y: block_sparse_train_fn(*y, mask, 0.125), *x)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    leaves = [t.requires_grad_() for t in x[:3]]
    out = block_sparse_train_fn(*leaves, mask, 0.125)
    first = torch.autograd.grad(out, leaves, x[3], retain_graph=True)
    again = torch.autograd.grad(out, leaves, x[3])
    assert all(torch.equal(a, b) for a, b in zip(first, again)) and torch.equal(first[0], want[1])
    ck = torch.utils.checkpoint.checkpoint(lambda *y: block_sparse_train_fn(*y, mask, 0.125), *leaves, use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(ck, leaves, x[3]), first))


def test_lse(dev):
    case("lse")
    (q, k, v, _), g = _inputs(3, FP32, 1, 2, 130, 300, 64)
    mask = _mask(g, 1, 2, 130, 300, 0.5)
    mask[0, 1, 2] = False
    for dtype, tol in ((FP32, 1e-5), (BF16, 2.0 ** -7), (FP16, 2.0 ** -10)):
        x = [t.to(dtype).to(dev) for t in (q, k, v)]
        kv = kv_list_from_mask(mask.to(dev), 1, 2, 3, 5)
        _, lse = block_sparse_attention_lse(*x, kv, 0.125)
        s = 0.125 * x[0].cpu().double() @ x[1].cpu().double().transpose(2, 3)
        allowed = mask.repeat_interleave(64, 2).repeat_interleave(64, 3)[..., :130, :300]
        want = torch.logsumexp(s.masked_fill(~allowed, -math.inf), 3) / math.log(2)
        lse = lse.cpu().double()
        assert lse.shape == (1, 2, 192) and (lse[..., 130:] == math.inf).all()
        empty = want == -math.inf
        assert empty.any() and (lse[..., :130][empty] == math.inf).all()
        # the row sum is of rounded terms: off by a factor within 1 + eps / 2 (twice, to be safe in logs)
        assert (lse[..., :130] - want)[~empty].abs().max() <= tol / math.log(2)


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Lq", [(2, 150), (40, 500)])
def test_key_bias(dev, dtype, D, H, Lq):
    # Biased keys, masked ones (-inf) and the type's lowest value; the first batch's block 1 is masked
    # whole, so that rows listing only it have no key at all.
    case(f"key bias {dtype} D={D} H={H}")
    B, Lk = 2, 230
    (q, k, v, do), g = _inputs(4, dtype, B, H, Lq, Lk, D)
    mask = _mask(g, B, H, Lq, Lk, 0.5)
    mask[0, 0, 1] = torch.tensor([False, True, False, False])
    bias = _rand(g, B, 1, Lk)
    bias[0, 0, 64:128] = -math.inf
    bias[1, 0, 5:40] = -math.inf
    bias[1, 0, 100:110] = torch.finfo(FP32).min
    want = reference(q, k, v, do, mask, 0.125, bias=bias)
    assert not want["dq"][0][0, 0, 64:128].any()
    b = bias.to(dev)
    got = _grads(lambda *x: block_sparse_train_fn(*x, mask.to(dev), 0.125, key_bias=b), *(t.to(dev) for t in (q, k, v, do)))
    check(got, want)
    assert not got[1][0, 0, 64:128].any() and not got[2][1, :, 5:40].any() and not got[3][1, :, 5:40].any()
    assert not got[2][1, :, 100:110].any()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
def test_scores_far_from_zero(dev, dtype):
    # Scores in the hundreds and rows whose every score is far below zero: exp2 of no raw score is in range.
    case(f"large scores {dtype}")
    (q, k, v, do), g = _inputs(5, dtype, 1, 2, 200, 180, 64)
    q, k = (12 * q.float()).to(dtype), (12 * k.float()).to(dtype)
    k = k.abs()
    q[:, :, 70:90] = -q[:, :, 70:90].abs()
    q[:, :, 90:100] = q[:, :, 90:100].abs()
    mask = _mask(g, 1, 2, 200, 180, 0.6)
    got = _grads(lambda *x: block_sparse_train_fn(*x, mask.to(dev), 0.125), *(t.to(dev) for t in (q, k, v, do)))
    check(got, reference(q, k, v, do, mask, 0.125))


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
def test_unlisted_and_unread_values_do_not_matter(dev, dtype):
    # NaN and infinities in key blocks that no row lists, and behind the tensors' last rows.
    case(f"unlisted NaN {dtype}")
    (q, k, v, do), g = _inputs(6, dtype, 1, 2, 150, 300, 64)
    mask = _mask(g, 1, 2, 150, 300, 0.5)
    mask[..., 2] = False
    want = reference(q, k, v, do, mask, 0.125)

    def behind(t, fill):
        wide = torch.full((t.shape[0], t.shape[1], t.shape[2] + 70, 64), fill, dtype=dtype, device=dev)
        wide[:, :, :t.shape[2]] = t.to(dev)
        return wide[:, :, :t.shape[2]]

    k, v = k.clone(), v.clone()
    k[:, :, 128:192], v[:, :, 128:192] = math.nan, math.inf
    got = _grads(lambda *x: block_sparse_train_fn(*x, mask.to(dev), 0.125), behind(q, math.nan), behind(k, math.nan),
                 behind(v, math.inf), behind(do, math.nan))
    check(got, want)
    assert not got[2][:, :, 128:192].any() and not got[3][:, :, 128:192].any()


def test_strides_shared_heads_and_partial_needs(dev):
    case("strides")
    B, H, L, D = 2, 3, 200, 64
    (q, k, v, do), g = _inputs(7, BF16, B, H, L, L, D)
    k, v = k[:, :1], v[:1]
    mask = _mask(g, B, 1, L, L, 0.6)
    want = reference(q, k.expand(B, H, L, D), v.expand(B, H, L, D), do, mask, 0.125)
    wide = torch.zeros(B, L, H, D + 8, dtype=BF16, device=dev)  # [B, L, H, D] rows of 72 values
    wide[..., :D] = q.transpose(1, 2).to(dev)
    ql = wide[..., :D].transpose(1, 2).detach().requires_grad_()
    odd = torch.zeros(B * L * D + 1, dtype=BF16, device=dev)  # base not 16-byte aligned
    odd[1:] = k.to(dev).flatten()
    kl = odd[1:].view(B, 1, L, D).detach().requires_grad_()
    vl = v.to(dev).requires_grad_()
    dos = do.to(dev).transpose(2, 3).contiguous().transpose(2, 3)  # last axis not contiguous
    out = block_sparse_train_fn(ql, kl.expand(B, H, L, D), vl.expand(B, H, L, D), mask.to(dev).expand(B, H, -1, -1), 0.125)
    dq, dk, dv = torch.autograd.grad(out, (ql, kl, vl), dos, retain_graph=True)
    check((out, dq), want)
    # shared heads: torch adds the heads' rounded gradients and rounds the sum once (bf16 2^-8)
    for got, name, dim in ((dk, "dk", 1), (dv, "dv", 0)):
        value, bound = (t.sum(dim, keepdim=True) for t in want[name])
        off = (got.double().cpu() - value).abs()
        assert (off <= bound + 2.0 ** -8 * (value.abs() + bound)).all(), name
    # only some gradients are asked for: the same bits
    kv = kv_list_from_mask(mask.to(dev).expand(B, H, -1, -1), B, H, 4, 4)
    full = [t.expand(B, H, L, D).to(dev) for t in (q, k, v)]
    o, lse = block_sparse_attention_lse(*full, kv, 0.125)
    every = block_sparse_attention_backward(do.to(dev), *full, o, lse, kv, 0.125)
    for needs in ((True, False, False), (False, True, False), (False, False, True), (False, True, True)):
        some = block_sparse_attention_backward(do.to(dev), *full, o, lse, kv, 0.125, needs=needs)
        for want_it, x, y in zip(needs, some, every):
            assert (x is None) if not want_it else torch.equal(x, y)
    v2 = full[2].clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(block_sparse_attention_train(*full[:2], v2, kv, 0.125), v2, do.to(dev))[0], every[2])
    # an expanded gradient (out.sum())
    s = block_sparse_attention_train(*full[:2], v2, kv, 0.125).float().sum()
    ones = block_sparse_attention_backward(torch.ones_like(o), *full, o, lse, kv, 0.125)[2]
    assert torch.equal(torch.autograd.grad(s, v2)[0], ones)


def test_lists_with_foreign_and_repeated_entries(dev):
    # As in the forward pass, entries outside the grid are skipped and a block listed twice counts twice.
    case("lists with foreign and repeated entries")
    (q, k, v, do), _ = _inputs(8, BF16, 1, 1, 128, 190, 64)
    idx = torch.tensor([[0, 2, 2, 99, -3], [1, 0, 7, 1, 0]], dtype=torch.int32)
    cnt = torch.tensor([5, 3], dtype=torch.int32)
    kv = KVList(idx.to(dev), cnt.to(dev), 1, 1, 2, 3)
    beg, qi = transpose_kv_list(kv)
    assert beg.tolist() == [[0, 2, 3, 5]] and qi[0, :5].tolist() == [0, 1, 1, 0, 0]
    times = torch.tensor([[1.0, 0.0, 2.0], [1.0, 1.0, 0.0]]).repeat_interleave(64, 0).repeat_interleave(64, 1)[None, None, :, :190]
    x = [t.to(dev) for t in (q, k, v, do)]
    check(_grads(lambda *y: block_sparse_attention_train(*y, kv, 0.125), *x), reference(q, k, v, do, None, 0.125, allowed=times))


@pytest.mark.parametrize("nqb,nkb,density", [(1, 1, 1.0), (3, 200, 0.4), (200, 3, 0.4), (130, 129, 0.1), (300, 300, 1.0),
                                             (257, 65, 0.0)])
def test_transposed_lists(dev, nqb, nkb, density):
    case(f"transposed lists {nqb} x {nkb}")
    g = torch.Generator().manual_seed(9)
    mask = torch.rand(2, 3, nqb, nkb, generator=g) < density
    kv = kv_list_from_mask(mask.to(dev), 2, 3, nqb, nkb)
    beg, idx = (t.cpu() for t in transpose_kv_list(kv))
    flat = mask.reshape(6, nqb, nkb)
    for bh in range(6):
        assert beg[bh, 0] == 0 and beg[bh, -1] == flat[bh].sum()
        for j in range(nkb):
            assert idx[bh, beg[bh, j]:beg[bh, j + 1]].tolist() == flat[bh, :, j].nonzero()[:, 0].tolist()


@pytest.mark.parametrize("block_m,block_n", [(128, 64), (64, 256), (256, 128)])
def test_larger_blocks(dev, block_m, block_n):
    case(f"blocks {block_m} x {block_n}")
    (q, k, v, do), g = _inputs(10, BF16, 1, 2, 500, 430, 64)
    mask = torch.rand(1, 2, math.ceil(500 / block_m), math.ceil(430 / block_n), generator=g) < 0.6
    allowed = mask.repeat_interleave(block_m, 2).repeat_interleave(block_n, 3)[..., :500, :430]
    got = _grads(lambda *x: block_sparse_train_fn(*x, mask.to(dev), 0.125, BLOCK_M=block_m, BLOCK_N=block_n),
                 *(t.to(dev) for t in (q, k, v, do)))
    check(got, reference(q, k, v, do, None, 0.125, allowed=allowed))


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
def test_offsets_past_32_bits(dev, dtype):
    # Batches 2^31 values apart.
    case(f"far batches {dtype}")
    (q, k, v, do), g = _inputs(21, dtype, 2, 2, 100, 100, 64)
    mask = _mask(g, 2, 2, 100, 100, 0.7).to(dev)
    tensors = [t.to(dev) for t in (q, k, v, do)]
    fn = lambda *x: block_sparse_train_fn(*x, mask, 0.125)
    want = _grads(fn, *tensors)
    n = 2 * 100 * 64
    base = torch.empty(2 ** 31 + 4 * n, dtype=dtype, device=dev)
    far = [base.as_strided((2, 2, 100, 64), (2 ** 31, 6400, 64, 1), i * n).copy_(t) for i, t in enumerate(tensors)]
    assert all(torch.equal(x, y) for x, y in zip(_grads(fn, *far), want))


def test_differences(dev):
    # <grad, step> against the loss on both sides of it: fp32, steps of 2^-9, whose third-order term and
    # rounding (2^-24 of the loss's terms over the step) are below 1e-3 of the change.
    case("differences")
    (q, k, v, do), g = _inputs(11, FP32, 1, 2, 140, 200, 64)
    mask = _mask(g, 1, 2, 140, 200, 0.5).to(dev)
    x = [t.to(dev) for t in (q, k, v)]
    do = do.to(dev)
    grads = _grads(lambda *y: block_sparse_train_fn(*y, mask, 0.125), *x, do)[1:]
    for i in range(3):
        step = torch.randn(x[i].shape, generator=g).to(dev)
        h = 2.0 ** -9
        side = []
        for sign in (1, -1):
            y = list(x)
            y[i] = x[i] + sign * h * step
            side.append((block_sparse_train_fn(*y, mask, 0.125).double() * do.double()).sum().item())
        want = (side[0] - side[1]) / (2 * h)
        got = (grads[i].double() * step.double()).sum().item()
        size = (grads[i].double() * step.double()).norm().item()
        assert abs(got - want) <= 2e-2 * size, (i, got, want, size)


def test_no_queries_or_no_keys(dev):
    case("no queries, no keys")
    for Lq, Lk in ((0, 64), (64, 0)):
        q = torch.randn(1, 2, Lq, 64, dtype=BF16, device=dev, requires_grad=True)
        k, v = (torch.randn(1, 2, Lk, 64, dtype=BF16, device=dev, requires_grad=True) for _ in range(2))
        mask = torch.ones(1, 2, math.ceil(Lq / 64), math.ceil(Lk / 64), dtype=torch.bool, device=dev)
        out = block_sparse_train_fn(q, k, v, mask, 0.125)
        assert out.shape == q.shape and not out.any()
        for x, t in zip(torch.autograd.grad(out, (q, k, v), torch.ones_like(out)), (q, k, v)):
            assert x.shape == t.shape and not x.any()


def test_steps_repeat_and_overlap(dev):
    # The same step twice, and two steps at once on two streams: the same bits.
    case("repeated and concurrent steps")
    steps = []
    for seed in (12, 13):
        (q, k, v, do), g = _inputs(seed, BF16, 2, 20, 900, 900, 64)
        steps.append(([t.to(dev) for t in (q, k, v, do)], _mask(g, 2, 20, 900, 900, 0.3).to(dev)))

    def run(i):
        x, mask = steps[i]
        return _grads(lambda *y: block_sparse_train_fn(*y, mask, 0.125), *x)

    want = [run(0), run(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev), torch.cuda.Stream(dev)]
    for _ in range(3):
        got = [None, None]
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = run(i)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_step(dev):
    # Forward and backward halves in one graph, replayed with new inputs between eager work.
    case("captured step")
    (q, k, v, do), g = _inputs(14, BF16, 1, 4, 500, 500, 64)
    kv = kv_list_from_mask(_mask(g, 1, 4, 500, 500, 0.4).to(dev), 1, 4, 8, 8)
    x = [t.to(dev) for t in (q, k, v, do)]

    def step(q, k, v, do):
        out, lse = block_sparse_attention_lse(q, k, v, kv, 0.125)
        return (out, *block_sparse_attention_backward(do, q, k, v, out, lse, kv, 0.125))

    step(*x)  # (fills the dispatch orders' cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*x)
    for seed in range(4):
        new, _ = _inputs(20 + seed, BF16, 1, 4, 500, 500, 64)
        for t, n in zip(x, new):
            t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        want = step(*(t.clone() for t in x))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_autograd_step(dev):
    # torch's own way: forward and autograd.grad captured with leaves of their own.
    case("captured autograd step")
    (q, k, v, do), g = _inputs(15, FP16, 1, 3, 300, 300, 64)
    mask = _mask(g, 1, 3, 300, 300, 0.5).to(dev)
    x = [t.to(dev) for t in (q, k, v, do)]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        _grads(lambda *y: block_sparse_train_fn(*y, mask, 0.125), *x)
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _grads(lambda *y: block_sparse_train_fn(*y, mask, 0.125), *x)
    for seed in range(3):
        new, _ = _inputs(30 + seed, FP16, 1, 3, 300, 300, 64)
        for t, n in zip(x, new):
            t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        want = _grads(lambda *y: block_sparse_train_fn(*y, mask, 0.125), *x)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(dev):
    case("refusals")
    q = torch.zeros(1, 2, 128, 64, dtype=BF16, device=dev, requires_grad=True)
    mask = torch.ones(1, 2, 2, 2, dtype=torch.bool, device=dev)
    bias = torch.zeros(1, 2, 128, device=dev)
    kv = dense_kv_list(1, 2, 2, 2, dev)
    with pytest.raises(TypeError):
        block_sparse_train_fn(q, q.float(), q, mask, 0.125)
    with pytest.raises(TypeError):
        block_sparse_train_fn(q.double(), q.double(), q.double(), mask, 0.125)
    with pytest.raises(ValueError):
        block_sparse_train_fn(q, q[:, :, :64], q, mask, 0.125)
    with pytest.raises(ValueError):
        block_sparse_train_fn(q, q, q, mask[:, :, :1], 0.125)
    with pytest.raises(NotImplementedError):
        block_sparse_train_fn(q[..., :32], q[..., :32], q[..., :32], mask, 0.125)
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            block_sparse_train_fn(q, q, q, mask, scale)
    with pytest.raises(NotImplementedError):
        block_sparse_train_fn(q.float(), q.float(), q.float(), mask, 0.125, key_bias=bias)
    with pytest.raises(ValueError):
        block_sparse_train_fn(q, q, q, mask, 0.125, key_bias=bias.clone().requires_grad_())
    with pytest.raises(ValueError):
        block_sparse_train_fn(q, q, q, mask, 0.125, key_bias=bias.half())
    with pytest.raises(ValueError):
        block_sparse_train_fn(q, q, q, mask, 0.125, key_bias=bias[..., :100])
    with pytest.raises(NotImplementedError):
        block_sparse_train_fn(q, q, q, torch.ones(1, 2, 4, 4, dtype=torch.bool, device=dev), 0.125, BLOCK_M=32, BLOCK_N=32)
    with pytest.raises(ValueError):
        block_sparse_train_fn(q, q, q, mask, 0.125, BLOCK_M=96)
    with pytest.raises(ValueError):
        block_sparse_attention_train(q, q, q, dense_kv_list(1, 2, 2, 3, dev), 0.125)
    with pytest.raises(ValueError):
        block_sparse_attention_train(q.cpu(), q, q, kv, 0.125)
    out, lse = block_sparse_attention_lse(q, q, q, kv, 0.125)
    with pytest.raises(ValueError):
        block_sparse_attention_backward(out[:, :, :64], q, q, q, out, lse, kv, 0.125)
    with pytest.raises(ValueError):
        block_sparse_attention_backward(out, q, q, q, out, lse[..., :64], kv, 0.125)
    y = block_sparse_train_fn(q, q, q, mask, 0.125)
    with pytest.raises(RuntimeError):  # differentiable once
        torch.autograd.grad(y.float().sum(), q, create_graph=True)
    # a change of a saved tensor in place is noticed
    x = q.detach().clone().requires_grad_()
    z = x * 1
    y = block_sparse_train_fn(z, z, z, mask, 0.125)
    z.add_(1)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.float().sum(), x)


def test_block_sparse_triton_fn_still_refuses_gradients(dev):
    case("block_sparse_triton_fn has no gradients")
    q = torch.randn(1, 1, 64, 64, dtype=BF16, device=dev, requires_grad=True)
    o = block_sparse_triton_fn(q, q, q, torch.ones(1, 1, 1, 1, dtype=torch.bool, device=dev), 0.125)
    with pytest.raises(NotImplementedError):
        o.float().sum().backward()
    assert block_sparse_attention(q.detach(), q.detach(), q.detach(), dense_kv_list(1, 1, 1, 1, dev), 0.125).shape == q.shape
