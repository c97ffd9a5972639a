"""A caller's block lists (KVList), as the trainable processors pass them, at the sizes where launches are dealt out in
special ways: last round by length, split text blocks, split remainders, split lists. Their key side is transposed by the
backward call; a mask's both sides are made by the forward call. Both lists are ascending, so all results agree bit for
bit."""
import dataclasses
import math

import pytest
import torch

from conftest import case
from grad_reference import check, reference, unit
from sparseattnfunctions_amd._kv import kv_list_from_mask
from sparseattnfunctions_amd.utils.block_sparse_attn_grad import (
    block_sparse_attention_backward, block_sparse_attention_lse, block_sparse_attention_train, block_sparse_train_fn,
    transpose_kv_list)

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32

# B, H, Lq, Lk, D, type, density, text blocks, bias
CASES = {
    "last round by length, 64": (1, 12, 4170, 4170, 64, BF16, 0.1, 0, False),
    "last round by length, 128": (1, 33, 2090, 2090, 128, FP16, 0.1, 0, False),
    "text blocks of the query pass": (2, 12, 330, 2700, 64, BF16, 0.2, 4, True),
    "text blocks of the key pass": (1, 24, 2700, 200, 128, BF16, 0.2, 9, False),
    "text blocks of both": (1, 3, 6200, 6150, 64, BF16, 0.2, 1, False),
    "fp32 remainder by two": (1, 9, 1100, 1080, 64, FP32, 0.3, 0, False),
    "fp32 remainder by three, text": (1, 17, 2100, 2080, 64, FP32, 0.3, 2, False),
    "fp32 remainder, 128": (1, 9, 2100, 2080, 128, FP32, 0.3, 0, False),
    "split lists of few query blocks": (1, 3, 70, 4500, 64, BF16, 0.4, 0, False),
    "split lists of few key blocks": (1, 3, 4500, 70, 64, BF16, 0.6, 0, False),
    "split lists of few key blocks, fp32": (1, 3, 4500, 70, 128, FP32, 0.6, 0, False),
    "split lists of few key blocks, bias": (1, 3, 4500, 70, 64, FP16, 0.6, 0, True),
    "one pair of waves": (2, 45, 580, 640, 64, BF16, 0.4, 0, False),
}


@pytest.mark.parametrize("name", CASES)
def test_lists_and_masks_agree(dev, name):
    B, H, Lq, Lk, D, dtype, density, text, biased = CASES[name]
    case(f"lists: {name}")
    g = torch.Generator().manual_seed(23)
    q, k, v, do = (torch.randn(B, H, L, D, generator=g).to(dtype) for L in (Lq, Lk, Lk, Lq))
    nq, nk = math.ceil(Lq / 64), math.ceil(Lk / 64)
    mask = torch.rand(B, H, nq, nk, generator=g) < density * 2 * torch.rand(B, H, nq, 1, generator=g)
    mask[:, :, :text] = True
    mask[..., :text] = True
    mask[:, :, -1] = False  # rows without a key
    bias = torch.randn(B, 1, Lk, generator=g) if biased else None
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
    dod, mask_d, bias_d = do.to(dev), mask.to(dev), None if bias is None else bias.to(dev)
    out = block_sparse_train_fn(*leaves, mask_d, 0.125, key_bias=bias_d, n_text_blocks=text)
    want = (out, *torch.autograd.grad(out, leaves, dod))
    kv = kv_list_from_mask(mask_d, B, H, nq, nk)
    out = block_sparse_attention_train(*leaves, kv, 0.125, key_bias=bias_d, n_text_blocks=text)
    got = (out, *torch.autograd.grad(out, leaves, dod))
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    # the two halves, and gradients of the key side alone
    with torch.no_grad():
        out, lse = block_sparse_attention_lse(*leaves, kv, 0.125, key_bias=bias_d, n_text_blocks=text)
        halves = block_sparse_attention_backward(dod, *leaves, out, lse, kv, 0.125, key_bias=bias_d, n_text_blocks=text,
                                                 needs=(False, True, True))
    assert halves[0] is None and all(torch.equal(x, y) for x, y in zip((out, *halves[1:]), (want[0], *want[2:])))
    # two heads against 64 bits
    some = slice(H - 2, H)
    check([x[:, some] for x in got], reference(*(t[:, some] for t in (q, k, v, do, mask)), 0.125, bias=bias),
          norm=1.5 * unit(dtype) if dtype != FP32 else 64 * 2.0 ** -24)


def test_transposing_refuses_lists_of_other_sizes(dev):
    # (the kernel would read past them)
    case("transposed lists, refusals")
    kv = kv_list_from_mask(torch.ones(1, 2, 3, 4, dtype=torch.bool, device=dev), 1, 2, 3, 4)
    assert transpose_kv_list(kv)[0].tolist() == [[0, 3, 6, 9, 12]] * 2
    for bad in (dict(idx=kv.idx.long()), dict(cnt=kv.cnt.long()), dict(cnt=kv.cnt[:5]), dict(idx=kv.idx[:4]), dict(H=3),
                dict(nqb=4), dict(idx=kv.idx.flatten()), dict(idx=kv.idx[:, ::2]), dict(cnt=kv.cnt.cpu())):
        with pytest.raises(ValueError):
            transpose_kv_list(dataclasses.replace(kv, **bad))
