"""What the backward pass cannot take is refused by the forward call already, where a gradient is to follow."""
import pytest
import torch

from conftest import case
from sparseattnfunctions_amd._kv import KVList
from sparseattnfunctions_amd.block_mask_attn import dense_kv_list
from sparseattnfunctions_amd.utils.block_sparse_attn_grad import (_plan, block_sparse_attention_train,
                                                                  block_sparse_train_fn)

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _leaves(dev, L=40, grads=(True, True, True)):
    g = torch.Generator().manual_seed(1)
    return [torch.randn(1, 1, L, 64, generator=g).to(BF16).to(dev).requires_grad_(x) for x in grads]


def test_tiny_scale(dev):
    case("sm_scale below the backward pass's")
    mask = torch.ones(1, 1, 1, 1, dtype=torch.bool, device=dev)
    leaves = _leaves(dev)
    with pytest.raises(NotImplementedError):
        block_sparse_train_fn(*leaves, mask, 1e-31)
    # without a gradient the forward pass takes it: the mean of v (off by its rounding and that of the sum)
    for followed in (False, True):
        with torch.set_grad_enabled(followed):
            x = [t.detach() for t in leaves] if followed else leaves
            out = block_sparse_train_fn(*x, mask, 1e-31)
        want = leaves[2].detach().double().mean(2, keepdim=True).expand(out.shape)
        assert not out.requires_grad
        assert ((out.double() - want).abs() <= 2 * 2.0 ** -8 * want.abs() + 2.0 ** -20).all()
    assert block_sparse_train_fn(*leaves, mask, 1e-29).requires_grad


def test_wide_lists(dev):
    # Lists wider than the transposed ones' counts: of a key or value's gradient alone.
    case("lists of more than 65535 entries")
    kv = dense_kv_list(1, 1, 1, 1, dev)
    idx = torch.zeros(1, 70000, dtype=torch.int32, device=dev)
    wide = KVList(idx, kv.cnt, 1, 1, 1, 1)
    for grads in ((True, True, True), (False, True, False), (False, False, True)):
        with pytest.raises(NotImplementedError):
            block_sparse_attention_train(*_leaves(dev, grads=grads), wide, 0.125)
    x = _leaves(dev, grads=(True, False, False))
    do = torch.ones_like(x[0])
    got = torch.autograd.grad(block_sparse_attention_train(*x, wide, 0.125), x[0], do)[0]
    assert torch.equal(got, torch.autograd.grad(block_sparse_attention_train(*x, kv, 0.125), x[0], do)[0])


def test_far_rows(dev):
    # Rows 32 MB apart: 40 of them lie within 2 GiB, and 64 more would not. q is refused; a gradient that
    # arrives so is copied.
    case("rows far apart")
    kv = dense_kv_list(1, 1, 1, 1, dev)
    leaves = _leaves(dev)
    step = 1 << 24
    base = torch.empty(40 * step, dtype=BF16, device=dev)
    far = base.as_strided((1, 1, 40, 64), (step, step, step, 1))
    far.copy_(leaves[0].detach())
    with torch.no_grad():
        want = block_sparse_attention_train(*leaves, kv, 0.125)
        assert torch.equal(block_sparse_attention_train(far, *leaves[1:], kv, 0.125), want)
    with pytest.raises(NotImplementedError):
        block_sparse_attention_train(far.detach().requires_grad_(), *leaves[1:], kv, 0.125)
    grads = [torch.autograd.grad(block_sparse_attention_train(*leaves, kv, 0.125), leaves, do)
             for do in (far.clone(memory_format=torch.contiguous_format), far)]
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_sizes_past_32_bits(dev):
    # A length cut to 32 bits would attend to 64 of the keys. (The lists' own checks come first, so the plan of such a call
    # is asked for directly.) More text blocks than a head has blocks mean all of them.
    case("sizes past 32 bits")
    plain = (64 * 64, 64 * 64, 64, 1)
    for shape, Lk in (((1, 1, 64, 64), 2 ** 32 + 64), ((1, 1, 2 ** 32 + 64, 64), 64), ((2 ** 32 + 1, 1, 64, 64), 64)):
        with pytest.raises(ValueError, match="32 bits"):
            _plan(BF16, dev, torch.Size(shape), Lk, plain, plain, plain, 1, 0.0, False, 0.125, 0, False)
    leaves = _leaves(dev)
    mask = torch.ones(1, 1, 1, 1, dtype=torch.bool, device=dev)
    want = block_sparse_train_fn(*leaves, mask, 0.125, n_text_blocks=1)
    assert torch.equal(block_sparse_train_fn(*leaves, mask, 0.125, n_text_blocks=2 ** 40), want)
