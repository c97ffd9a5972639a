"""Gradients over lists so long that single probabilities are far below one."""
import pytest
import torch

from conftest import case
from sparseattnfunctions_amd.utils.block_sparse_attn_grad import block_sparse_train_fn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_even_attention_over_many_keys(dev, dtype, bias, D):
    # q = 0: every probability is 1 / n, 83.5 steps of fp16's subnormal numbers at this n. dv is 1 / n of the sum of the
    # rows' do (positive ones, so that nothing cancels): off by a rounding of P and of dv, u each, of the row sum (the
    # sum of n equal rounded terms, u) and of fp32 sums.
    case(f"even attention over 200925 keys {dtype} bias={bias} D={D}")
    n, Lq = 200925, 70
    g = torch.Generator().manual_seed(5)
    q = torch.zeros(1, 1, Lq, D, dtype=dtype)
    k, v = (torch.randn(1, 1, n, D, generator=g).to(dtype) for _ in range(2))
    do = (1000 * (0.5 + torch.rand(1, 1, Lq, D, generator=g))).to(dtype)
    mask = torch.ones(1, 1, 2, (n + 63) // 64, dtype=torch.bool, device=dev)
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
    key_bias = torch.zeros(1, 1, n, device=dev) if bias else None
    out = block_sparse_train_fn(*leaves, mask, 0.125, key_bias=key_bias)
    (dv,) = torch.autograd.grad(out, leaves[2:], do.to(dev))
    want = do.double().sum(2, keepdim=True) / n
    u = torch.finfo(dtype).eps / 2
    off = (dv.double().cpu() - want).abs() / want
    assert off.max() <= 3 * u + 2.0 ** -15, off.max().item()


@pytest.mark.parametrize("D", [64, 128])
def test_long_fp16_lists_split_over_workgroups(dev, D):
    # Few key blocks that many rows list, in lists wide enough for scaled probabilities: one block's entries are split and
    # merged. The same rows over a list of those blocks alone: dv differs by roundings of P and of dv.
    case(f"wide lists, split D={D}")
    Lq, Lk = 4500, 64 * 260
    g = torch.Generator().manual_seed(6)
    q, k, v, do = (torch.randn(1, 1, L, D, generator=g).half().to(dev) for L in (Lq, Lk, Lk, Lq))
    mask = torch.zeros(1, 1, (Lq + 63) // 64, Lk // 64, dtype=torch.bool, device=dev)
    mask[..., :2] = True

    def grads(k, v, mask):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = block_sparse_train_fn(*leaves, mask, 0.125)
        return (out, *torch.autograd.grad(out, leaves, do))

    wide, narrow = grads(k, v, mask), grads(k[:, :, :128], v[:, :, :128], mask[..., :2])
    s = torch.softmax(0.125 * q.double().cpu() @ k[:, :, :128].double().cpu().transpose(2, 3), 3)
    reach = s.transpose(2, 3) @ do.double().cpu().abs()
    u = 2.0 ** -11
    for x in (wide, narrow):
        # a rounding each of P (below fp16's normal range 2^-25), of the row sum's terms and of dv
        want = s.transpose(2, 3) @ do.double().cpu()
        off = (x[3][:, :, :128].double().cpu() - want).abs()
        small = 2.0 ** -25 * do.double().cpu().abs().sum(2, keepdim=True)
        assert (off <= 1.05 * 3 * u * reach + small + u * want.abs()).all()
    assert not wide[3][:, :, 128:].any()
