"""Attention with score rules on the GPU at the ends of what its arguments allow, against 64 bits."""
import pytest
import torch

import scored_reference as ref
from conftest import case
from sparseattnfunctions_amd.utils.scored_attn import row_ranges, scored_attention

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
NAMES = ("out", "dq", "dk", "dv", "dtable")


@pytest.mark.parametrize("cut", ["longer", "every other", "one for all"])
def test_moved_ranges(dev, cut):
    case(f"ranges cut out of others ({cut}), moved by hooks")
    B, L = 3, 320
    lengths = torch.tensor([[100, 150], [320, 0], [7, 300]] * 2, device=dev)
    many = torch.full((2 * B, 500, 2), -2 ** 31, dtype=torch.int32, device=dev)
    many[:, :L] = row_ranges(lengths, L)
    ranges = {"longer": many[:B, :L], "every other": many[::2, :L], "one for all": many[:1, :L]}[cut]
    q, k, v, do = ref.inputs(12, B, 2, 1, L, L, 64, FP32, dev)
    for t in (q, k, v):
        t.requires_grad_()
    want = ref.train(q, k, v, do, 0.2, ranges=ranges)
    with torch.autograd.graph.save_on_cpu():
        out = scored_attention(q, k, v, 0.2, ranges=ranges)
        got = [out, *torch.autograd.grad(out, (q, k, v), do)]
    for n, x in zip(NAMES, got):
        ref.check(n, x, want[n])
