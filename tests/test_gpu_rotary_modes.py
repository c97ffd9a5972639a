"""Rotary positions across autograd's modes."""
import copy
import pickle

import pytest
import torch

from conftest import case
from sparseattnfunctions_amd.block_mask_attn import BlockSparseAttention
from sparseattnfunctions_amd.utils.rotary import VideoRotary, apply_rotary, rotary_table, video_positions
from sparseattnfunctions_amd.workloads import Geometry

pytestmark = pytest.mark.gpu

GEOM = Geometry(text_len=70, T=2, Hp=6, Wp=10)


def _qkv(dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(1, 2, GEOM.L, 64, generator=g).bfloat16().to(dev) for _ in range(4)]


@pytest.mark.parametrize("given", [False, True])
def test_table_made_in_inference_mode_serves_training(dev, given):
    # A validation pass before the first step: the cached table must not be an inference tensor.
    case(f"table made in inference mode, positions given: {given}")
    q, k, v, do = _qkv(dev)
    positions = None
    if given:
        with torch.inference_mode():
            positions = video_positions(GEOM, device=dev)
    rotary = VideoRotary(GEOM, positions=positions)
    proc = BlockSparseAttention(64, keep_ratio=0.6, geometry=GEOM, trainable=True, rotary=rotary)
    with torch.inference_mode():
        seen = proc(q, k, v)
    assert not rotary.table(dev).is_inference()
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = proc(*leaves)
    grads = torch.autograd.grad(out, leaves, do)
    assert torch.equal(out, seen)
    fresh = BlockSparseAttention(64, keep_ratio=0.6, geometry=GEOM, trainable=True, rotary=VideoRotary(GEOM))
    want = torch.autograd.grad(fresh(*leaves), leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(grads, want))


@pytest.mark.parametrize("trained", ["q", "k"])
def test_a_frozen_side_has_no_gradient(dev, trained):
    # Only q or only k is followed: the turned other one is not, so that the attention behind it computes no gradient of it.
    case(f"only {trained} followed")
    q, k, v, do = _qkv(dev, 1)
    rotary = VideoRotary(GEOM)
    want = rotary(q, k)
    leaf = (q if trained == "q" else k).requires_grad_()
    turned = rotary(q, k)
    assert [t.requires_grad for t in turned] == [trained == "q", trained == "k"]
    assert all(torch.equal(a, b) for a, b in zip(turned, want))
    if trained == "q":
        assert not apply_rotary(q, k, rotary.table(dev), skip=GEOM.text_len)[1].requires_grad
    proc = BlockSparseAttention(64, keep_ratio=0.6, geometry=GEOM, trainable=True, rotary=rotary)
    out = proc(q, k, v)
    wanted = [f is not None for f, _ in out.grad_fn.next_functions[:3]]
    assert wanted == [trained == "q", trained == "k", False]
    (only,) = torch.autograd.grad(out, leaf, do)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    both = torch.autograd.grad(proc(*leaves), leaves, do)
    assert torch.equal(only, both[0 if trained == "q" else 1])
    with torch.no_grad():
        assert not any(t.requires_grad for t in rotary(q, k))


def test_sizes_past_32_bits_are_refused(dev):
    # Expanded tensors take no memory; a length cut to 32 bits would turn four tokens.
    case("rotary sizes past 32 bits")
    n = 2 ** 32 + 4
    q = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16, device=dev)
    table = torch.zeros(4, 32, 2, device=dev)
    rows = torch.zeros(1, dtype=torch.int32, device=dev)
    for far in (q.expand(1, 1, n, 64), q.expand(n, 1, 1, 64), q.expand(1, n, 1, 64)):
        for a, b in ((far, None), (q, far) if far.shape[1] == n else (far, far)):
            with pytest.raises(ValueError, match="at most"):
                apply_rotary(a, b, table, rows=rows.expand(a.shape[2]))
    with pytest.raises(ValueError, match="at most"):
        apply_rotary(q, None, table[:1].expand(n, 32, 2))


def test_positions_are_not_differentiated(dev):
    # A gradient that would silently be lost is refused, as one of the table is.
    case("positions that require gradients")
    positions = torch.arange(5.0, device=dev, requires_grad=True)
    with pytest.raises(ValueError, match="detach"):
        rotary_table(positions, 64)
    with pytest.raises(ValueError, match="detach"):
        VideoRotary(GEOM, positions=video_positions(GEOM).float().requires_grad_()).table(dev)
    assert torch.equal(rotary_table(positions.detach(), 64), rotary_table(torch.arange(5, device=dev), 64))


def test_processors_can_be_copied_and_pickled(dev):
    # An averaged copy of a model copies its processors, tables made or not; the copy makes its own.
    case("copied processors")
    q, k, v, _ = _qkv(dev)
    proc = BlockSparseAttention(64, keep_ratio=0.6, geometry=GEOM, trainable=True, rotary=VideoRotary(GEOM))
    want = proc(q, k, v)
    for copied in (copy.deepcopy(proc), pickle.loads(pickle.dumps(proc.rotary))):
        got = copied(q, k, v) if isinstance(copied, BlockSparseAttention) else copied(q, k)
        ref = (want,) if isinstance(copied, BlockSparseAttention) else proc.rotary(q, k)
        assert all(torch.equal(a, b) for a, b in zip((got,) if torch.is_tensor(got) else got, ref))
