"""Rotary positions, the mask builders, attention and their gradients together, as a layer's training
step uses them, against 64-bit torch with autograd on the lists that the processor chose."""
import math

import pytest
import torch

from conftest import case
from sparseattnfunctions_amd.block_mask_attn import BlockSparseAttention
from sparseattnfunctions_amd.combined_attn import CombinedAttn
from sparseattnfunctions_amd.utils.rotary import VideoRotary, rotary_frequencies, video_positions
from sparseattnfunctions_amd.workloads import Geometry, cogvideox_qkv

pytestmark = pytest.mark.gpu

GEOM = Geometry(text_len=70, T=3, Hp=10, Wp=12)
AXES = (16, 24, 24)


def _turn(x, geom, layout):
    """x [B,H,L,64] in 64 bits, differentiable."""
    ang = torch.cat([p.double()[:, None] * torch.tensor(rotary_frequencies(d)[0], dtype=torch.float64)
                     for p, d in zip(video_positions(geom), AXES)], 1)
    cos, sin = ang.cos(), ang.sin()
    text, video = x[:, :, :geom.text_len], x[:, :, geom.text_len:]
    if layout == "interleaved":
        a, b = video[..., 0::2], video[..., 1::2]
        video = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(3)
    else:
        a, b = video[..., :32], video[..., 32:]
        video = torch.cat((a * cos - b * sin, b * cos + a * sin), 3)
    return torch.cat((text, video), 2)


def _attend(q, k, v, mask, scale):
    L = q.shape[2]
    seen = mask.repeat_interleave(64, 2).repeat_interleave(64, 3)[..., :L, :L]
    return torch.softmax((scale * q @ k.transpose(2, 3)).masked_fill(~seen, -math.inf), 3) @ v


def _leaves(seed, dev, B=2, H=3, geom=GEOM):
    q, k, v = cogvideox_qkv(seed, B=B, H=H, geom=geom)
    do = torch.randn(q.shape, generator=torch.Generator().manual_seed(seed + 100)).bfloat16()
    return [t.to(dev).requires_grad_() for t in (q, k, v)], do.to(dev)


def _check(got, want):
    # Relative 2-norm errors: the turned q and k, P or dS, the row sum, out in delta, the result and the
    # gradient of the rotation are rounded to bf16, each off by at most 2^-8 / sqrt(3) in the mean square:
    # sqrt(7) 2^-8 / sqrt(3) = 1.53 2^-8. A turned key's rounding moves scores of the size 10 by up to 2^-8
    # of them, which counts as that many more: 3 2^-8.
    for name, x, y in zip(("out", "dq", "dk", "dv"), got, want):
        x, y = x.detach().double().cpu(), y.detach().double()
        assert torch.isfinite(x).all()
        off = ((x - y).norm() / y.norm()).item()
        assert off <= 3 * 2.0 ** -8, (name, off)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("kind", ["topk", "dense", "combined", "combined warm"])
def test_layer_step(dev, kind, layout):
    case(f"layer step {kind} {layout}")
    rotary = VideoRotary(GEOM, AXES, layout=layout)
    leaves, do = _leaves(3, dev)
    if kind in ("topk", "dense"):
        proc = BlockSparseAttention(64, keep_ratio=0.4, geometry=GEOM, trainable=True, rotary=rotary)
        plain = BlockSparseAttention(64, keep_ratio=0.4, geometry=GEOM, rotary=rotary)
        out = proc(*leaves) if kind == "topk" else proc.forward_dense(*leaves)
    else:
        warm = 1 if kind == "combined warm" else 0
        proc = CombinedAttn(warmup_epoch=warm, geometry=GEOM, global_ratio=0.3, window=(1, 2, 2), trainable=True,
                            rotary=rotary)
        out = proc(*leaves)
    grads = torch.autograd.grad(out, leaves, do)
    n = math.ceil(GEOM.L / 64)
    mask = proc.last_kv.to_mask().cpu() if kind in ("topk", "combined") else torch.ones(2, 3, n, n, dtype=torch.bool)
    assert kind in ("dense", "combined warm") or not mask.all()
    ref = [t.detach().cpu().double().requires_grad_() for t in leaves]
    # (the layer rounds the turned q and k to bf16, and the oracle does so too)
    turned = []
    for t in ref[:2]:
        y = _turn(t, GEOM, layout)
        turned.append(y + (y.detach().bfloat16().double() - y.detach()))
    want = _attend(*turned, ref[2], mask, 1 / 8)
    _check((out, *grads), (want, *torch.autograd.grad(want, ref, do.cpu().double())))
    if kind == "topk":  # without gradients: the same lists
        with torch.no_grad():
            plain(*leaves)
        assert torch.equal(plain.last_kv.to_mask().cpu(), mask)


def test_steps_of_a_small_model(dev):
    # Two layers with weights of their own, two optimizer steps: every gradient against 64-bit autograd on
    # the lists that the layers chose.
    case("two layers")
    geom = Geometry(text_len=20, T=2, Hp=6, Wp=10)
    rotary = VideoRotary(geom, AXES)
    g = torch.Generator().manual_seed(5)
    H, E = 2, 48
    x = torch.randn(1, geom.L, E, generator=g)
    weights = [torch.randn(E, 3 * H * 64, generator=g) / math.sqrt(E) for _ in range(2)]
    outs = [torch.randn(H * 64, E, generator=g) / math.sqrt(H * 64) for _ in range(2)]
    procs = [BlockSparseAttention(64, keep_ratio=0.6, geometry=geom, trainable=True, rotary=rotary) for _ in range(2)]
    params = [t.to(dev).requires_grad_() for t in (*weights, *outs)]

    def model(params, attention, x):
        for i in range(2):
            q, k, v = (x @ params[i]).unflatten(2, (3, H, 64)).permute(2, 0, 3, 1, 4)
            x = x + attention(i, q, k, v).transpose(1, 2).flatten(2) @ params[2 + i]
        return x

    for step in range(2):
        y = model(params, lambda i, q, k, v: procs[i](q.bfloat16(), k.bfloat16(), v.bfloat16()).float(), x.to(dev))
        loss = y.square().mean()
        got = torch.autograd.grad(loss, params)
        masks = [p.last_kv.to_mask().cpu() for p in procs]
        ref = [t.detach().cpu().double().requires_grad_() for t in params]
        want = model(ref, lambda i, q, k, v: _attend(_turn(q, geom, "interleaved"), _turn(k, geom, "interleaved"), v, masks[i],
                                                     1 / 8), x.double()).square().mean()
        want = torch.autograd.grad(want, ref)
        for a, b in zip(got, want):
            # q, k, v, the turned ones, P or dS, out, and their gradients: some twenty bf16 roundings in a
            # chain of two layers, sqrt(20) 2^-8 / sqrt(3) = 2.6 2^-8, and their effect on scores
            off = ((a.cpu().double() - b).norm() / b.norm()).item()
            assert off <= 5 * 2.0 ** -8, off
        with torch.no_grad():
            for t, d in zip(params, got):
                t -= 0.1 * d


def test_captured_layer_step(dev):
    # Rotary, lists, forward and backward of a layer in one graph, replayed on new inputs.
    case("captured layer step")
    rotary = VideoRotary(GEOM, AXES)
    proc = BlockSparseAttention(64, keep_ratio=0.4, geometry=GEOM, trainable=True, rotary=rotary)
    leaves, do = _leaves(7, dev)

    def step():
        fresh = [t.detach().requires_grad_() for t in leaves]  # leaves of the graph's own
        out = proc(*fresh)
        return (out, *torch.autograd.grad(out, fresh, do))

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in range(3):
        new, d = _leaves(20 + seed, dev)
        with torch.no_grad():
            for t, n in zip((*leaves, do), (*new, d)):
                t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_processors_without_gradients_are_unchanged(dev):
    case("processors as before")
    leaves, _ = _leaves(9, dev)
    q, k, v = (t.detach() for t in leaves)
    a = BlockSparseAttention(64, keep_ratio=0.4, geometry=GEOM)
    b = BlockSparseAttention(64, keep_ratio=0.4, geometry=GEOM, trainable=True)
    out = a(q, k, v)
    assert not a(*leaves).requires_grad
    got = b(q, k, v)
    assert torch.equal(a.last_kv.to_mask(), b.last_kv.to_mask()) and not got.requires_grad
    # fp16 scores in one, bf16 in the other: 2^-6 in the exponent at most
    assert (out.float() - got.float()).abs().max() <= 2e-2
    with pytest.raises(NotImplementedError):
        b.forward_backup(q, k, v)
    with pytest.raises(NotImplementedError):
        CombinedAttn(trainable=True, head_routing=True)
    with pytest.raises(NotImplementedError):
        CombinedAttn(trainable=True)(q, k, v, use_rearranger=True)
    with pytest.raises(ValueError):
        VideoRotary(GEOM, (16, 24))
    with pytest.raises(ValueError):
        VideoRotary(GEOM, layout="pairs")
    with pytest.raises(ValueError):
        VideoRotary(GEOM, positions=torch.zeros(3, 5))
    # another stream than the one that made the table
    rotary = VideoRotary(GEOM, AXES, positions=0.5 * video_positions(GEOM).float())
    want = rotary(q, k)
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        got = rotary(q, k)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
