"""What the backward call of attention with score rules is given when hooks have moved its saved tensors, without a GPU: the
library's launches are recorded, not made."""
import contextlib

import pytest
import torch

from sparseattnfunctions_amd import _lib
from sparseattnfunctions_amd.utils import scored_attn


class Recorder:
    """The library, but for the two calls that launch kernels."""

    def __init__(self, lib):
        self.lib, self.calls = lib, []

    def __getattr__(self, name):
        if name in ("sa_attn_scored_fwd", "sa_attn_scored_bwd"):
            return lambda args, stream: self.calls.append(args) or 0
        return getattr(self.lib, name)


@pytest.fixture
def recorder(monkeypatch):
    r = Recorder(_lib.load())
    monkeypatch.setattr(_lib, "load", lambda: r)
    monkeypatch.setattr(_lib, "on", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "stream_of", lambda t: None)
    return r


B, H, L, D = 3, 2, 320, 64


def moved_copy(t, how):
    if how == "contiguous":
        return t.clone(memory_format=torch.contiguous_format)
    # between other values, and 4 bytes off
    wide = torch.zeros(*t.shape[:-1], 3, dtype=t.dtype)
    wide[..., 1:] = t
    return wide[..., 1:]


@pytest.mark.parametrize("how", ["contiguous", "apart"])
@pytest.mark.parametrize("cut", ["longer", "every other", "one for all", "whole"])
def test_moved_ranges(recorder, cut, how):
    g = torch.Generator().manual_seed(1)
    many = torch.randint(0, L, (2 * B, 500, 2), generator=g, dtype=torch.int32)
    ranges = {"longer": many[:B, :L], "every other": many[::2, 100:100 + L], "one for all": many[:1, :L],
              "whole": many[:B, :L].clone()}[cut]
    q, k, v, do = (torch.randn(B, H, L, D, generator=g) for _ in range(4))
    slopes, table, buckets = torch.randn(H, generator=g), torch.randn(9, H, generator=g), torch.zeros(7, dtype=torch.int32)
    checked = scored_attn._check_ranges(ranges, q, B, L)
    _, state = scored_attn._forward(q, k, v, 0.2, 0.0, slopes, table, buckets, checked, None, 0, scored_attn._KEYS)
    i = [t is checked for t in state.tensors].index(True)
    tensors = list(state.tensors)
    tensors[i] = moved_copy(checked, how)
    if how == "apart":
        tensors[-3:] = (torch.stack((t, t), -1)[..., 1] for t in tensors[-3:])
    scored_attn._backward(do, scored_attn.ScoredState(tuple(tensors), state.call, state.args), (True, True, True, False))
    forward, backward = recorder.calls
    assert forward.ranges == ranges.data_ptr() and forward.ranges_stride == (0 if cut == "one for all" else ranges.stride(0) // 2)
    if how == "contiguous":
        assert backward.ranges == tensors[i].data_ptr() and backward.ranges_stride == L
    else:  # not as the kernels read them: copied
        assert backward.ranges != tensors[i].data_ptr() and backward.ranges % 8 == 0
        assert backward.ranges_stride == L
        assert all(getattr(backward, n) != t.data_ptr() for n, t in zip(("slopes", "table", "buckets"), tensors[-3:]))
