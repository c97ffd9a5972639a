"""Rotary positions of queries and keys, on MI355X.

The reference's processors receive q and k that the host model has turned by their tokens' positions
(text first, then video tokens in (t, h, w) order, SildingTileAttention.py:100-105); this module is
that step:

  * `rotary_table(positions, axes)`: the cosines and sines of a sequence's positions, made once per
    geometry (`sa_rotary_table`); `video_positions(geometry)` are those of a video;
  * `apply_rotary(q, k, table)`: q and k turned in one launch (`sa_rotary_apply`), differentiable;
    `apply_rotary_(q, k, table)` does it in place;
  * `VideoRotary(geometry)`: both for a video, as the processors take it.

A head's first 2 * pairs values turn in pairs, (a, b) -> (a cos - b sin, b cos + a sin), computed in
fp32 and rounded once; the others stay. Layouts: "interleaved" pairs values 2i and 2i + 1, "half"
values i and i + pairs.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional, Sequence, Union

import torch
from torch.autograd import forward_ad

from .. import _lib

LAYOUTS = ("interleaved", "half")
MAX_PAIRS = 128
MAX_SIZE = 2 ** 31 - 256  # of a dimension (`sa_rotary_apply` takes 32-bit ones)
_POSITION_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2, torch.float64: 3}
_SCALINGS = {"linear": {"factor"}, "ntk": {"factor"},
             "yarn": {"factor", "original_length", "beta_fast", "beta_slow"}}


def rotary_frequencies(dims: int, theta: float = 10000.0, scaling: Optional[dict] = None):
    """(frequencies, factor) of an axis of `dims` values: radians per position of its dims / 2 pairs,
    theta^(-2i/dims), and the factor of their cosines and sines. `scaling` stretches them for contexts
    `factor` times as long as the trained one:

      {"type": "linear", "factor": s}   positions divided by s;
      {"type": "ntk", "factor": s}      theta * s^(dims / (dims - 2)): the slowest pair is stretched s
                                        times, the fastest is not;
      {"type": "yarn", "factor": s, "original_length": n, "beta_fast": 32, "beta_slow": 1}
                                        pairs with more than beta_fast turns over the trained length n
                                        keep their frequency, those with fewer than beta_slow are
                                        divided by s, linearly in the turns between; cosines and
                                        sines times 0.1 ln(s) + 1.

    This is YaRN's ramp as its paper writes it. Checkpoints are also trained with one that is linear in the pair's
    index between the two limits, whose frequencies differ by up to a factor of two in the middle: not this
    function's.
    """
    if dims <= 0 or dims % 2:
        raise ValueError(f"an axis has an even number of values, got {dims}")
    if not (math.isfinite(theta) and theta > 0):
        raise ValueError(f"theta must be finite and > 0, got {theta}")
    kind, s = None, 1.0
    if scaling is not None:
        kind = scaling.get("type")
        unknown = set(scaling) - {"type"} - _SCALINGS.get(kind, set())
        if kind not in _SCALINGS or unknown:
            raise ValueError(f"scaling {scaling}: type 'linear', 'ntk' or 'yarn' with its own entries")
        s = float(scaling["factor"]) if "factor" in scaling else math.nan
        if not (math.isfinite(s) and s >= 1):
            raise ValueError(f"scaling {scaling}: factor must be finite and >= 1")
    if kind == "ntk" and dims > 2:  # (the one pair of two values does not depend on theta)
        theta = theta * s ** (dims / (dims - 2))
    freq = [theta ** (-2.0 * i / dims) for i in range(dims // 2)]
    if kind == "linear":
        freq = [f / s for f in freq]
    if kind != "yarn":
        return freq, 1.0
    n, fast, slow = (float(scaling.get(x, d)) for x, d in (("original_length", math.nan), ("beta_fast", 32),
                                                           ("beta_slow", 1)))
    if not (math.isfinite(n) and n > 0 and fast > slow):
        raise ValueError(f"scaling {scaling}: original_length > 0 and beta_fast > beta_slow")
    out = []
    for f in freq:
        keep = min(1.0, max(0.0, (n * f / (2 * math.pi) - slow) / (fast - slow)))
        out.append(keep * f + (1 - keep) * f / s)
    return out, 0.1 * math.log(s) + 1.0


@functools.lru_cache(maxsize=256)
def _frequency_arrays(axes, theta, scaling):
    """The host arrays of `sa_rotary_table`, which depend on nothing but these settings."""
    freq, factors = [], []
    for dims in axes:
        f, m = rotary_frequencies(dims, theta, dict(scaling) if scaling is not None else None)
        freq += f
        factors.append(m)
    if len(freq) > MAX_PAIRS or len(axes) > 4:
        raise ValueError(f"axes {axes}: at most 4 axes and {2 * MAX_PAIRS} values")
    return ((ctypes.c_int32 * len(axes))(*(d // 2 for d in axes)), (ctypes.c_double * len(freq))(*freq),
            (ctypes.c_double * len(axes))(*factors), len(freq))


def rotary_table(positions: torch.Tensor, axes: Union[int, Sequence[int]], theta: float = 10000.0,
                 scaling: Optional[dict] = None) -> torch.Tensor:
    """fp32 [L, pairs, 2]: cosine and sine of every token's pairs.

    `positions` [L] or [n_axes, L] on the GPU, int32, int64, fp32 or fp64 (any strides); `axes` how many
    of the head's values turn with each axis of the positions, e.g. 64 for one, (16, 24, 24) for (t, h,
    w): consecutive pairs, axis by axis, each with its own frequencies (`rotary_frequencies`). At most 4
    axes and 256 values. Angles are formed and reduced in 64 bits, so positions in the millions keep
    full accuracy."""
    axes = (int(axes),) if isinstance(axes, int) else tuple(int(d) for d in axes)
    _lib.require_gpu(positions)
    if positions.dtype not in _POSITION_TYPES:
        raise TypeError(f"positions must be int32, int64, fp32 or fp64, got {positions.dtype}")
    if positions.requires_grad:
        raise ValueError("positions are not differentiated; pass positions.detach()")
    if positions.dim() == 1:
        positions = positions[None]
    if positions.dim() != 2 or positions.shape[0] != len(axes):
        raise ValueError(f"positions of shape {tuple(positions.shape)} for {len(axes)} axes")
    pairs_of, freq, factors, pairs = _frequency_arrays(
        axes, float(theta), tuple(sorted(scaling.items())) if scaling is not None else None)
    L = positions.shape[1]
    table = torch.empty(L, pairs, 2, dtype=torch.float32, device=positions.device)
    if L == 0:
        return table
    with _lib.on(positions.device):
        rc = _lib.load().sa_rotary_table(positions.data_ptr(), _POSITION_TYPES[positions.dtype],
                                         _lib.i64(*positions.stride()), L, len(axes), pairs_of, freq, factors,
                                         table.data_ptr(), _lib.stream_of(positions))
    _lib.check(rc, "sa_rotary_table")
    return table


def video_positions(geometry, device=None) -> torch.Tensor:
    """int32 [3, n_video]: (t, h, w) of the video tokens of a `workloads.Geometry`, in their order;
    their table goes with `skip=geometry.text_len`."""
    t, h, w = torch.meshgrid(*(torch.arange(n, dtype=torch.int32, device=device)
                               for n in (geometry.T, geometry.Hp, geometry.Wp)), indexing="ij")
    return torch.stack((t.reshape(-1), h.reshape(-1), w.reshape(-1)))


class VideoRotary:
    """The rotary positions of a video's tokens, as a processor's `rotary`: `rotary(q, k)` is
    `apply_rotary` with the table of `geometry` (a `workloads.Geometry`), its text tokens left alone.

    `axes` are the values of a head that turn with t, h and w (`rotary_table`); `positions` ([3,
    n_video]) replaces `video_positions`, e.g. for a grid rescaled to the trained one. The table of a
    device is made by its first call, which waits for it, so that later calls may run on any stream; a call
    captured into a graph needs one before."""

    def __init__(self, geometry, axes: Sequence[int] = (16, 24, 24), theta: float = 10000.0,
                 scaling: Optional[dict] = None, layout: str = "interleaved",
                 positions: Optional[torch.Tensor] = None):
        if layout not in LAYOUTS:
            raise ValueError(f"layout must be one of {LAYOUTS}, got {layout!r}")
        if len(axes) != 3:
            raise ValueError(f"axes {tuple(axes)}: one number of values each for t, h and w")
        _frequency_arrays(tuple(axes), float(theta), tuple(sorted(scaling.items())) if scaling is not None else None)
        if positions is not None and tuple(positions.shape) != (3, geometry.n_video):
            raise ValueError(f"positions of shape {tuple(positions.shape)}, expected (3, {geometry.n_video})")
        self.geometry, self.axes, self.theta, self.scaling = geometry, tuple(axes), theta, scaling
        self.layout, self.positions = layout, positions
        self._tables = {}  # device -> (table, the stream it was made on)

    def __getstate__(self):  # a copy makes its own tables (streams can neither be copied nor pickled)
        return {**self.__dict__, "_tables": {}}

    def table(self, device) -> torch.Tensor:
        device = torch.device(device)
        if device.index is None:
            device = torch.device(device.type, torch.cuda.current_device())
        made = self._tables.get(device)
        if made is None:
            positions = self.positions
            if positions is None:
                positions = video_positions(self.geometry)
            stream = torch.cuda.current_stream(device)
            with torch.inference_mode(False):  # (an inference tensor could not be saved for a later backward pass)
                table = rotary_table(positions.to(device), self.axes, self.theta, self.scaling)
            stream.synchronize()
            made = self._tables[device] = (table, stream)
        table, stream = made
        here = torch.cuda.current_stream(device)
        if here != stream:
            table.record_stream(here)
        return table

    def __call__(self, q, k):
        q_out, k_out = apply_rotary(q, k, self.table(q.device), layout=self.layout, skip=self.geometry.text_len)
        return (q_out.detach() if q_out.requires_grad and not q.requires_grad else q_out), k_out


def _check(q, k, table, layout, skip, rows):
    device, dtype = q.device, q.dtype
    if device.type != "cuda" or table.device != device or (k is not None and k.device != device) \
            or (rows is not None and rows.device != device):
        _lib.require_gpu(table, rows, q, k)
        raise ValueError("q, k, table and rows must be on one device")
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {LAYOUTS}, got {layout!r}")
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError(f"q and k must be [B, H, L, D], got {', '.join(str(tuple(x.shape)) for x in (q, k) if x is not None)}")
    if dtype not in _lib.DTYPES or (k is not None and k.dtype != dtype):
        raise TypeError("q and k must share one of bf16, fp16 and fp32, got "
                        + ", ".join(str(x.dtype) for x in (q, k) if x is not None))
    B, _, L, D = q.shape
    if k is not None and (k.shape[0], *k.shape[2:]) != (B, L, D):
        raise ValueError(f"shape mismatch q{tuple(q.shape)} k{tuple(k.shape)}")
    if q.numel() > MAX_SIZE < max(q.shape) or (k is not None and k.numel() > MAX_SIZE < max(k.shape)) \
            or (table.dim() and table.shape[0] > MAX_SIZE):
        raise ValueError(f"q, k and table may have at most {MAX_SIZE} tokens and rows")
    if table.dim() != 3 or table.shape[2] != 2 or table.dtype != torch.float32 or not table.is_contiguous():
        raise ValueError("table must be a contiguous fp32 [rows, pairs, 2] tensor (rotary_table)")
    if table.requires_grad:
        raise ValueError("table is not differentiated; pass table.detach()")
    if not 0 < 2 * table.shape[1] <= D or D > 2 * MAX_PAIRS:
        raise ValueError(f"a table of {table.shape[1]} pairs for head dim {D} (at most {2 * MAX_PAIRS})")
    if not 0 <= skip <= L:
        raise ValueError(f"skip={skip} of {L} tokens")
    if rows is None:
        if L - skip > table.shape[0]:
            raise ValueError(f"{L - skip} tokens after {skip} for a table of {table.shape[0]} rows")
    else:
        if skip:
            raise ValueError("skip with rows: mark those tokens with -1 in rows")
        if rows.dtype != torch.int32 or tuple(rows.shape) not in ((L,), (B, L)):
            raise ValueError(f"rows must be int32 [{L}] or [{B}, {L}], got {rows.dtype} {tuple(rows.shape)}")


def _launch(q, q_out, k, k_out, table, layout, skip, rows, inverse):
    B, H, L, D = q.shape
    if B * H * L == 0 or table.shape[0] == 0 or (k is not None and k.shape[1] == 0):
        raise ValueError(f"nothing to turn: q{tuple(q.shape)}, a table of {table.shape[0]} rows")
    if k is not None:
        strides = _lib.i64(*q.stride()[:3], *q_out.stride()[:3], *k.stride()[:3], *k_out.stride()[:3])
    else:
        strides = _lib.i64(*q.stride()[:3], *q_out.stride()[:3], 0, 0, 0, 0, 0, 0)
    with _lib.on(q.device):
        rc = _lib.load().sa_rotary_apply(
            _lib.DTYPES[q.dtype], q.data_ptr(), q_out.data_ptr(), _lib.ptr(k), _lib.ptr(k_out), strides, B, H,
            k.shape[1] if k is not None else 0, L, D, table.data_ptr(), table.shape[0], table.shape[1], _lib.ptr(rows),
            rows.stride(0) if rows is not None and rows.dim() == 2 else 0, int(skip), int(layout == "half"),
            int(inverse), _lib.stream_of(q))
    _lib.check(rc, "sa_rotary_apply")


def _turned(q, k, table, layout, skip, rows, inverse):
    """New tensors of q's and k's (either may be None) memory layouts."""
    if q is not None and k is not None and q.stride(-1) == k.stride(-1) == 1 and q.numel() and k.numel() \
            and table.shape[0]:
        q_out, k_out = torch.empty_like(q), torch.empty_like(k)
        if q_out.stride(-1) == k_out.stride(-1) == 1:
            _launch(q, q_out, k, k_out, table, layout, skip, rows, inverse)
            return q_out, k_out
    xs = [x if x.stride(-1) == 1 else x.contiguous() for x in (q, k) if x is not None]
    outs = [torch.empty_like(x) for x in xs]
    outs = [o if o.stride(-1) == 1 else torch.empty(o.shape, dtype=o.dtype, device=o.device) for o in outs]
    live = [i for i, x in enumerate(xs) if x.numel()]
    if live:
        if table.shape[0] == 0:  # (no token has a row)
            for i in live:
                outs[i].copy_(xs[i])
        else:
            second = (xs[live[1]], outs[live[1]]) if len(live) > 1 else (None, None)
            _launch(xs[live[0]], outs[live[0]], *second, table, layout, skip, rows, inverse)
    it = iter(outs)
    return tuple(next(it) if x is not None else None for x in (q, k))


class _ApplyRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, table, layout, skip, rows, inverse):
        ctx.save_for_backward(table, rows)
        ctx.args = layout, skip, inverse
        ctx.set_materialize_grads(False)
        out = _turned(q, k, table, layout, skip, rows, inverse)
        if k is not None and not ctx.needs_input_grad[1]:
            ctx.mark_non_differentiable(out[1])
        return out

    @staticmethod
    def backward(ctx, dq, dk):
        table, rows = ctx.saved_tensors
        layout, skip, inverse = ctx.args
        if not ctx.needs_input_grad[0]:
            dq = None
        if not ctx.needs_input_grad[1]:
            dk = None
        if dq is None and dk is None:
            return (None,) * 7
        # The transpose turns back; linear, so it is differentiable itself.
        if not torch.is_grad_enabled():
            return (*_turned(dq, dk, table, layout, skip, rows, not inverse), None, None, None, None, None)
        return (*_ApplyRotary.apply(dq, dk, table, layout, skip, rows, not inverse), None, None, None, None, None)


def apply_rotary(q, k, table, layout: str = "interleaved", skip: int = 0, rows: Optional[torch.Tensor] = None,
                 inverse: bool = False):
    """(q, k) turned by the rows of `table`, in new tensors of the same memory layout; differentiable.

    q [B,H,L,D] and k [B,Hk,L,D] (or None) on the GPU, bf16, fp16 or fp32, any strides with a
    contiguous last axis; D at most 256; `table` fp32 [rows, pairs, 2] from `rotary_table`, 2 * pairs
    at most D. Token t takes table row t - skip, and the first `skip` tokens (text) stay as they are;
    or, with `rows` (int32 [L], or [B, L] for sequences at places of their own), row rows[t], and a
    token whose entry lies outside the table stays as it is: permuted layouts, single new tokens,
    padding. `inverse` turns back. Where autograd follows q and not k, it does not follow the turned k either;
    the other way round the turned q counts as followed (detach it, and nobody computes its gradient)."""
    _check(q, k, table, layout, skip, rows)
    rows = rows if rows is None or rows.stride(-1) == 1 else rows.contiguous()
    if _followed(q) or _followed(k):
        return _ApplyRotary.apply(q, k, table, layout, int(skip), rows, bool(inverse))
    return _turned(q, k, table, layout, int(skip), rows, bool(inverse))


def _followed(x) -> bool:
    """Whether autograd has to know of an operation on x (entering it costs a call of one token 4 us of 17).
    Forward-mode tangents are left to autograd, which refuses them."""
    return x is not None and (x.requires_grad and torch.is_grad_enabled()
                              or forward_ad.unpack_dual(x).tangent is not None)


def apply_rotary_(q, k, table, layout: str = "interleaved", skip: int = 0, rows: Optional[torch.Tensor] = None,
                  inverse: bool = False):
    """`apply_rotary` in place (values that do not turn are not touched); returns (q, k). Not for tensors
    that autograd follows, nor for ones whose elements share memory, within one or between the two (views
    of one fused tensor with values of their own may be turned)."""
    _check(q, k, table, layout, skip, rows)
    for x in (q, k):
        if x is None:
            continue
        if x.requires_grad and torch.is_grad_enabled():
            raise ValueError("apply_rotary_ on a tensor that requires gradients; use apply_rotary")
        if x.stride(-1) != 1:
            raise ValueError("apply_rotary_ needs a contiguous last axis")
        if any(s == 0 and n > 1 for s, n in zip(x.stride(), x.shape)):
            raise ValueError("apply_rotary_ on an expanded tensor: its elements share memory")
    if k is not None and k.data_ptr() == q.data_ptr() and q.numel() and k.numel():
        raise ValueError("apply_rotary_ of one tensor as q and k")
    live = [x for x in (q, k) if x is not None and x.numel()]
    if live and table.shape[0]:
        rows = rows if rows is None or rows.stride(-1) == 1 else rows.contiguous()
        second = live[1] if len(live) > 1 else None
        _launch(live[0], live[0], second, second, table, layout, skip, rows, inverse)
        torch.autograd.graph.increment_version(live)
    return q, k
