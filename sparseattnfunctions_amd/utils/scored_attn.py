"""Attention whose scores follow a rule besides the dot product, differentiable, on MI355X: scores
capped by a tanh, less a slope times the distance, plus a learned bias by buckets of the distance, over
documents, prefixes, causal rows and frames, windows and blocks of a mask. Beyond the reference, whose
attention takes a block mask (special_attentions/utils/block_sparse_attn_kernel.py:211-265).

  * `scored_attention(q, k, v, sm_scale, ...)`: the call, differentiable in q, k, v and the bias table;
  * `scored_attention_forward` and `scored_attention_backward`: its two halves without autograd, e.g. for
    a step captured into a HIP graph;
  * `row_ranges`: which rows see each key, from the lengths of the documents that a sequence packs;
  * `distance_buckets`: the buckets of a learned bias.

With d = i + q_start - j the distance of query row i from key j of query head h, whose keys are those of
key head h // (H // Hk), the score is

  s = sm_scale q.k;  cap: s = cap tanh(s / cap);  slopes: s -= slopes[h] |d|;
  table: s += table[buckets[clamp(d, -R, R) + R], h], 2 R + 1 = len(buckets)

and row i sees key j where ranges[b, j, 0] <= i < ranges[b, j, 1] and block_mask[b, h, i // 64, j // 64].
A row that sees no key has a zero output and zero gradients, a key that no row sees zero gradients.

The backward pass recomputes the probabilities block by block (`sa_attn_scored_bwd`); between the two a
call holds q, k, v, out, a float per row (three with slopes) and its lists of blocks (eight bytes for each pair of 64-token
blocks of a sequence, with a block mask of a head). Blocks of which no pair is seen are not read. Gradients
of a 16-bit call round P and dS to its type; sums are fp32 in a fixed order, so that a step repeats bit
for bit. In fp16, dS has the range of the type: scale the loss as usual.

Rows (of q and, in the backward pass, of the output's gradient), keys and values of 64 x 64 blocks that hold
a visible pair (without a mask and up to 256 rows and keys, all of them) enter the products whole: they have
to be finite, also where a mask hides them, as do the slopes and the table; but a table's value of -inf, or
below -2.3e38 (the lowest of bf16 and fp32), hides its pairs. The calls are differentiable once; ranges, the
mask and the slopes are not differentiated.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional

import torch

from .. import _lib
from .block_sparse_attn_grad import _rows16
from .block_sparse_attn_kernel import BLOCK

MOST_RADIUS = 1024  # distances that a bias tells apart
_KEYS, _TABLE = 1, 2  # SA_SCORED_KEYS, SA_SCORED_TABLE


def distance_buckets(n_buckets: int, radius: int, bidirectional: bool = True, device="cuda") -> torch.Tensor:
    """Buckets int32 [2 radius + 1] of the distances -radius .. radius (i - j: positive for keys before the
    row) for `scored_attention`'s table; distances past the radius share the last one's.

    Of the buckets of a side (unless bidirectional there is one, and keys behind the row have bucket 0)
    the first half hold one distance each, the others grow in proportion to it, up to the radius. Bidirectional,
    bucket 0 is distance 0 and each side has (n_buckets - 1) // 2: the last one of an even number is not used."""
    n_buckets, radius = int(n_buckets), int(radius)
    if not 0 <= radius <= MOST_RADIUS:
        raise ValueError(f"radius {radius} (0 to {MOST_RADIUS})")
    if n_buckets < 1:
        raise ValueError(f"n_buckets {n_buckets}")
    side = (n_buckets - 1) // 2 if bidirectional else n_buckets - 1
    exact = max(1, side // 2)
    places = []
    for d in range(-radius, radius + 1):
        a = abs(d) if bidirectional else max(d, 0)
        if a > exact:
            a = exact + int((side - exact) * math.log(a / exact) / math.log(radius / exact)) + 1
        a = min(side, a)
        places.append(a if d >= 0 or not bidirectional or a == 0 else side + a)
    return torch.tensor(places, dtype=torch.int32, device=device)


_INTEGERS = (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8)


def _int32(t, most):
    """t as contiguous int32 (64-bit numbers no larger than `most`, above which they all mean the same)."""
    if t.dtype != torch.int32:
        t = (t.clamp(-1, most) if t.dtype == torch.int64 else t).to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


def row_ranges(lengths: torch.Tensor, L: int, causal: bool = True, prefix: Optional[torch.Tensor] = None, frame: int = 1,
               window: int = 0) -> torch.Tensor:
    """ranges int32 [B, L, 2] of B sequences that pack documents of `lengths` (integers [B, n], or [n] for
    one sequence) one after the other from token 0, made on the GPU (`sa_row_ranges`). Rows see the keys of
    their own document; tokens behind the last document are seen by no row, and see none.

    Of a document, its first prefix[b, i] tokens (none by default) are seen by all its rows. Of the others
    a causal row sees itself and those before it, with `frame` > 1 those of its own and earlier groups of
    `frame` tokens, counted from behind the prefix; a row that is not causal sees all. With a window a key
    outside the prefix is seen by no row that lies `window` tokens or more behind it (or, not causal,
    before it)."""
    device = lengths.device
    if device.type != "cuda":
        _lib.require_gpu(lengths)
    if lengths.dim() == 1:
        lengths = lengths[None]
    if lengths.dim() != 2 or lengths.shape[1] == 0 or lengths.dtype not in _INTEGERS:
        raise ValueError(f"lengths must be integers [B, n], got {lengths.dtype} {tuple(lengths.shape)}")
    B, n = lengths.shape
    L, frame, window = int(L), int(frame), int(window)
    if L < 0:
        raise ValueError(f"L={L}")
    if max(L, frame, window) >= 2 ** 31:
        raise ValueError(f"L={L} frame={frame} window={window}: sizes of 32 bits")
    if prefix is not None:
        if prefix.device != device:
            _lib.require_gpu(prefix)
            raise ValueError("lengths and prefix must be on one device")
        if prefix.dtype not in _INTEGERS:
            raise ValueError(f"prefix must be integers, got {prefix.dtype}")
        if prefix.shape != (B, n):
            if prefix.dim() > 2 or any(x not in (1, y) for x, y in zip(prefix.shape[::-1], (n, B))):
                raise ValueError(f"prefix must be [{B}, {n}], or of one sequence or number, got {tuple(prefix.shape)}")
            prefix = prefix.expand(B, n)
        prefix = _int32(prefix, L)
    lengths = _int32(lengths, L)
    out = torch.empty((B, L, 2), dtype=torch.int32, device=device)
    if B == 0 or L == 0:
        return out
    with _lib.on(device):
        rc = _lib.load().sa_row_ranges(lengths.data_ptr(), None if prefix is None else prefix.data_ptr(), B, n, L,
                                       1 if causal else 0, frame, window, out.data_ptr(), _lib.stream_of(out))
    _lib.check(rc, "sa_row_ranges")
    return out


def check_rule(q, H: int, cap, slopes, table, buckets):
    """The checked parameters of a score rule: (cap, slopes, table, buckets, radius)."""
    if cap is not None and not (cap > 0 and math.isfinite(cap)):
        raise ValueError(f"cap {cap} must be positive and finite")
    if slopes is not None:
        if slopes.requires_grad:
            raise ValueError("slopes are not differentiated; pass slopes.detach()")
        if slopes.dtype != torch.float32 or slopes.shape != (H,):
            raise ValueError(f"slopes must be fp32 [{H}], got {slopes.dtype} {tuple(slopes.shape)}")
        slopes = slopes.contiguous()
    if (table is None) != (buckets is None):
        raise ValueError("a table needs buckets, and buckets a table")
    radius = 0
    if table is not None:
        if table.dtype not in _lib.DTYPES:
            raise TypeError(f"table must be bf16, fp16 or fp32, got {table.dtype}")
        if table.dim() != 2 or table.shape[1] != H or table.shape[0] == 0:
            raise ValueError(f"table must be [buckets, {H}], got {tuple(table.shape)}")
        if buckets.dtype != torch.int32 or buckets.dim() != 1 or buckets.numel() % 2 == 0:
            raise ValueError("buckets must be int32 [2 radius + 1]")
        radius = buckets.numel() // 2
        if radius > MOST_RADIUS:
            raise NotImplementedError(f"distances up to {radius} told apart (at most {MOST_RADIUS})")
        table, buckets = table.contiguous(), buckets.contiguous()
    device = q.device
    for t in (slopes, table, buckets):
        if t is not None and t.device != device:
            _lib.require_gpu(t)
            raise ValueError("q, k, v and the rule's tensors must be on one device")
    return 0.0 if cap is None else float(cap), slopes, table, buckets, radius


def check_heads(q, k, v):
    """(B, H, Hk, Lq, Lk, D) of q [B,H,Lq,D] and k, v [B,Hk,Lk,D]."""
    device = q.device
    if device.type != "cuda" or k.device != device or v.device != device:
        _lib.require_gpu(q, k, v)
        raise ValueError("q, k and v must be on one device")
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"q, k, v must be [B, H, L, D], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if q.dtype not in _lib.DTYPES or not q.dtype == k.dtype == v.dtype:
        raise TypeError(f"q, k, v must share one of bf16, fp16 and fp32, got {q.dtype}, {k.dtype}, {v.dtype}")
    B, H, Lq, D = q.shape
    Hk, Lk = k.shape[1:3]
    if k.shape != (B, Hk, Lk, D) or v.shape != k.shape:
        raise ValueError(f"shape mismatch q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}")
    if (H % Hk if Hk else H) != 0:
        raise ValueError(f"{H} query heads over {Hk} key heads")
    if D not in (64, 128):
        raise NotImplementedError(f"head_dim {D} (64 or 128)")
    return B, H, Hk, Lq, Lk, D


class ScoredState:
    """What `scored_attention_forward` keeps for `scored_attention_backward`: q, k, v, out, one buffer (the
    plan, the rows' log2-sum-exp2 and what out's rounding leaves), ranges, slopes, table and buckets, and the
    call's description."""

    __slots__ = ("tensors", "call", "args")

    def __init__(self, tensors, call, args):
        self.tensors, self.call, self.args = tensors, call, args


_ORDER = ("q", "k", "v", "out", "dout", "dq", "dk", "dv")  # of AttnScored.strides


class _Call:
    """What calls of one shape share: a description without pointers, and the sizes of their buffers."""

    def __init__(self, dtype, q_shape, k_shape, strides, sm_scale, cap, q_start, slopes, table, ranges, mask, follow):
        (B, H, Lq, D), (_, Hk, Lk, _) = q_shape, k_shape
        args = self.args = _lib.AttnScored(dtype=_lib.DTYPES[dtype], B=B, H=H, Hk=Hk, Lq=Lq, Lk=Lk, D=D, q_start=q_start,
                                           sm_scale=sm_scale, cap=cap, follow=follow or 0)
        self.strides = strides  # of q, k and v; the others' are contiguous, dout's are set where they are not
        of_q, of_k = (H * Lq * D, Lq * D, D), (Hk * Lk * D, Lk * D, D)
        args.strides[:] = (*(x for t in strides for x in t[:3]), *of_q, *of_q, *of_q, *of_k, *of_k)
        if slopes:
            args.slopes = 1  # (the sizes depend on what there is; the pointers follow)
        if table is not None:
            args.table = args.buckets = 1
            args.table_dtype, args.n_buckets, args.radius = _lib.DTYPES[table[0]], table[1], table[2]
        if ranges is not None:
            args.ranges, args.ranges_stride = 1, ranges
        if mask is not None:
            args.mask = 1
            args.mask_strides[:] = mask
        n = (ctypes.c_int64 * 3)()
        _lib.check(_lib.load().sa_attn_scored_sizes(args, n), "sa_attn_scored_sizes")
        args.plan_bytes, self.fwd_bytes, self.bwd_bytes = n[0], n[1], n[2]
        self.out, self.grads = (B, H, Lq, D), ((B, H, Lq, D), (B, Hk, Lk, D), (B, Hk, Lk, D))
        self.contiguous = (*of_q, 1)
        # The buffer: the plan (a multiple of 256 bytes), the sums, the rest of out.
        self.lse_at = n[0]
        rows = B * H * (-(-Lq // BLOCK)) * BLOCK
        self.lo_at = self.lse_at + 4 * rows if follow is not None and dtype != torch.float32 else None
        self.buffer_bytes = self.lse_at + 4 * rows + (0 if self.lo_at is None else 2 * B * H * Lq * D)


_call = functools.lru_cache(maxsize=1024)(_Call)


def _point(call, args, q, k, v, out, buffer, ranges, slopes, table, buckets):
    args.q, args.k, args.v, args.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    args.plan = at = buffer.data_ptr()
    args.lse = at + call.lse_at
    if call.lo_at is not None:
        args.out_lo = at + call.lo_at
    if ranges is not None:
        args.ranges = ranges.data_ptr()
    if slopes is not None:
        args.slopes = slopes.data_ptr()
    if table is not None:
        args.table, args.buckets = table.data_ptr(), buckets.data_ptr()


def _check_ranges(ranges, q, B, Lk):
    if ranges is None:
        return None
    if ranges.device != q.device:
        _lib.require_gpu(ranges)
        raise ValueError("q, k, v and ranges must be on one device")
    if ranges.dtype != torch.int32 or ranges.dim() not in (2, 3) or ranges.shape[-2:] != (Lk, 2) \
            or (ranges.dim() == 3 and ranges.shape[0] not in (1, B)):
        raise ValueError(f"ranges must be int32 [{B}, {Lk}, 2], got {ranges.dtype} {tuple(ranges.shape)}")
    return _pairs(ranges if ranges.dim() == 3 else ranges[None]).expand(B, -1, -1)


def _pairs(ranges):
    """ranges [b, Lk, 2] as the kernels read them: a sequence's pairs one after the other, 8-byte aligned."""
    sb, sl, s1 = ranges.stride()
    if s1 != 1 or (sl != 2 and ranges.shape[1] > 1) or sb % 2 or ranges.data_ptr() % 8:
        ranges = ranges.clone(memory_format=torch.contiguous_format)
    return ranges


def _check_mask(mask, q, B, H, nqb, nkb):
    if mask is None:
        return None
    if mask.device != q.device:
        _lib.require_gpu(mask)
        raise ValueError("q, k, v and the block mask must be on one device")
    if mask.dim() != 4:
        raise ValueError(f"block mask must be 4-D [B,H,nqb,nkb], got {tuple(mask.shape)}")
    if mask.shape[0] not in (1, B) or mask.shape[1] not in (1, H):
        raise ValueError(f"block mask {tuple(mask.shape)} of other sequences or heads than ({B}, {H})")
    if mask.shape[2] < nqb or mask.shape[3] < nkb:
        raise ValueError(f"block mask {tuple(mask.shape)} smaller than the block grid ({nqb}, {nkb})")
    if mask.dtype != torch.bool:
        mask = mask != 0
    return mask.expand(B, H, -1, -1)


def _check(q, k, v, cap, slopes, table, buckets, ranges, block_mask, q_start):
    B, H, Hk, Lq, Lk, D = check_heads(q, k, v)
    cap, slopes, table, buckets, _ = check_rule(q, H, cap, slopes, table, buckets)
    if not -2 ** 29 < q_start < 2 ** 29:
        raise ValueError(f"q_start {q_start}")
    ranges = _check_ranges(ranges, q, B, Lk)
    block_mask = _check_mask(block_mask, q, B, H, -(-Lq // BLOCK), -(-Lk // BLOCK))
    return cap, slopes, table, buckets, ranges, block_mask


def _forward(q, k, v, sm_scale, cap, slopes, table, buckets, ranges, mask, q_start, follow):
    """(out, state) on checked arguments. follow: _KEYS and _TABLE, or None: no gradient."""
    q, k, v = _rows16(q), _rows16(k), _rows16(v)
    device = q.device
    call = _call(q.dtype, q.shape, k.shape, (q.stride(), k.stride(), v.stride()), sm_scale, cap, q_start, slopes is not None,
                 None if table is None else (table.dtype, table.shape[0], buckets.numel() // 2),
                 None if ranges is None else ranges.stride(0) // 2, None if mask is None else mask.stride(), follow)
    out = torch.empty(call.out, dtype=q.dtype, device=device)
    buffer = torch.empty(call.buffer_bytes, dtype=torch.uint8, device=device)
    args = _lib.AttnScored.from_buffer_copy(call.args)
    _point(call, args, q, k, v, out, buffer, ranges, slopes, table, buckets)
    if mask is not None:
        args.mask = mask.data_ptr()
    if call.fwd_bytes:
        ws = torch.empty(call.fwd_bytes, dtype=torch.uint8, device=device)
        args.workspace, args.workspace_bytes = ws.data_ptr(), call.fwd_bytes
    with _lib.on(device):
        rc = _lib.load().sa_attn_scored_fwd(args, _lib.stream_of(q))
    if rc:
        _lib.check(rc, "sa_attn_scored_fwd")
    return out, ScoredState((q, k, v, out, buffer, ranges, slopes, table, buckets), call, args)


def _backward(dout, state, needs):
    """(dq, dk, dv, dtable), None where not needed."""
    q, k, v, out, buffer, ranges, slopes, table, buckets = state.tensors
    call = state.call
    args = _lib.AttnScored.from_buffer_copy(state.args)  # (this may run twice, or in two threads)
    if (q.stride(), k.stride(), v.stride()) != call.strides or out.stride() != call.contiguous \
            or not all(t.data_ptr() % 16 == 0 for t in (q, k, v, out)):  # (hooks on saved tensors have moved them)
        q, k, v, out = _rows16(q), _rows16(k), _rows16(v), out.contiguous()
        args.strides[:9] = (*q.stride()[:3], *k.stride()[:3], *v.stride()[:3])
    if slopes is not None:
        slopes = slopes.contiguous()
    if table is not None:
        table, buckets = table.contiguous(), buckets.contiguous()
    if ranges is not None:
        ranges = _pairs(ranges)
        args.ranges_stride = ranges.stride(0) // 2
    _point(call, args, q, k, v, out, buffer, ranges, slopes, table, buckets)
    if dout.stride() != call.contiguous or dout.data_ptr() % 16:
        dout = _rows16(dout)
        if (dout.shape[2] + BLOCK) * dout.stride(2) * dout.element_size() >= 1 << 30:  # (rows far apart: 32-bit offsets)
            dout = dout.contiguous()
        args.strides[12:15] = dout.stride()[:3]
    args.dout = dout.data_ptr()
    device, dtype = q.device, q.dtype
    grads = [None] * 4
    for i, name in enumerate(("dq", "dk", "dv")):
        if needs[i]:
            grads[i] = g = torch.empty(call.grads[i], dtype=dtype, device=device)
            setattr(args, name, g.data_ptr())
    if needs[3]:
        grads[3] = torch.empty_like(table)
        args.dtable = grads[3].data_ptr()
    ws = torch.empty(call.bwd_bytes, dtype=torch.uint8, device=device)
    args.workspace, args.workspace_bytes = ws.data_ptr(), call.bwd_bytes
    with _lib.on(device):
        rc = _lib.load().sa_attn_scored_bwd(args, _lib.stream_of(q))
    if rc:
        _lib.check(rc, "sa_attn_scored_bwd")
    return grads


def scored_attention_forward(q, k, v, sm_scale: float, *, cap: Optional[float] = None, slopes=None, table=None, buckets=None,
                             ranges=None, block_mask=None, q_start: int = 0):
    """(out, state): `scored_attention` without autograd, and what `scored_attention_backward` needs of it."""
    checked = _check(q, k, v, cap, slopes, table, buckets, ranges, block_mask, int(q_start))
    if not (sm_scale > 0 and math.isfinite(sm_scale)):
        raise ValueError(f"sm_scale {sm_scale} must be positive and finite")
    if q.numel() == 0 or k.numel() == 0:
        raise ValueError(f"no query or no key: q{tuple(q.shape)} k{tuple(k.shape)}")
    with torch.no_grad():
        return _forward(q, k, v, float(sm_scale), *checked, int(q_start), _KEYS | (0 if table is None else _TABLE))


def scored_attention_backward(dout, state: ScoredState, needs=(True, True, True, True)):
    """(dq, dk, dv, dtable) for the gradient dout of `scored_attention_forward`'s out, whose tensors must be as
    they were; None where `needs` is false, and for dtable without a table."""
    q, table = state.tensors[0], state.tensors[7]
    _lib.require_gpu(dout)
    if dout.shape != q.shape or dout.dtype != q.dtype or dout.device != q.device:
        raise ValueError(f"dout must be like q: {tuple(q.shape)} {q.dtype}, got {tuple(dout.shape)} {dout.dtype}")
    with torch.no_grad():
        return tuple(_backward(dout, state, (*needs[:3], needs[3] and table is not None)))


class _ScoredAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, sm_scale, cap, slopes, buckets, ranges, mask, q_start, follow):
        out, state = _forward(q, k, v, sm_scale, cap, slopes, table, buckets, ranges, mask, q_start, follow)
        ctx.call, ctx.args = state.call, state.args
        ctx.save_for_backward(*state.tensors)
        return out

    @staticmethod
    def backward(ctx, dout):
        if torch.is_grad_enabled():
            raise RuntimeError("scored attention is differentiable once (create_graph=True is not supported)")
        grads = _backward(dout, ScoredState(ctx.saved_tensors, ctx.call, ctx.args), ctx.needs_input_grad)
        return (*grads, None, None, None, None, None, None, None, None)


class _Nothing(torch.autograd.Function):
    """The output where there is no query or no key: zeros, with zero gradients."""

    @staticmethod
    def forward(ctx, q, k, v, table):
        ctx.save_for_backward(q, k, v, table)
        return torch.zeros(q.shape, dtype=q.dtype, device=q.device)

    @staticmethod
    def backward(ctx, dout):
        return tuple(None if t is None else torch.zeros_like(t) for t in ctx.saved_tensors)


def scored_attention(q, k, v, sm_scale: float, *, cap: Optional[float] = None, slopes: Optional[torch.Tensor] = None,
                     table: Optional[torch.Tensor] = None, buckets: Optional[torch.Tensor] = None,
                     ranges: Optional[torch.Tensor] = None, block_mask: Optional[torch.Tensor] = None,
                     q_start: int = 0) -> torch.Tensor:
    """softmax attention under the score rule of this module, differentiable (once) in q, k, v and table.

    q [B,H,Lq,D], k and v [B,Hk,Lk,D] (H a multiple of Hk) on the GPU, bf16, fp16 or fp32 (one type), D = 64
    or 128, any strides (tensors whose rows are not 16-byte aligned are copied). cap: a number between 1e-30 and
    1e30; slopes: fp32 [H]; table: [n, H] of any of the three types, with buckets int32 [2 R + 1] (R up to 1024;
    entries outside [0, n) count as the nearest one); ranges: int32 [B or 1, Lk, 2] (`row_ranges`, or a caller's
    own); block_mask: bool or integer [B or 1, H or 1, >= ceil(Lq / 64), >= ceil(Lk / 64)]; q_start: the position
    of row 0 where key 0 has position 0, for the distances alone (ranges count rows from 0).

    The tensors must stay as they are until the backward pass has run. A call captured into a HIP graph needs
    leaves that no eager graph holds (autograd ties a leaf's gradient to the stream of its first use)."""
    cap, slopes, table, buckets, ranges, block_mask = _check(q, k, v, cap, slopes, table, buckets, ranges, block_mask,
                                                             int(q_start))
    if not (sm_scale > 0 and math.isfinite(sm_scale)):
        raise ValueError(f"sm_scale {sm_scale} must be positive and finite")
    if q.numel() == 0 or k.numel() == 0:
        return _Nothing.apply(q, k, v, table)
    follow = None
    if torch.is_grad_enabled():
        of_keys, of_table = k.requires_grad or v.requires_grad, table is not None and table.requires_grad
        if q.requires_grad or of_keys or of_table:
            follow = (_KEYS if of_keys else 0) | (_TABLE if of_table else 0)
            # (what a validation pass made in inference mode could not be saved)
            if slopes is not None and slopes.is_inference():
                slopes = slopes.clone()
            if buckets is not None and buckets.is_inference():
                buckets = buckets.clone()
            if ranges is not None and ranges.is_inference():
                ranges = ranges.clone()
    return _ScoredAttention.apply(q, k, v, table, float(sm_scale), cap, slopes, buckets, ranges, block_mask, int(q_start),
                                  follow)
