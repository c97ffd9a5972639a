"""Attention of a few new tokens over cached keys and values, with the score rule of scored_attn.py, on
MI355X: one token of each sequence at a time, or some proposed ones, over a cache of its own and, where a
batch continues one prompt, over a prefix that is held once for all. Beyond the reference, whose attention
has no cache.

Sequence b has lengths[b] cached tokens, the last Ln of them the new ones (their keys and values are
written into the cache before the call); a shared prefix of Lp tokens lies before them. New token i is its
sequence's token t = lengths[b] - Ln + i and sees the keys up to itself: the prefix's, at the distance
d = Lp + t - j, and its own, at d = t - j; with a window those at d < window (of the prefix too, which a
window of `row_ranges` leaves alone). Scores are those of `scored_attention` at these distances. The new
tokens of one call are causal among themselves: there are no frames, nor a block mask.

The lengths stay on the device: a call reads none of them on the host, and its launches depend on the
shapes alone, so that a captured call serves sequences as they grow.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional, Tuple

import torch

from .. import _lib
from .block_sparse_attn_grad import _rows16
from .scored_attn import check_heads, check_rule


class _Call:
    """What calls of one shape share: a description without pointers, and the bytes of its workspace."""

    def __init__(self, dtype, q_shape, k_shape, strides, prefix_shape, sm_scale, cap, window, slopes, table):
        (B, H, Ln, D), (_, Hk, L, _) = q_shape, k_shape
        if not (sm_scale > 0 and math.isfinite(sm_scale)):
            raise ValueError(f"sm_scale {sm_scale} must be positive and finite")
        if not 0 <= window < 2 ** 31:
            raise ValueError(f"window {window}")
        size = dtype.itemsize
        q, k, v, pk, pv = strides
        for name, shape, s in (("k", k_shape, k), ("v", k_shape, v), ("the prefix's k", prefix_shape, pk),
                               ("the prefix's v", prefix_shape, pv)):
            if s is not None and (s[-1] != 1 or any(n > 1 and x * size % 16 for n, x in zip(shape, s[:-1]))):
                raise ValueError(f"{name} must have a contiguous last axis and 16-byte aligned rows (strides {s})")
        self.nothing = 0 in q_shape or L == 0
        if self.nothing:
            return
        Lp = 0 if prefix_shape is None else prefix_shape[1]
        args = self.args = _lib.AttnCached(dtype=_lib.DTYPES[dtype], B=B, H=H, Hk=Hk, Ln=Ln, L=L, Lp=Lp, D=D, window=window,
                                           sm_scale=sm_scale, cap=cap)
        # {b, h, l}, 0 where there is one
        k, v, pk, pv = ([x if n > 1 else 0 for n, x in zip(shape, s)] if s is not None else None
                        for shape, s in ((k_shape, k), (k_shape, v), (prefix_shape, pk), (prefix_shape, pv)))
        args.strides[:12] = (*q[:3], H * Ln * D, Ln * D, D, *k[:3], *v[:3])
        if Lp:
            args.strides[12:] = (0, *pk[:2], 0, *pv[:2])
        if slopes:
            args.slopes = 1
        if table is not None:
            args.table = args.buckets = 1
            args.table_dtype, args.n_buckets, args.radius = _lib.DTYPES[table[0]], table[1], table[2]
        n = ctypes.c_int64(0)
        _lib.check(_lib.load().sa_attn_cached_workspace(args, ctypes.byref(n)), "sa_attn_cached_workspace")
        self.bytes = n.value


_call = functools.lru_cache(maxsize=1024)(_Call)


def _aligned(name, t):
    if t.data_ptr() % 16:
        raise ValueError(f"{name} must have 16-byte aligned rows")


class _NotDifferentiable(torch.autograd.Function):
    """The output of a call on tensors that autograd follows."""

    @staticmethod
    def forward(ctx, out, *tensors):
        return out

    @staticmethod
    def backward(ctx, dout):
        raise NotImplementedError("cached_attention has no backward pass; train with scored_attention")


def cached_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor, sm_scale: float, *,
                     cap: Optional[float] = None, slopes: Optional[torch.Tensor] = None,
                     table: Optional[torch.Tensor] = None, buckets: Optional[torch.Tensor] = None, window: int = 0,
                     prefix: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> torch.Tensor:
    """out [B,H,Ln,D] of the new tokens q [B,H,Ln,D] over the caches k and v [B,Hk,L,D] (H a multiple of Hk)
    with lengths int32 [B] (counted with the new tokens, clamped to [0, L]); bf16, fp16 or fp32 (one type),
    D = 64 or 128. Not differentiable: the backward pass of an output whose inputs autograd follows raises.

    prefix: (k, v) of the shared prefix, each [Hk,Lp,D] or [1,Hk,Lp,D]. The caches and the prefix may have
    any strides with a contiguous last axis and 16-byte aligned rows; they are not copied. Cached rows that no
    new token sees, from lengths[b] on or before a window, are not used, whatever they hold. A new token before
    its sequence's first (lengths[b] < Ln) sees nothing: zeros. cap, slopes, table and buckets as in
    `scored_attention`; window: see above (0: none). The keys are read again for every 32 rows of a key head
    (its query heads times Ln): it is a call for single tokens and a few."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or slopes is not None and slopes.requires_grad or table is not None and table.requires_grad
                                    or prefix is not None and (prefix[0].requires_grad or prefix[1].requires_grad)):
        with torch.no_grad():
            out = cached_attention(q, k, v, lengths, sm_scale, cap=cap, slopes=slopes, table=table, buckets=buckets,
                                   window=window, prefix=prefix)
        tensors = (q, k, v, slopes, table, *(prefix or ()))
        return _NotDifferentiable.apply(out, *(t for t in tensors if t is not None))
    B, H, Hk, Ln, L, D = check_heads(q, k, v)
    cap, slopes, table, buckets, radius = check_rule(q, H, cap, None if slopes is None else slopes.detach(), table, buckets)
    if lengths.device != q.device:
        _lib.require_gpu(lengths)
        raise ValueError("q, k, v and lengths must be on one device")
    if lengths.dtype != torch.int32 or lengths.shape != (B,):
        raise ValueError(f"lengths must be int32 [{B}], got {lengths.dtype} {tuple(lengths.shape)}")
    pk = pv = None
    if prefix is not None:
        pk, pv = (t[0] if t.dim() == 4 and t.shape[0] == 1 else t for t in prefix)
        for t in (pk, pv):
            if t.device != q.device:
                _lib.require_gpu(t)
                raise ValueError("q, k, v and the prefix must be on one device")
            if t.dtype != q.dtype:
                raise TypeError(f"the prefix must be {q.dtype}, got {t.dtype}")
            if t.dim() != 3 or t.shape != pk.shape or t.shape[0] != Hk or t.shape[2] != D:
                raise ValueError(f"the prefix must be two [{Hk}, Lp, {D}], got {tuple(pk.shape)} and {tuple(pv.shape)}")
        if pk.shape[1]:
            _aligned("the prefix's k", pk)
            _aligned("the prefix's v", pv)
        else:
            pk = pv = None
    _aligned("k", k)
    _aligned("v", v)
    q = _rows16(q)
    call = _call(q.dtype, q.shape, k.shape, (q.stride(), k.stride(), v.stride(), None if pk is None else pk.stride(),
                                             None if pv is None else pv.stride()),
                 None if pk is None else pk.shape, float(sm_scale), cap, int(window), slopes is not None,
                 None if table is None else (table.dtype, table.shape[0], radius))
    out = torch.empty((B, H, Ln, D), dtype=q.dtype, device=q.device)
    if call.nothing:  # no sequence has a token
        return out.zero_()
    args = _lib.AttnCached.from_buffer_copy(call.args)
    args.q, args.out, args.k, args.v = q.data_ptr(), out.data_ptr(), k.data_ptr(), v.data_ptr()
    if pk is not None:
        args.prefix_k, args.prefix_v = pk.data_ptr(), pv.data_ptr()
    if not lengths.is_contiguous():
        lengths = lengths.contiguous()
    args.lengths = lengths.data_ptr()
    if slopes is not None:
        args.slopes = slopes.data_ptr()
    if table is not None:
        args.table, args.buckets = table.data_ptr(), buckets.data_ptr()
    if call.bytes:
        ws = torch.empty(call.bytes, dtype=torch.uint8, device=q.device)
        args.workspace, args.workspace_bytes = ws.data_ptr(), call.bytes
    with _lib.on(q.device):
        rc = _lib.load().sa_attn_cached_fwd(args, _lib.stream_of(q))
    if rc:
        _lib.check(rc, "sa_attn_cached_fwd")
    return out
