"""Attention of a few new tokens over cached keys and values, with the score rule of scored_attn.py, on
MI355X: one token of each sequence at a time, or some proposed ones, over a cache of its own and, where a
batch continues one prompt, over a prefix that is held once for all. Beyond the reference, whose attention
has no cache.

Sequence b has lengths[b] cached tokens, the last Ln of them the new ones (their keys and values are
written into the cache before the call); a shared prefix of Lp tokens lies before them. New token i is its
sequence's token t = lengths[b] - Ln + i and sees the keys up to itself: the prefix's, at the distance
d = Lp + t - j, and its own, at d = t - j; with a window those at d < window. Scores are those of
`scored_attention` at these distances.

The lengths stay on the device: a call reads none of them on the host, and its launches depend on the
shapes alone, so that a captured call serves sequences as they grow.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from .. import _lib
from .block_sparse_attn_grad import _rows16
from .scored_attn import check_heads, check_rule


def _check_rows(name, t):
    size = t.element_size()
    if t.stride(-1) != 1 or any(n > 1 and s * size % 16 for n, s in zip(t.shape, t.stride()[:-1])) or t.data_ptr() % 16:
        raise ValueError(f"{name} must have a contiguous last axis and 16-byte aligned rows (strides {tuple(t.stride())})")


def _set(call, at, t):
    """Strides {b, h, l} of [B, H, L, D], or of [H, L, D] (b unused); 0 where there is one."""
    strides = [s if n > 1 else 0 for n, s in zip(t.shape, t.stride())]
    call.strides[at:at + 3] = strides[:3] if t.dim() == 4 else (0, *strides[:2])


@torch.no_grad()
def cached_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor, sm_scale: float, *,
                     cap: Optional[float] = None, slopes: Optional[torch.Tensor] = None,
                     table: Optional[torch.Tensor] = None, buckets: Optional[torch.Tensor] = None, window: int = 0,
                     prefix: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> torch.Tensor:
    """out [B,H,Ln,D] of the new tokens q [B,H,Ln,D] over the caches k and v [B,Hk,L,D] (H a multiple of Hk)
    with lengths int32 [B] (counted with the new tokens, clamped to [0, L]); bf16, fp16 or fp32 (one type),
    D = 64 or 128. No autograd.

    prefix: (k, v) of the shared prefix, each [Hk,Lp,D] or [1,Hk,Lp,D]. The caches and the prefix may have
    any strides with a contiguous last axis and 16-byte aligned rows; they are not copied. Cached rows from
    lengths[b] on are not used, whatever they hold. A new token before its sequence's first (lengths[b] <
    Ln) sees nothing: zeros. cap, slopes, table and buckets as in `scored_attention`; window: see above
    (0: none)."""
    B, H, Hk, Ln, L, D = check_heads(q, k, v)
    cap, slopes, table, buckets, radius = check_rule(q, H, cap, None if slopes is None else slopes.detach(), table, buckets)
    if lengths.device != q.device:
        _lib.require_gpu(lengths)
        raise ValueError("q, k, v and lengths must be on one device")
    if lengths.dtype != torch.int32 or lengths.shape != (B,):
        raise ValueError(f"lengths must be int32 [{B}], got {lengths.dtype} {tuple(lengths.shape)}")
    if not (sm_scale > 0 and math.isfinite(sm_scale)):
        raise ValueError(f"sm_scale {sm_scale} must be positive and finite")
    window = int(window)
    if not 0 <= window < 2 ** 31:
        raise ValueError(f"window {window}")
    _check_rows("k", k)
    _check_rows("v", v)
    Lp = 0
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
        Lp = pk.shape[1]
    out = torch.empty((B, H, Ln, D), dtype=q.dtype, device=q.device)
    if out.numel() == 0:
        return out
    if L == 0:  # no sequence has a token
        return out.zero_()
    q = _rows16(q)
    call = _lib.AttnCached(dtype=_lib.DTYPES[q.dtype], B=B, H=H, Hk=Hk, Ln=Ln, L=L, Lp=Lp, D=D, window=window, radius=radius,
                           sm_scale=sm_scale, cap=cap)
    call.q, call.out, call.k, call.v = q.data_ptr(), out.data_ptr(), k.data_ptr(), v.data_ptr()
    for i, t in enumerate((q, out, k, v)):
        _set(call, 3 * i, t)
    if Lp:
        _check_rows("the prefix's k", pk)
        _check_rows("the prefix's v", pv)
        call.prefix_k, call.prefix_v = pk.data_ptr(), pv.data_ptr()
        _set(call, 12, pk)
        _set(call, 15, pv)
    lengths = lengths.contiguous()
    call.lengths = lengths.data_ptr()
    if slopes is not None:
        call.slopes = slopes.data_ptr()
    if table is not None:
        call.table, call.buckets = table.data_ptr(), buckets.data_ptr()
        call.table_dtype, call.n_buckets = _lib.DTYPES[table.dtype], table.shape[0]
    n = ctypes.c_int64(0)
    _lib.check(_lib.load().sa_attn_cached_workspace(call, ctypes.byref(n)), "sa_attn_cached_workspace")
    if n.value:
        ws = torch.empty(n.value, dtype=torch.uint8, device=q.device)
        call.workspace, call.workspace_bytes = ws.data_ptr(), n.value
    with _lib.on(q.device):
        rc = _lib.load().sa_attn_cached_fwd(call, _lib.stream_of(q))
    _lib.check(rc, "sa_attn_cached_fwd")
    return out
