"""Block-sparse attention that can be trained: the forward pass of block_sparse_attn_kernel.py with
its gradients, on MI355X.

The reference's autograd function raises NotImplementedError in its backward pass
(special_attentions/utils/block_sparse_attn_kernel.py:278-281), and `block_sparse_triton_fn` here
does as well. Training code calls this module instead:

  * `block_sparse_train_fn(q, k, v, block_sparse_mask, sm_scale)`: the mask-level call, differentiable
    in q, k and v;
  * `block_sparse_attention_train(q, k, v, kv, sm_scale)`: the same on block lists (`KVList`), as the
    processors' mask builders give them;
  * `block_sparse_attention_lse` and `block_sparse_attention_backward`: its two halves without
    autograd, e.g. for a step captured into a HIP graph.

The forward pass is the kernel of `block_sparse_attention` with bf16 (fp16, fp32) scores and also
stores each row's log2-sum-exp2; the backward pass recomputes the probabilities from it, block by
block, and keeps nothing of the size of the attention map (`sa_block_sparse_bwd`). Gradients of a
16-bit call round P and dS to its type, sums are fp32 in a fixed order, so that a step repeats bit for
bit. In fp16, dS has the range of the type: scale the loss as usual. A query row without a key (an
empty list, or keys all biased to -inf) has a zero output and zero gradients; a key block in no list
has zero gradients. The mask, the lists and key_bias are not differentiated.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .._kv import KVList, kv_list_from_mask
from .block_sparse_attn_kernel import (BLOCK, F32_TERMS_BLOCKS, cell_kv_list, f32_terms_workspace, shares_text_rows,
                                       split_parts, split_workspace_bytes, work_order)

_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """t with a contiguous last axis and 16-byte aligned rows (a copy where it has not)."""
    per16 = 16 // t.element_size()
    if t.stride(-1) != 1 or t.data_ptr() % 16 or any(s < 0 or s % per16 for s in t.stride()[:-1]):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _check_inputs(q, k, v, kv: KVList, key_bias):
    _lib.require_gpu(q, k, v, key_bias, kv.idx, kv.cnt)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"q, k, v must be [B, H, L, D], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if q.dtype not in _TYPES or not q.dtype == k.dtype == v.dtype:
        raise TypeError(f"q, k, v must share one of bf16, fp16 and fp32, got {q.dtype}, {k.dtype}, {v.dtype}")
    B, H, Lq, D = q.shape
    Lk = k.shape[2]
    if k.shape != (B, H, Lk, D) or v.shape != (B, H, Lk, D):
        raise ValueError(f"shape mismatch q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}")
    if D not in (64, 128):
        raise NotImplementedError(f"head_dim {D} (64 or 128)")
    if any(x is not None and x.device != q.device for x in (k, v, key_bias, kv.idx, kv.cnt)):
        raise ValueError("q, k, v, the lists and key_bias must be on one device")
    nqb, nkb = math.ceil(Lq / BLOCK), math.ceil(Lk / BLOCK)
    if (kv.B, kv.H, kv.nqb, kv.nkb) != (B, H, nqb, nkb) or kv.rows != B * H * nqb:
        raise ValueError(f"kv lists of {kv.B} x {kv.H} x {kv.nqb} x {kv.nkb} blocks, expected {B} x {H} x {nqb} x {nkb}")
    for t in (kv.idx, kv.cnt):
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError("kv lists must be contiguous int32 tensors")
    if key_bias is not None:
        if q.dtype == torch.float32:
            raise NotImplementedError("fp32 inputs: plain block lists only (no key_bias)")
        if key_bias.requires_grad:
            raise ValueError("key_bias is not differentiated; pass key_bias.detach()")
        if key_bias.dtype != torch.float32 or key_bias.shape[-1] != Lk or key_bias.stride(-1) != 1:
            raise ValueError("key_bias must be fp32 [B,H,Lk] with a contiguous key axis")
        key_bias = key_bias.expand(B, H, Lk)
    return key_bias


def _bias_args(key_bias):
    if key_bias is None:
        return None, None
    return key_bias.data_ptr(), _lib.i64(key_bias.stride(0), key_bias.stride(1))


def _forward(q, k, v, kv: KVList, sm_scale: float, key_bias, n_text_blocks: int):
    """(out, lse) of checked, aligned inputs; key_bias expanded."""
    B, H, Lq, D = q.shape
    Lk = k.shape[2]
    nqb = kv.nqb
    out = torch.empty(B, H, Lq, D, dtype=q.dtype, device=q.device)
    lse = torch.empty(B, H, nqb * BLOCK, dtype=torch.float32, device=q.device)
    # The launch variants of block_sparse_attention: key-range parts for few blocks over long lists,
    # else a work order; fp32 on split operands where it takes them.
    parts, ws, order = 1, None, None
    if q.dtype == torch.float32:
        if nqb >= F32_TERMS_BLOCKS:
            ws = f32_terms_workspace(B, H, Lk, D, q.device)
    elif key_bias is None:
        parts = split_parts(B * H * nqb, kv.max_cnt, D)
        if parts > 1:
            ws = torch.empty(split_workspace_bytes(B * H * nqb, D, parts), dtype=torch.uint8, device=q.device)
    if parts == 1:
        # (lists of unknown length count as short beside the text rows')
        row_blocks = kv.row_blocks if kv.row_blocks is not None else 0.0
        share_text = q.dtype != torch.float32 and shares_text_rows(B * H * nqb, kv.nkb, n_text_blocks, row_blocks, D)
        order = work_order(B, H, nqb, n_text_blocks, q.device, share_text)
    bias_ptr, bias_strides = _bias_args(key_bias)
    with _lib.on(q.device):
        rc = _lib.load().sa_block_sparse_fwd_lse(
            _lib.DTYPES[q.dtype], q.data_ptr(), _lib.i64(*q.stride()[:3]), k.data_ptr(), _lib.i64(*k.stride()[:3]),
            v.data_ptr(), _lib.i64(*v.stride()[:3]), out.data_ptr(), _lib.i64(*out.stride()[:3]), B, H, Lq, Lk, D,
            kv.idx.data_ptr(), kv.cnt.data_ptr(), kv.max_cnt, bias_ptr, bias_strides, float(sm_scale),
            _lib.ptr(order), order.numel() if order is not None else 0, parts, _lib.ptr(ws),
            ws.numel() if ws is not None else 0, lse.data_ptr(), _lib.stream_of(q))
    _lib.check(rc, "sa_block_sparse_fwd_lse")
    return out, lse


def transpose_kv_list(kv: KVList) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q_beg int32 [B*H, nkb + 1], q_idx int32 [B*H, nqb * max_cnt]): the query blocks that list each
    key block, ascending (`sa_kv_list_transpose`); key block j of a head has entries
    q_idx[q_beg[j]:q_beg[j + 1]] of the head's row."""
    _lib.require_gpu(kv.idx, kv.cnt)
    BH = kv.B * kv.H
    beg = torch.empty(BH, kv.nkb + 1, dtype=torch.int32, device=kv.idx.device)
    idx = torch.empty(BH, kv.nqb * kv.max_cnt, dtype=torch.int32, device=kv.idx.device)
    with _lib.on(kv.idx.device):
        rc = _lib.load().sa_kv_list_transpose(kv.idx.data_ptr(), kv.cnt.data_ptr(), BH, kv.nqb, kv.nkb, kv.max_cnt,
                                              beg.data_ptr(), idx.data_ptr(), _lib.stream_of(kv.idx))
    _lib.check(rc, "sa_kv_list_transpose")
    return beg, idx


def _backward(dout, q, k, v, out, lse, kv: KVList, sm_scale: float, key_bias, n_text_blocks: int, needs):
    """(dq, dk, dv), None where not needed; q, k, v checked and aligned, key_bias expanded."""
    B, H, Lq, D = q.shape
    Lk = k.shape[2]
    dout = _rows16(dout)
    dq = torch.empty(B, H, Lq, D, dtype=q.dtype, device=q.device) if needs[0] else None
    dk, dv = (torch.empty(B, H, Lk, D, dtype=q.dtype, device=q.device) if n else None for n in needs[1:])
    strides = [s for t in (q, k, v, out, dout, dq, dk, dv) for s in (t.stride()[:3] if t is not None else (0, 0, 0))]
    lib = _lib.load()
    n = ctypes.c_int64(0)
    _lib.check(lib.sa_block_sparse_bwd_workspace(B, H, Lq, ctypes.byref(n)), "sa_block_sparse_bwd_workspace")
    ws = torch.empty(n.value, dtype=torch.uint8, device=q.device)
    q_beg, q_idx = transpose_kv_list(kv) if needs[1] or needs[2] else (None, None)
    q_order = work_order(B, H, kv.nqb, n_text_blocks, q.device)
    k_order = work_order(B, H, kv.nkb, n_text_blocks, q.device)
    bias_ptr, bias_strides = _bias_args(key_bias)
    with _lib.on(q.device):
        rc = lib.sa_block_sparse_bwd(
            _lib.DTYPES[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr(),
            lse.data_ptr(), _lib.ptr(dq), _lib.ptr(dk), _lib.ptr(dv), _lib.i64(*strides), B, H, Lq, Lk, D,
            kv.idx.data_ptr(), kv.cnt.data_ptr(), kv.max_cnt, _lib.ptr(q_beg), _lib.ptr(q_idx), bias_ptr, bias_strides,
            float(sm_scale), q_order.data_ptr(), q_order.numel(), k_order.data_ptr(), k_order.numel(), ws.data_ptr(),
            ws.numel(), _lib.stream_of(q))
    _lib.check(rc, "sa_block_sparse_bwd")
    return dq, dk, dv


def block_sparse_attention_lse(q, k, v, kv: KVList, sm_scale: float, key_bias: Optional[torch.Tensor] = None,
                               n_text_blocks: int = 0):
    """(out, lse): `block_sparse_attention` (q [B,H,Lq,D], k/v [B,H,Lk,D], bf16, fp16 or fp32, D 64 or
    128; key_bias fp32 [B,H,Lk], not with fp32) and the rows' log2-sum-exp2, fp32
    [B, H, 64 * ceil(Lq / 64)], +inf for rows without a key and past Lq. No autograd.
    `n_text_blocks` only affects scheduling, as there."""
    key_bias = _check_inputs(q, k, v, kv, key_bias)
    with torch.no_grad():
        return _forward(_rows16(q), _rows16(k), _rows16(v), kv, sm_scale, key_bias, n_text_blocks)


def block_sparse_attention_backward(dout, q, k, v, out, lse, kv: KVList, sm_scale: float,
                                    key_bias: Optional[torch.Tensor] = None, n_text_blocks: int = 0,
                                    needs=(True, True, True)):
    """(dq, dk, dv) for the gradient dout of out, with the inputs and results of
    `block_sparse_attention_lse`; None in the places where `needs` is false."""
    key_bias = _check_inputs(q, k, v, kv, key_bias)
    _lib.require_gpu(dout, out, lse)
    for name, t in (("dout", dout), ("out", out)):
        if t.shape != q.shape or t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{name} must be like q: {tuple(q.shape)} {q.dtype}, got {tuple(t.shape)} {t.dtype}")
    if lse.dtype != torch.float32 or tuple(lse.shape) != (q.shape[0], q.shape[1], kv.nqb * BLOCK) \
            or not lse.is_contiguous() or lse.device != q.device:
        raise ValueError("lse must be block_sparse_attention_lse's")
    with torch.no_grad():
        return _backward(dout, _rows16(q), _rows16(k), _rows16(v), _rows16(out), lse, kv, sm_scale, key_bias,
                         n_text_blocks, tuple(needs))


class _TrainAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, kv_idx, kv_cnt, key_bias, shape, sm_scale, n_text_blocks):
        kv = KVList(kv_idx, kv_cnt, *shape[:4], row_blocks=shape[4])
        q, k, v = _rows16(q), _rows16(k), _rows16(v)
        out, lse = _forward(q, k, v, kv, sm_scale, key_bias, n_text_blocks)
        ctx.save_for_backward(q, k, v, out, lse, kv_idx, kv_cnt, key_bias)
        ctx.args = shape, sm_scale, n_text_blocks
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, kv_idx, kv_cnt, key_bias = ctx.saved_tensors
        shape, sm_scale, n_text_blocks = ctx.args
        kv = KVList(kv_idx, kv_cnt, *shape[:4])
        grads = _backward(dout, q, k, v, out, lse, kv, sm_scale, key_bias, n_text_blocks, ctx.needs_input_grad[:3])
        return (*grads, None, None, None, None, None, None)


class _NoKeys(torch.autograd.Function):
    """The output where there is no query or no key: zeros, with zero gradients."""

    @staticmethod
    def forward(ctx, q, k, v):
        ctx.save_for_backward(q, k, v)
        return torch.zeros(q.shape, dtype=q.dtype, device=q.device)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        return tuple(torch.zeros_like(t) for t in ctx.saved_tensors)


def block_sparse_attention_train(q, k, v, kv: KVList, sm_scale: float, key_bias: Optional[torch.Tensor] = None,
                                 n_text_blocks: int = 0) -> torch.Tensor:
    """`block_sparse_attention` over the blocks of `kv`, differentiable in q, k and v (once).

    q [B,H,Lq,D], k/v [B,H,Lk,D] on the GPU, bf16, fp16 or fp32 (one type), D = 64 or 128, any strides
    (tensors whose rows are not 16-byte aligned are copied); key_bias fp32 [B,H,Lk] or None, not
    differentiated, not with fp32. `n_text_blocks` only affects scheduling: so many first block rows
    and columns are listed by every other block. The lists (and key_bias) must stay as they are until
    the backward pass has run."""
    key_bias = _check_inputs(q, k, v, kv, key_bias)
    return _TrainAttention.apply(q, k, v, kv.idx, kv.cnt, key_bias, (kv.B, kv.H, kv.nqb, kv.nkb, kv.row_blocks),
                                 float(sm_scale), int(n_text_blocks))


def block_sparse_train_fn(q, k, v, block_sparse_mask, sm_scale, key_bias: Optional[torch.Tensor] = None,
                          n_text_blocks: int = 0, BLOCK_M: int = 64, BLOCK_N: int = 64) -> torch.Tensor:
    """`block_sparse_triton_fn` that can be trained: attention over the blocks that
    block_sparse_mask [B,H,>=ceil(Lq/BLOCK_M),>=ceil(Lk/BLOCK_N)] (bool or integer, any strides) keeps,
    differentiable in q, k and v. BLOCK_M and BLOCK_N are powers of two from 64 to 1024, as of
    `sparse_attention_factory`; smaller blocks have no gradients (NotImplementedError). See
    `block_sparse_attention_train`."""
    _lib.require_gpu(q, k, v, block_sparse_mask)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4 or block_sparse_mask.dim() != 4:
        raise ValueError("q, k, v and the block mask must be 4-D")
    B, H, Lq, D = q.shape
    Lk = k.shape[2]
    if B * H * Lq == 0 or Lk == 0:
        if q.dtype not in _TYPES or not q.dtype == k.dtype == v.dtype:
            raise TypeError(f"q, k, v must share one of bf16, fp16 and fp32, got {q.dtype}, {k.dtype}, {v.dtype}")
        if k.shape != (B, H, Lk, D) or v.shape != (B, H, Lk, D):
            raise ValueError(f"shape mismatch q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}")
        return _NoKeys.apply(q, k, v)
    if BLOCK_M == BLOCK and BLOCK_N == BLOCK:
        kv = kv_list_from_mask(block_sparse_mask, B, H, math.ceil(Lq / BLOCK), math.ceil(Lk / BLOCK))
    elif min(BLOCK_M, BLOCK_N) < BLOCK:
        raise NotImplementedError(f"gradients of {BLOCK_M} x {BLOCK_N} blocks: blocks smaller than 64")
    else:
        kv, _ = cell_kv_list(block_sparse_mask, B, H, Lq, Lk, int(BLOCK_M), int(BLOCK_N))
    return block_sparse_attention_train(q, k, v, kv, sm_scale, key_bias, n_text_blocks)
