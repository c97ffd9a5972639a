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


_OPERANDS = ("q", "k", "v", "out", "dout", "dq", "dk", "dv")  # in the order of AttnTrain.strides


def _set(call, **tensors):
    for name, t in tensors.items():
        setattr(call, name, t.data_ptr())
        i = 3 * _OPERANDS.index(name)
        call.strides[i:i + 3] = t.stride()[:3]


def _set_bias(call, key_bias):
    if key_bias is not None:
        call.key_bias = key_bias.data_ptr()
        call.bias_strides[:] = key_bias.stride()[:2]


_WORKSPACE_BYTES = {}


class _Call:
    """What the backward pass needs of a call beside its tensors: the description of the call on checked,
    aligned inputs (key_bias expanded), its dispatch orders and the size of its workspace."""

    def __init__(self, q, k, v, kv: KVList, sm_scale: float, key_bias, n_text_blocks: int):
        B, H, Lq, D = q.shape
        Lk = k.shape[2]
        self.args = _lib.AttnTrain(dtype=_lib.DTYPES[q.dtype], B=B, H=H, Lq=Lq, Lk=Lk, D=D, max_cnt=kv.max_cnt, parts=1,
                                   kv_idx=kv.idx.data_ptr(), kv_cnt=kv.cnt.data_ptr(), sm_scale=sm_scale)
        _set(self.args, q=q, k=k, v=v)
        _set_bias(self.args, key_bias)
        self.shapes = (B, H, Lq, D), (B, H, Lk, D), (B, H, Lk, D)  # of the gradients, contiguous
        sq, sk = (H * Lq * D, Lq * D, D), (H * Lk * D, Lk * D, D)
        self.args.strides[15:24] = (*sq, *sk, *sk)
        self.orders = [work_order(B, H, n, n_text_blocks, q.device) for n in (kv.nqb, kv.nkb)]
        (self.args.q_order, self.args.n_q_slots), (self.args.k_order, self.args.n_k_slots) = (
            (o.data_ptr(), o.numel()) for o in self.orders)
        key = (self.args.dtype, B, H, Lq, Lk, D, kv.max_cnt)
        self.bytes = _WORKSPACE_BYTES.get(key)
        if self.bytes is None:
            n = ctypes.c_int64(0)
            _lib.check(_lib.load().sa_block_sparse_bwd_workspace(self.args, ctypes.byref(n)),
                       "sa_block_sparse_bwd_workspace")
            self.bytes = _WORKSPACE_BYTES[key] = n.value


def _forward(call: _lib.AttnTrain, q, k, v, kv: KVList, n_text_blocks: int):
    """(out, lse) of a call."""
    B, H, Lq, D = q.shape
    n_items = B * H * kv.nqb
    out = torch.empty(B, H, Lq, D, dtype=q.dtype, device=q.device)
    lse = torch.empty(B, H, kv.nqb * BLOCK, dtype=torch.float32, device=q.device)
    # The launch variants of block_sparse_attention: key-range parts for few blocks over long lists,
    # else a work order; fp32 on split operands where it takes them.
    ws = None
    if q.dtype == torch.float32:
        if kv.nqb >= F32_TERMS_BLOCKS:
            ws = f32_terms_workspace(B, H, k.shape[2], D, q.device)
    elif not call.key_bias:
        call.parts = split_parts(n_items, kv.max_cnt, D)
        if call.parts > 1:
            ws = torch.empty(split_workspace_bytes(n_items, D, call.parts), dtype=torch.uint8, device=q.device)
    if call.parts == 1:
        # Lists of unknown length count as short ones beside the text rows': [1, 15, 17776, 64] with a
        # fifth of the blocks 376 / 338 us without / with shared text rows, [1, 30, 4546, 64] 91 / 73 (were
        # they all long after all: [1, 15, 17776, 64] dense 1 185 / 1 364).
        row_blocks = kv.row_blocks if kv.row_blocks is not None or kv.dense else 0.0
        share_text = q.dtype != torch.float32 and shares_text_rows(n_items, kv.nkb, n_text_blocks, row_blocks, D)
        order = work_order(B, H, kv.nqb, n_text_blocks, q.device, share_text)
        call.fwd_order, call.n_fwd_slots = order.data_ptr(), order.numel()
    call.workspace, call.workspace_bytes = (ws.data_ptr(), ws.numel()) if ws is not None else (None, 0)
    _set(call, out=out)
    call.lse = lse.data_ptr()
    with _lib.on(q.device):
        rc = _lib.load().sa_block_sparse_fwd_lse(call, _lib.stream_of(q))
    _lib.check(rc, "sa_block_sparse_fwd_lse")
    return out, lse


def _backward(args: _lib.AttnTrain, call: _Call, dout, needs):
    """[dq, dk, dv], None where not needed; args describes the call with its operands, out and lse."""
    dout = _rows16(dout)
    device = dout.device
    args.dout = dout.data_ptr()
    args.strides[12:15] = dout.stride()[:3]
    grads = [torch.empty(shape, dtype=dout.dtype, device=device) if n else None for n, shape in zip(needs, call.shapes)]
    args.dq, args.dk, args.dv = (t.data_ptr() if t is not None else None for t in grads)
    ws = torch.empty(call.bytes, dtype=torch.uint8, device=device)
    args.workspace, args.workspace_bytes = ws.data_ptr(), call.bytes
    with _lib.on(device):
        rc = _lib.load().sa_block_sparse_bwd(args, _lib.stream_of(dout))
    _lib.check(rc, "sa_block_sparse_bwd")
    return grads


def transpose_kv_list(kv: KVList) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q_beg int32 [B*H, nkb + 1], q_idx int32 [B*H, nqb * max_cnt]): the query blocks that list each
    key block, ascending (`sa_kv_list_transpose`); key block j of a head has entries
    q_idx[q_beg[j]:q_beg[j + 1]] of the head's row. The backward pass makes its own."""
    _lib.require_gpu(kv.idx, kv.cnt)
    BH = kv.B * kv.H
    beg = torch.empty(BH, kv.nkb + 1, dtype=torch.int32, device=kv.idx.device)
    idx = torch.empty(BH, kv.nqb * kv.max_cnt, dtype=torch.int32, device=kv.idx.device)
    with _lib.on(kv.idx.device):
        rc = _lib.load().sa_kv_list_transpose(kv.idx.data_ptr(), kv.cnt.data_ptr(), BH, kv.nqb, kv.nkb, kv.max_cnt,
                                              beg.data_ptr(), idx.data_ptr(), _lib.stream_of(kv.idx))
    _lib.check(rc, "sa_kv_list_transpose")
    return beg, idx


def block_sparse_attention_lse(q, k, v, kv: KVList, sm_scale: float, key_bias: Optional[torch.Tensor] = None,
                               n_text_blocks: int = 0):
    """(out, lse): `block_sparse_attention` (q [B,H,Lq,D], k/v [B,H,Lk,D], bf16, fp16 or fp32, D 64 or
    128; key_bias fp32 [B,H,Lk], not with fp32) and the rows' log2-sum-exp2, fp32
    [B, H, 64 * ceil(Lq / 64)], +inf for rows without a key and past Lq. No autograd.
    `n_text_blocks` only affects scheduling, as there."""
    key_bias = _check_inputs(q, k, v, kv, key_bias)
    with torch.no_grad():
        q, k, v = _rows16(q), _rows16(k), _rows16(v)
        return _forward(_Call(q, k, v, kv, float(sm_scale), key_bias, n_text_blocks).args, q, k, v, kv, n_text_blocks)


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
        q, k, v, out = _rows16(q), _rows16(k), _rows16(v), _rows16(out)
        call = _Call(q, k, v, kv, float(sm_scale), key_bias, n_text_blocks)
        _set(call.args, out=out)
        call.args.lse = lse.data_ptr()
        return tuple(_backward(call.args, call, dout, needs))


class _TrainAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, kv, sm_scale, key_bias, n_text_blocks):
        q, k, v = _rows16(q), _rows16(k), _rows16(v)
        call = ctx.call = _Call(q, k, v, kv, sm_scale, key_bias, n_text_blocks)
        out, lse = _forward(call.args, q, k, v, kv, n_text_blocks)
        saved = (q, k, v, out, lse, kv.idx, kv.cnt, key_bias)
        ctx.save_for_backward(*saved)
        ctx.places = [(t.data_ptr(), t.stride()) for t in saved if t is not None]
        return out

    @staticmethod
    def backward(ctx, dout):
        if torch.is_grad_enabled():
            raise RuntimeError("block-sparse attention is differentiable once (create_graph=True is not supported)")
        saved = ctx.saved_tensors
        # A copy of the forward pass's description: this may run twice, or in two threads.
        args = _lib.AttnTrain.from_buffer_copy(ctx.call.args)
        if ctx.places != [(t.data_ptr(), t.stride()) for t in saved if t is not None]:
            # Hooks on saved tensors have moved them.
            q, k, v, out, lse, kv_idx, kv_cnt, key_bias = saved
            q, k, v, out = _rows16(q), _rows16(k), _rows16(v), _rows16(out)
            _set(args, q=q, k=k, v=v, out=out)
            args.lse, args.kv_idx, args.kv_cnt = lse.data_ptr(), kv_idx.data_ptr(), kv_cnt.data_ptr()
            _set_bias(args, key_bias)
        return (*_backward(args, ctx.call, dout, ctx.needs_input_grad[:3]), None, None, None, None)


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
    and columns are listed by every other block, beside shorter lists. The lists (and key_bias) must stay as they are until
    the backward pass has run."""
    key_bias = _check_inputs(q, k, v, kv, key_bias)
    return _TrainAttention.apply(q, k, v, kv, float(sm_scale), key_bias, int(n_text_blocks))


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
