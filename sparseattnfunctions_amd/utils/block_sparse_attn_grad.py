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

The forward pass is the kernel of `block_sparse_attention` with bf16 (fp16) scores, or fp32 on split
operands, and also stores each row's log2-sum-exp2; the backward pass recomputes the probabilities
from it, block by block, and keeps nothing of the size of the attention map (`sa_block_sparse_bwd`).
Between the two a call holds q, k, v and out, a float per row and its lists: a mask's lists of both
sides are full width, eight bytes for each pair of blocks (191 MB at [1, 48, 45104, 64], whose q has
277 MB), a caller's are the caller's own and their key side is made in the backward call.

Gradients of a 16-bit call round P and dS to its type, those of an fp32 call take operands below 3.39e38
in size (from there on bf16 rounds to infinity) as three exact bf16 terms (values below about 1e-33 lose
their low ones); sums are fp32 in a fixed order, so that a step repeats bit for bit. In fp16, dS has the
range of the type: scale the loss as usual; P, which that does not help, takes a factor of 4096 of its
own where lists may hold more than 16 384 keys.

The attention is differentiable once, and `create_graph=True` is refused as a whole: take the gradient of
a penalty on another part of the graph with `torch.autograd.grad` of that part. A query row without a key
(an empty list, or keys all biased to -inf) has a zero output and zero gradients; a key block in no list
has zero gradients. The mask, the lists and key_bias are not differentiated.

A key_bias is added to the scores in fp32, in both passes alike, so that one as large as 1e9 leaves a
row that lists nothing else few of its scores' bits. One below -2.35e38 (the type's lowest value among
them) counts as -inf, and keys that it masks still enter the products: their k and v have to be finite,
as with any additive mask. Keys in blocks that no row lists, and memory behind the last row, are not
read into any sum.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .._kv import KVList
from .block_sparse_attn_kernel import (BLOCK, cell_kv_list, f32_terms_workspace, shares_text_rows,
                                       split_parts, split_workspace_bytes, work_order)


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """t [B,H,L,D] with a contiguous last axis and 16-byte aligned rows (a copy where it has not)."""
    sb, sh, sl, sd = t.stride()
    if sd != 1 or (sb | sh | sl) * t.element_size() % 16 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


class _MaskLists:
    """The lists of a 64 x 64 block mask, which the forward call makes, and room for the rows'
    log2-sum-exp2: one buffer of entries, counts, sums (with `biased` and the rows' offsets) and, with `keys`, the
    key blocks' entries and counts for the backward pass."""

    def __init__(self, mask, B, H, nqb, nkb, keys, biased):
        if mask.shape[2] < nqb or mask.shape[3] < nkb:
            raise ValueError(f"block mask {tuple(mask.shape)} smaller than the block grid ({nqb}, {nkb})")
        if mask.dtype != torch.bool:
            mask = mask != 0
        if mask.shape[:2] != (B, H):
            mask = mask.expand(B, H, -1, -1)
        self.mask, self.nkb, self.keys = mask, nkb, keys
        n = nqb * (nkb + 1 + (2 if biased else 1) * BLOCK) + (nkb * (nqb + 1) if keys else 0)
        self.idx = mask.new_empty(B * H * n, dtype=torch.int32)
        self.cnt = None


def _check_lists(kv, B, H, nqb, nkb):
    if (kv.B, kv.H, kv.nqb, kv.nkb) != (B, H, nqb, nkb) or kv.cnt.numel() != B * H * nqb or kv.idx.dim() != 2 \
            or kv.idx.shape[0] != B * H * nqb:
        raise ValueError(f"kv lists of {kv.B} x {kv.H} x {kv.nqb} x {kv.nkb} blocks, expected {B} x {H} x {nqb} x {nkb}")
    if kv.idx.dtype != torch.int32 or kv.cnt.dtype != torch.int32 or not kv.idx.is_contiguous() \
            or not kv.cnt.is_contiguous():
        raise ValueError("kv lists must be contiguous int32 tensors")


def _check_inputs(q, k, v, kv, key_bias):
    """key_bias expanded. kv: a caller's lists, or ones for these shapes (_MaskLists)."""
    own_lists = type(kv) is _MaskLists
    tensors = (k, v, kv.idx) if own_lists else (k, v, kv.idx, kv.cnt)
    if key_bias is not None:
        tensors += (key_bias,)
    device = q.device
    if device.type != "cuda":
        _lib.require_gpu(q)
    for t in tensors:
        if t.device != device:
            _lib.require_gpu(*tensors)
            raise ValueError("q, k, v, the lists and key_bias must be on one device")
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"q, k, v must be [B, H, L, D], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if q.dtype not in _lib.DTYPES or not q.dtype == k.dtype == v.dtype:
        raise TypeError(f"q, k, v must share one of bf16, fp16 and fp32, got {q.dtype}, {k.dtype}, {v.dtype}")
    B, H, Lq, D = q.shape
    Lk = k.shape[2]
    if k.shape != (B, H, Lk, D) or v.shape != (B, H, Lk, D):
        raise ValueError(f"shape mismatch q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}")
    if D not in (64, 128):
        raise NotImplementedError(f"head_dim {D} (64 or 128)")
    nqb, nkb = (Lq + BLOCK - 1) // BLOCK, (Lk + BLOCK - 1) // BLOCK
    if not own_lists:
        _check_lists(kv, B, H, nqb, nkb)
    if key_bias is not None:
        if q.dtype == torch.float32:
            raise NotImplementedError("fp32 inputs: plain block lists only (no key_bias)")
        if key_bias.requires_grad:
            raise ValueError("key_bias is not differentiated; pass key_bias.detach()")
        if key_bias.dtype != torch.float32 or key_bias.dim() == 0 or key_bias.shape[-1] != Lk \
                or (Lk > 1 and key_bias.stride(-1) != 1):
            raise ValueError("key_bias must be fp32 [B,H,Lk] with a contiguous key axis")
        key_bias = key_bias.expand(B, H, Lk)
    return key_bias


_OPERANDS = ("q", "k", "v", "out", "dout", "dq", "dk", "dv")  # in the order of AttnTrain.strides


def _set(call, **tensors):
    for name, t in tensors.items():
        setattr(call, name, t.data_ptr())
        i = 3 * _OPERANDS.index(name)
        call.strides[i:i + 3] = t.stride()[:3]


def _set_lists(call, plan, idx, cnt, lse=None):
    """cnt None: a _MaskLists' buffer, which has the lse too. lse with a bias: [2, ...], the sums and the offsets."""
    call.kv_idx = at = idx.data_ptr()
    if cnt is None:
        call.kv_cnt = at = at + 4 * plan.rows * call.max_cnt
        call.lse = at = at + 4 * plan.rows
        at += 4 * BLOCK * plan.rows
        if plan.biased:
            call.row_max = at
            at += 4 * BLOCK * plan.rows
        if plan.keys:
            call.q_idx = at
            call.q_cnt = at + 4 * plan.rows * call.max_cnt
    else:
        call.kv_cnt = cnt.data_ptr()
        if lse is not None:
            _set_lse(call, plan, lse)


def _set_lse(call, plan, lse):
    call.lse = at = lse.data_ptr()
    if plan.biased:
        call.row_max = at + 4 * BLOCK * plan.rows


def _set_bias(call, key_bias):
    if key_bias is not None:
        call.key_bias = key_bias.data_ptr()
        call.bias_strides[:] = key_bias.stride()[:2]


class _Plan:
    """What calls of one shape share: a description without pointers, launch variants, dispatch orders
    and workspace sizes."""

    def __init__(self, dtype, device, q_shape, Lk, q_strides, k_strides, v_strides, max_cnt, row_blocks, biased, sm_scale,
                 n_text_blocks, keys):
        B, H, Lq, D = q_shape
        if max(B, H, Lq, Lk, max_cnt) >= 2 ** 31 - BLOCK:
            raise ValueError(f"B={B} H={H} Lq={Lq} Lk={Lk}: sizes of 32 bits")
        n_text_blocks = min(n_text_blocks, max(Lq, Lk))  # (no head has more)
        self.keys, self.biased = keys, biased  # keys: with key blocks' lists (_MaskLists)
        nqb, nkb = math.ceil(Lq / BLOCK), math.ceil(Lk / BLOCK)
        n_items = B * H * nqb
        args = self.args = _lib.AttnTrain(dtype=_lib.DTYPES[dtype], B=B, H=H, Lq=Lq, Lk=Lk, D=D, max_cnt=max_cnt, parts=1,
                                          sm_scale=sm_scale, n_text_blocks=n_text_blocks)
        self.out, self.rows = (B, H, Lq, D), n_items
        self.lse = (2, B, H, nqb * BLOCK) if biased else (B, H, nqb * BLOCK)
        self.grads = (B, H, Lq, D), (B, H, Lk, D), (B, H, Lk, D)
        sq, sk = (H * Lq * D, Lq * D, D), (H * Lk * D, Lk * D, D)
        self.square = Lq == Lk  # dk and dv are like dout
        self.plain_q = tuple(q_strides) == (*sq, 1)
        args.strides[:] = (*q_strides[:3], *k_strides[:3], *v_strides[:3], *sq, *sq, *sq, *sk, *sk)
        # The forward pass takes block_sparse_attention's launch variants: key-range parts for few blocks
        # over long lists, else a work order. fp32 takes split operands for few query blocks too: 30 heads of one
        # block over 1, 4, 8 and 63 blocks 16.6 / 17.6, 46 / 18, 87 / 25 and 697 / 102 us without / with.
        self.terms = dtype == torch.float32
        if dtype != torch.float32 and not biased:
            args.parts = split_parts(n_items, max_cnt, D)
        self.forward_bytes = split_workspace_bytes(n_items, D, args.parts) if args.parts > 1 else 0
        # Lists of unknown length count as short ones beside the text rows': [1, 15, 17776, 64] with a
        # fifth of the blocks 376 / 338 us without / with shared text rows, [1, 30, 4546, 64] 91 / 73 (were
        # they all long after all: [1, 15, 17776, 64] dense 1 185 / 1 364).
        share_text = dtype != torch.float32 and shares_text_rows(n_items, nkb, n_text_blocks, row_blocks, D)
        self.orders = [work_order(B, H, nqb, n_text_blocks, device, share_text), work_order(B, H, nqb, n_text_blocks, device),
                       work_order(B, H, nkb, n_text_blocks, device)]
        for name, order in zip(("fwd", "q", "k"), self.orders):
            setattr(args, name + "_order", order.data_ptr())
            setattr(args, "n_" + name + "_slots", order.numel())
        n = ctypes.c_int64(0)
        # (whether there are any is all that this reads)
        args.q_idx, args.key_bias = 1 if keys else None, 1 if biased else None
        _lib.check(_lib.load().sa_block_sparse_bwd_workspace(args, ctypes.byref(n)), "sa_block_sparse_bwd_workspace")
        args.q_idx = args.key_bias = None
        self.backward_bytes = n.value
        # Why the backward pass refuses such calls, without and with dk or dv: nobody is to learn it there.
        self.refusals = []
        args.q_idx, args.key_bias = 1 if keys else None, 1 if biased else None
        for wanted in (None, 1):
            args.dk = wanted
            rc = _lib.load().sa_block_sparse_bwd_check(args)
            self.refusals.append(_lib.load().sa_last_error().decode() if rc == _lib.SA_ERR_UNSUPPORTED else None)
        args.q_idx = args.key_bias = args.dk = None

    def check_backward(self, needs):
        refusal = self.refusals[bool(needs[1] or needs[2])]
        if any(needs[:3]) and refusal is not None:
            raise NotImplementedError(refusal)


_plan = functools.lru_cache(maxsize=1024)(_Plan)


def _describe(q, k, v, kv, sm_scale: float, key_bias, n_text_blocks: int):
    """(plan, description) of a call on checked, aligned inputs; key_bias expanded."""
    masked = type(kv) is _MaskLists
    if masked:
        max_cnt, row_blocks = kv.nkb, 0.0
    else:
        max_cnt, row_blocks = kv.idx.shape[1], kv.row_blocks if kv.row_blocks is not None or kv.dense else 0.0
    plan = _plan(q.dtype, q.device, q.shape, k.shape[2], q.stride(), k.stride(), v.stride(), max_cnt, row_blocks,
                 key_bias is not None, sm_scale, n_text_blocks, masked and kv.keys)
    args = _lib.AttnTrain.from_buffer_copy(plan.args)
    args.q, args.k, args.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    _set_lists(args, plan, kv.idx, kv.cnt)
    if masked:
        args.mask = kv.mask.data_ptr()
        args.mask_strides[:] = kv.mask.stride()
    _set_bias(args, key_bias)
    return plan, args


def _forward(plan: _Plan, args: _lib.AttnTrain, q):
    """(out, lse) of a call, whose description then has them; lse None where it has room for it."""
    device = q.device
    # (empty_like is the cheaper call: 1.1 us on the host, empty 2.1)
    out = torch.empty_like(q) if plan.plain_q else torch.empty(plan.out, dtype=q.dtype, device=device)
    lse = None
    if not args.lse:
        lse = torch.empty(plan.lse, dtype=torch.float32, device=device)
        _set_lse(args, plan, lse)
    ws = None
    if plan.terms:
        ws = f32_terms_workspace(args.B, args.H, args.Lk, args.D, device)
    elif plan.forward_bytes:
        ws = torch.empty(plan.forward_bytes, dtype=torch.uint8, device=device)
    args.workspace, args.workspace_bytes = (ws.data_ptr(), ws.numel()) if ws is not None else (None, 0)
    args.out = out.data_ptr()
    with _lib.on(device):
        rc = _lib.load().sa_block_sparse_fwd_lse(args, _lib.stream_of(q))
    _lib.check(rc, "sa_block_sparse_fwd_lse")
    return out, lse


def _backward(plan: _Plan, args: _lib.AttnTrain, dout, needs):
    """(dq, dk, dv), None where not needed; args describes the call with its operands, out and lse."""
    plain = dout.is_contiguous() and dout.data_ptr() % 16 == 0
    if not plain:
        dout = _rows16(dout)
        if (dout.shape[2] + BLOCK) * dout.stride(2) * dout.element_size() >= 1 << 30:  # (rows far apart: 32-bit offsets)
            dout = dout.contiguous()
        args.strides[12:15] = dout.stride()[:3]
    args.dout = dout.data_ptr()
    device = dout.device
    dq = dk = dv = None
    if needs[0]:
        dq = torch.empty_like(dout) if plain else dout.new_empty(plan.grads[0])
        args.dq = dq.data_ptr()
    plain = plain and plan.square
    if needs[1]:
        dk = torch.empty_like(dout) if plain else dout.new_empty(plan.grads[1])
        args.dk = dk.data_ptr()
    if needs[2]:
        dv = torch.empty_like(dout) if plain else dout.new_empty(plan.grads[2])
        args.dv = dv.data_ptr()
    ws = dout.new_empty(plan.backward_bytes, dtype=torch.uint8)
    args.workspace, args.workspace_bytes = ws.data_ptr(), plan.backward_bytes
    with _lib.on(device):
        rc = _lib.load().sa_block_sparse_bwd(args, _lib.stream_of(dout))
    _lib.check(rc, "sa_block_sparse_bwd")
    return dq, dk, dv


def transpose_kv_list(kv: KVList) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q_beg int32 [B*H, nkb + 1], q_idx int32 [B*H, nqb * max_cnt]): the query blocks that list each
    key block, ascending (`sa_kv_list_transpose`); key block j of a head has entries
    q_idx[q_beg[j]:q_beg[j + 1]] of the head's row. The backward pass makes its own."""
    _lib.require_gpu(kv.idx, kv.cnt)
    if kv.cnt.device != kv.idx.device:
        raise ValueError("the lists must be on one device")
    _check_lists(kv, kv.B, kv.H, kv.nqb, kv.nkb)
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
    [B, H, 64 * ceil(Lq / 64)], +inf for rows without a key and past Lq. With key_bias [2, B, H, ...]: the
    log2-sum-exp2 of the scores less an offset of each row, and that offset; their sum is the whole, rounded to
    the bias's magnitude. No autograd.
    `n_text_blocks` only affects scheduling, as there."""
    key_bias = _check_inputs(q, k, v, kv, key_bias)
    with torch.no_grad():
        q, k, v = _rows16(q), _rows16(k), _rows16(v)
        return _forward(*_describe(q, k, v, kv, float(sm_scale), key_bias, int(n_text_blocks)), q)


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
    shape = (q.shape[0], q.shape[1], kv.nqb * BLOCK)
    if key_bias is not None:
        shape = (2, *shape)
    if lse.dtype != torch.float32 or tuple(lse.shape) != shape or not lse.is_contiguous() or lse.device != q.device:
        raise ValueError("lse must be block_sparse_attention_lse's")
    with torch.no_grad():
        q, k, v, out = _rows16(q), _rows16(k), _rows16(v), _rows16(out)
        plan, args = _describe(q, k, v, kv, float(sm_scale), key_bias, int(n_text_blocks))
        _set(args, out=out)
        _set_lse(args, plan, lse)
        return _backward(plan, args, dout, needs)


def _places(q, k, v, out, kv_idx, kv_cnt, lse, key_bias):
    """Where a call's saved tensors lie (lists and sums are contiguous)."""
    at = (q.data_ptr(), q.stride(), k.data_ptr(), k.stride(), v.data_ptr(), v.stride(), out.data_ptr(), out.stride(),
          kv_idx.data_ptr())
    if kv_cnt is not None:
        at += (kv_cnt.data_ptr(), lse.data_ptr())
    return at if key_bias is None else at + (key_bias.data_ptr(), key_bias.stride())


class _TrainAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, kv, sm_scale, key_bias, n_text_blocks, followed):
        q, k, v = _rows16(q), _rows16(k), _rows16(v)
        ctx.plan, ctx.args = _describe(q, k, v, kv, sm_scale, key_bias, n_text_blocks)
        if followed:
            ctx.plan.check_backward(ctx.needs_input_grad)
        out, lse = _forward(ctx.plan, ctx.args, q)
        ctx.args.mask = None  # (read by the forward call alone)
        ctx.save_for_backward(q, k, v, out, kv.idx, kv.cnt, lse, key_bias)
        ctx.places = _places(q, k, v, out, kv.idx, kv.cnt, lse, key_bias)
        return out

    @staticmethod
    def backward(ctx, dout):
        if torch.is_grad_enabled():
            raise RuntimeError("block-sparse attention is differentiable once (create_graph=True is not supported)")
        saved = ctx.saved_tensors
        # A copy of the forward pass's description: this may run twice, or in two threads.
        args = _lib.AttnTrain.from_buffer_copy(ctx.args)
        if ctx.places != _places(*saved):
            # Hooks on saved tensors have moved them.
            q, k, v, out, kv_idx, kv_cnt, lse, key_bias = saved
            q, k, v, out = _rows16(q), _rows16(k), _rows16(v), _rows16(out)
            _set(args, q=q, k=k, v=v, out=out)
            _set_lists(args, ctx.plan, kv_idx, kv_cnt, lse)
            _set_bias(args, key_bias)
        return (*_backward(ctx.plan, args, dout, ctx.needs_input_grad), None, None, None, None, None)


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
    and columns are listed by every other block, beside shorter lists. The lists (and key_bias) must
    stay as they are until the backward pass has run.

    A call captured into a HIP graph needs an eager one of its shapes before it (which makes the
    dispatch orders), and leaves that no eager graph holds: autograd ties a leaf's gradient to the
    stream of the leaf's first use, and its backward pass outside the capture would end the process."""
    key_bias = _check_inputs(q, k, v, kv, key_bias)
    return _TrainAttention.apply(q, k, v, kv, float(sm_scale), key_bias, int(n_text_blocks), torch.is_grad_enabled())


def block_sparse_train_fn(q, k, v, block_sparse_mask, sm_scale, key_bias: Optional[torch.Tensor] = None,
                          n_text_blocks: int = 0, BLOCK_M: int = 64, BLOCK_N: int = 64) -> torch.Tensor:
    """`block_sparse_triton_fn` that can be trained: attention over the blocks that
    block_sparse_mask [B,H,>=ceil(Lq/BLOCK_M),>=ceil(Lk/BLOCK_N)] (bool or integer, any strides) keeps,
    differentiable in q, k and v. BLOCK_M and BLOCK_N are powers of two from 64 to 1024, as of
    `sparse_attention_factory`; smaller blocks have no gradients (NotImplementedError). See
    `block_sparse_attention_train`."""
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4 or block_sparse_mask.dim() != 4:
        raise ValueError("q, k, v and the block mask must be 4-D")
    B, H, Lq, D = q.shape
    Lk = k.shape[2]
    if B * H * Lq == 0 or Lk == 0:
        _lib.require_gpu(q, k, v, block_sparse_mask)
        if q.dtype not in _lib.DTYPES or not q.dtype == k.dtype == v.dtype:
            raise TypeError(f"q, k, v must share one of bf16, fp16 and fp32, got {q.dtype}, {k.dtype}, {v.dtype}")
        if k.shape != (B, H, Lk, D) or v.shape != (B, H, Lk, D):
            raise ValueError(f"shape mismatch q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}")
        return _NoKeys.apply(q, k, v)
    if BLOCK_M == BLOCK and BLOCK_N == BLOCK:
        keys = torch.is_grad_enabled() and (k.requires_grad or v.requires_grad)
        kv = _MaskLists(block_sparse_mask, B, H, math.ceil(Lq / BLOCK), math.ceil(Lk / BLOCK), keys, key_bias is not None)
    elif min(BLOCK_M, BLOCK_N) < BLOCK:
        raise NotImplementedError(f"gradients of {BLOCK_M} x {BLOCK_N} blocks: blocks smaller than 64")
    else:
        _lib.require_gpu(q, k, v, block_sparse_mask)
        kv, _ = cell_kv_list(block_sparse_mask, B, H, Lq, Lk, int(BLOCK_M), int(BLOCK_N))
    key_bias = _check_inputs(q, k, v, kv, key_bias)
    return _TrainAttention.apply(q, k, v, kv, float(sm_scale), key_bias, int(n_text_blocks), torch.is_grad_enabled())
