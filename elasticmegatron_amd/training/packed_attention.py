"""Attention within documents, with its gradients.

    s = scale q . k  over the keys that a query sees,  out = softmax(s) v

The probabilities are never kept: the backward pass computes them again from the sums that forward leaves.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from .. import _native
from ._common import DTYPE_CODES, dtype_code, on_device, refuse_tangents, run_on, workspace


def _operand(t: torch.Tensor):
    """``t`` [rows, heads, dim] with unit stride along dim, and its other strides."""
    if t.stride(2) != 1 and t.shape[2] > 1:
        t = t.detach().contiguous()
    (rows, heads, dim), (row, head, _) = t.size(), t.stride()
    return t, (row if rows > 1 else heads * dim, head if heads > 1 else dim)


class _Call:
    """The checked arguments of one attention, and the record that the native calls take."""

    def __init__(self, q, k, v, offsets, key_offsets, causal, scale):
        if not isinstance(q, torch.Tensor):
            raise TypeError("q is no tensor")
        device = self.device = q.device
        for what, t in (("q", q), ("k", k), ("v", v)):
            on_device(what, t, device)
            dtype_code(t, what, (torch.bfloat16, torch.float16))
            if t.dtype != q.dtype:
                raise TypeError(f"{what} is {t.dtype}, q {q.dtype}")
            if t.dim() != q.dim() or t.dim() not in (3, 4):
                raise ValueError(f"{what} has {t.dim()} dimensions: [rows, heads, dim], or [batch, rows, heads, dim] for all three, is wanted")
        batch = q.shape[0] if q.dim() == 4 else 1
        if k.shape != v.shape or k.shape[-1] != q.shape[-1] or (q.dim() == 4 and k.shape[0] != batch):
            raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not fit q {tuple(q.shape)}")
        heads, dim, kv_heads = q.shape[-2], q.shape[-1], k.shape[-2]
        if not heads or not kv_heads or heads % kv_heads:
            raise ValueError(f"{heads} heads and {kv_heads} of keys: a multiple is wanted")
        if not 1 <= dim <= _native.EMRS_ATTENTION_MAX_DIM:
            raise ValueError(f"heads of {dim} elements: 1 to {_native.EMRS_ATTENTION_MAX_DIM} are wanted")
        if offsets is None:
            if key_offsets is not None:
                raise ValueError("key_offsets without offsets")
            documents = batch
        else:
            if q.dim() == 4:
                raise ValueError("offsets are of packed documents: [rows, heads, dim] is wanted")
            key_offsets = offsets if key_offsets is None else key_offsets
            if key_offsets is offsets and k.shape[0] != q.shape[0]:
                raise ValueError(f"{k.shape[0]} rows of keys for {q.shape[0]} of queries: key_offsets are wanted")
            for what, t in (("offsets", offsets), ("key_offsets", key_offsets)):
                on_device(what, t, device)
                if t.dtype not in (torch.int32, torch.int64):
                    raise TypeError(f"{what} is {t.dtype}: torch.int32 or torch.int64 is wanted")
            if offsets.dim() != 1 or offsets.shape[0] < 2 or key_offsets.shape != offsets.shape or key_offsets.dtype != offsets.dtype:
                raise ValueError(f"offsets {tuple(offsets.shape)} and key_offsets {tuple(key_offsets.shape)}: [documents + 1] of one type are wanted")
            documents = offsets.shape[0] - 1
        if scale is None:
            scale = 1 / math.sqrt(dim)
        if not 0 < scale < math.inf:
            raise ValueError(f"scale is {scale}: a positive number is wanted")
        a = self.record = _native.Attention()
        (q3, a.q_strides[:]), (k3, a.k_strides[:]), (v3, a.v_strides[:]) = (_operand(t if t.dim() == 3 else t.flatten(0, 1)) for t in (q, k, v))
        self._keep = [q3, k3, v3]
        a.dtype, a.causal, a.heads, a.kv_heads, a.dim = DTYPE_CODES[q.dtype], int(bool(causal)), heads, kv_heads, dim
        a.rows, a.key_rows, a.documents, a.scale = q3.shape[0], k3.shape[0], max(1, documents), scale
        if offsets is not None:
            offsets, key_offsets = offsets.contiguous(), key_offsets.contiguous()
            self._keep += [offsets, key_offsets]
            a.offsets, a.key_offsets, a.offset_bytes = offsets.data_ptr(), key_offsets.data_ptr(), offsets.element_size()
        a.q, a.k, a.v = q3.data_ptr(), k3.data_ptr(), v3.data_ptr()
        self.dtype, self.shape, self.key_shape = q.dtype, q.size(), k.size()

    def _run(self, call, backward):
        a = self.record
        size = _native.attention_workspace(a, backward)
        if size:
            scratch = workspace(size, self.device)
            a.workspace, a.workspace_bytes = scratch.data_ptr(), scratch.numel()
        run_on(self.device, call, a)

    def forward(self, with_lse):
        a = self.record
        out = torch.empty(self.shape, dtype=self.dtype, device=self.device)
        lse = torch.empty((a.heads, a.rows), dtype=torch.float32, device=self.device) if with_lse else None
        if a.rows:
            a.out, a.lse = out.data_ptr(), None if lse is None else lse.data_ptr()
            self._run(_native.attention_forward, False)
        return out, lse

    def backward(self, out, lse, grad_out, want_q, want_kv):
        a = self.record
        room = lambda shape: torch.empty(shape, dtype=self.dtype, device=self.device)  # noqa: E731
        gq = room(self.shape) if want_q else None
        gk, gv = (room(self.key_shape), room(self.key_shape)) if want_kv else (None, None)
        grad_out = grad_out.to(self.dtype)
        grad, a.grad_out_strides[:] = _operand(grad_out if grad_out.dim() == 3 else grad_out.flatten(0, 1))
        out, lse = out.contiguous(), lse.contiguous()
        a.out, a.lse, a.grad_out = out.data_ptr(), lse.data_ptr(), grad.data_ptr()
        a.grad_q = None if gq is None else gq.data_ptr()
        a.grad_k, a.grad_v = (gk.data_ptr(), gv.data_ptr()) if want_kv else (None, None)
        if a.rows or (want_kv and a.key_rows):
            self._run(_native.attention_backward, True)
        return gq, gk, gv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, offsets, key_offsets, causal, scale):
        out, lse = _Call(q, k, v, offsets, key_offsets, causal, scale).forward(True)
        ctx.save_for_backward(q, k, v, offsets, key_offsets, out, lse)
        ctx.causal, ctx.scale = causal, scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        q, k, v, offsets, key_offsets, out, lse = ctx.saved_tensors  # raises where one was changed in place
        call = _Call(q, k, v, offsets, key_offsets, ctx.causal, ctx.scale)
        on_device("the output", out, call.device)
        on_device("the sums", lse, call.device)
        need = ctx.needs_input_grad
        gq, gk, gv = call.backward(out, lse, grad_out, need[0], need[1] or need[2])
        return gq, gk if need[1] else None, gv if need[2] else None, None, None, None, None


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, offsets: Optional[torch.Tensor] = None,
              key_offsets: Optional[torch.Tensor] = None, causal: bool = True, scale: Optional[float] = None) -> torch.Tensor:
    """Softmax attention of ``q`` [rows, heads, dim] to ``k`` and ``v`` [key rows, kv_heads, dim], all bf16 or all fp16;
    out is of ``q``'s shape.  Head h reads the keys of head ``h // (heads // kv_heads)``; dim goes up to 128.

    ``offsets`` [documents + 1] (int32 or int64, on the same device) says where packed documents begin and end:
    queries see the keys of their own document only.  ``key_offsets`` does the same for rows of keys, where they are
    others than those of queries.  Without offsets all rows are one document; [batch, rows, heads, dim] tensors hold
    ``batch`` of them.  Offsets are held within the rows, and one that goes back counts as the one before it.

    ``causal``: of n queries and m keys, query i sees the keys j <= i + m - n; the last sees all.  A query that sees
    nothing (more queries than keys, or rows of no document) gives zeros, and gets and gives zero gradients.
    ``scale`` defaults to 1 / sqrt(dim).

    Differentiable once, to ``q``, ``k`` and ``v``.  Probabilities and their gradients are rounded to the operands' type on
    their way into the sums.  What is not finite in a key or value reaches queries of its own document that do not
    see it."""
    refuse_tangents(q, k, v)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (q, k, v)):
        return _Attention.apply(q, k, v, offsets, key_offsets, causal, scale)
    return _Call(q, k, v, offsets, key_offsets, causal, scale).forward(False)[0]
