"""Attention within documents, with its gradients.

    s = scale q . k  over the keys that a query sees,  out = softmax(s) v

The probabilities are never kept: the backward pass computes them again from the sums that forward leaves.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from .. import _native
from ._common import DTYPE_CODES, dtype_code, lies, on_device, refuse_tangents, run_on, workspace


def _operand(t: torch.Tensor):
    """``t`` [rows, heads, dim] with unit stride along dim, and its other strides."""
    if t.stride(2) != 1 and t.shape[2] > 1:
        t = t.detach().contiguous()
    (rows, heads, dim), (row, head, _) = t.size(), t.stride()
    return t, (row if rows > 1 else heads * dim, head if heads > 1 else dim)


def _refuse(q, k, v, offsets, key_offsets) -> None:
    """Raises for the first argument that is not as it has to be."""
    if not isinstance(q, torch.Tensor):
        raise TypeError("q is no tensor")
    device = q.device
    for what, t in (("q", q), ("k", k), ("v", v)):
        on_device(what, t, device)
        dtype_code(t, what, (torch.bfloat16, torch.float16))
        if t.dtype != q.dtype:
            raise TypeError(f"{what} is {t.dtype}, q {q.dtype}")
        if t.dim() != q.dim() or t.dim() not in (3, 4):
            raise ValueError(f"{what} has {t.dim()} dimensions: [rows, heads, dim], or [batch, rows, heads, dim] for all three, is wanted")
    if k.shape != v.shape or k.shape[-1] != q.shape[-1] or (q.dim() == 4 and k.shape[0] != q.shape[0]):
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not fit q {tuple(q.shape)}")
    if offsets is None:
        if key_offsets is not None:
            raise ValueError("key_offsets without offsets")
        return
    if q.dim() == 4:
        raise ValueError("offsets are of packed documents: [rows, heads, dim] is wanted")
    for what, t in (("offsets", offsets), ("key_offsets", offsets if key_offsets is None else key_offsets)):
        on_device(what, t, device)
        if t.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{what} is {t.dtype}: torch.int32 or torch.int64 is wanted")
    if key_offsets is None and k.shape[0] != q.shape[0]:
        raise ValueError(f"{k.shape[0]} rows of keys for {q.shape[0]} of queries: key_offsets are wanted")
    others = offsets if key_offsets is None else key_offsets
    if offsets.dim() != 1 or offsets.shape[0] < 2 or others.shape != offsets.shape or others.dtype != offsets.dtype:
        raise ValueError(f"offsets {tuple(offsets.shape)} and key_offsets {tuple(others.shape)}: [documents + 1] of one type are wanted")


class _Call:
    """The checked arguments of one attention, and the record that the native calls take."""

    def __init__(self, q, k, v, offsets, key_offsets, causal, scale):
        _refuse(q, k, v, offsets, key_offsets)
        self.device, self.dtype, self.shape, self.key_shape = q.device, q.dtype, q.size(), k.size()
        heads, dim, kv_heads = *self.shape[-2:], self.key_shape[-2]
        if not heads or not kv_heads or heads % kv_heads:
            raise ValueError(f"{heads} heads and {kv_heads} of keys: a multiple is wanted")
        if not 1 <= dim <= _native.EMRS_ATTENTION_MAX_DIM:
            raise ValueError(f"heads of {dim} elements: 1 to {_native.EMRS_ATTENTION_MAX_DIM} are wanted")
        if scale is None:
            scale = 1 / math.sqrt(dim)
        if not 0 < scale < math.inf:
            raise ValueError(f"scale is {scale}: a positive number is wanted")
        a = self.record = _native.Attention()
        (q, a.q_strides[:]), (k, a.k_strides[:]), (v, a.v_strides[:]) = (_operand(t if t.dim() == 3 else t.detach().flatten(0, 1)) for t in (q, k, v))
        a.dtype, a.causal, a.heads, a.kv_heads, a.dim = DTYPE_CODES[self.dtype], 1 if causal else 0, heads, kv_heads, dim
        a.rows, a.key_rows, a.scale = q.shape[0], k.shape[0], scale
        a.documents = max(1, self.shape[0]) if len(self.shape) == 4 else 1
        if offsets is not None:
            others = offsets if key_offsets is None else key_offsets
            offsets = offsets.contiguous()
            key_offsets = offsets if others is offsets else others.contiguous()
            a.offsets, a.key_offsets, a.offset_bytes, a.documents = offsets.data_ptr(), key_offsets.data_ptr(), offsets.element_size(), offsets.shape[0] - 1
        self.read = (q, k, v, offsets, key_offsets)
        a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()

    def again(self, *read) -> "_Call":
        """The same call on tensors that autograd hands back: itself where they are where they were, and checked anew where not."""
        a = self.record
        if lies(*read) == self.lies:
            call = object.__new__(_Call)
            call.__dict__.update(self.__dict__)
            call.record = _native.Attention.from_buffer_copy(a)
            return call
        call = _Call(*read, a.causal, a.scale)
        b = call.record
        if (b.rows, b.key_rows, b.heads, b.kv_heads, b.dim) != (a.rows, a.key_rows, a.heads, a.kv_heads, a.dim):
            raise ValueError("the saved tensors are not those of the forward pass")
        b.documents, call.shape, call.key_shape = a.documents, self.shape, self.key_shape  # batches are saved as rows
        return call

    def release(self) -> None:
        """What is left knows where its tensors were, and does not keep them."""
        self.lies = lies(*self.read)
        self.read = None

    def _run(self, call, backward):
        a = self.record
        size = _native.attention_workspace(a, backward)
        if size:
            scratch = workspace(size, self.device)
            a.workspace, a.workspace_bytes = scratch.data_ptr(), scratch.numel()
        run_on(self.device, call, a)

    def forward(self, for_backward):
        """``(out, what its rounding left over, lse)``, the last two for the backward pass alone."""
        a = self.record
        out = torch.empty(self.shape, dtype=self.dtype, device=self.device)
        rest = lse = None
        if for_backward:
            rest = torch.empty(self.shape, dtype=self.dtype, device=self.device)
            lse = torch.empty((a.heads, a.rows), dtype=torch.float32, device=self.device)
        if a.rows:
            a.out = out.data_ptr()
            if for_backward:
                a.out_rest, a.lse = rest.data_ptr(), lse.data_ptr()
            self._run(_native.attention_forward, False)
        return out, rest, lse

    def backward(self, out, rest, lse, grad_out, want_q, want_kv):
        """Gradients of q, k and v; each may be None."""
        a, device = self.record, self.device
        for what, t, shape, dtype in (("output", out, self.shape, self.dtype), ("output's rest", rest, self.shape, self.dtype),
                                      ("sums", lse, (a.heads, a.rows), torch.float32), ("gradient", grad_out, self.shape, None)):
            if t.device != device or t.size() != shape or not (dtype is None or t.dtype is dtype):
                raise ValueError(f"the {what} is {tuple(t.shape)}, {t.dtype}, on {t.device}: not what the forward pass made")
        gq = torch.empty(self.shape, dtype=self.dtype, device=device) if want_q else None
        gk = gv = None
        if want_kv:
            gk, gv = (torch.empty(self.key_shape, dtype=self.dtype, device=device) for _ in range(2))
        if grad_out.dtype is not self.dtype:
            grad_out = grad_out.to(self.dtype)
        grad, a.grad_out_strides[:] = _operand(grad_out if grad_out.dim() == 3 else grad_out.flatten(0, 1))
        out, rest, lse = out.contiguous(), rest.contiguous(), lse.contiguous()
        a.out, a.out_rest, a.lse, a.grad_out = out.data_ptr(), rest.data_ptr(), lse.data_ptr(), grad.data_ptr()
        a.grad_q = None if gq is None else gq.data_ptr()
        a.grad_k, a.grad_v = (gk.data_ptr(), gv.data_ptr()) if want_kv else (None, None)
        if (want_q and a.rows) or (want_kv and a.key_rows):
            self._run(_native.attention_backward, True)
        return gq, gk, gv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, offsets, key_offsets, causal, scale):
        call = _Call(q, k, v, offsets, key_offsets, causal, scale)
        out, rest, lse = call.forward(True)
        # What the kernels read: the inputs, or the copies that had to be made of them.  The graph alone keeps them.
        ctx.save_for_backward(*call.read, out, rest, lse)
        ctx.call = call
        call.release()
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        *read, out, rest, lse = ctx.saved_tensors  # raises where one was changed in place
        need = ctx.needs_input_grad
        gq, gk, gv = ctx.call.again(*read).backward(out, rest, lse, grad_out, need[0], need[1] or need[2])
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
    see it, and what is not finite in a query or its gradient the gradients of keys there that it does not see."""
    refuse_tangents(q, k, v)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (q, k, v)):
        return _Attention.apply(q, k, v, offsets, key_offsets, causal, scale)
    return _Call(q, k, v, offsets, key_offsets, causal, scale).forward(False)[0]
