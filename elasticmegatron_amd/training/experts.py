"""Products of every token with its expert's weight matrix, over experts of ragged sizes.

    y_t = W_e x_t   for the rows t of expert e,  grad_x_t = W_e^T grad_y_t,  grad_W_e = sum_t grad_y_t x_t^T

Rows lie by expert, as a dispatcher leaves them; how many each expert has is on the device and stays there.
"""

from __future__ import annotations

import ctypes
from typing import Sequence, Union

import torch

from .. import _native
from ._common import DTYPE_CODES, dtype_code, lies, on_device, refuse_tangents, run_on, workspace

Weights = Union[torch.Tensor, Sequence[torch.Tensor]]


def _rows(t: torch.Tensor):
    """``t`` [n, k] with unit column stride and rows that do not overlap, and the stride between them."""
    (n, k), (over, along) = t.size(), t.stride()
    if (k > 1 and along != 1) or (n > 1 and not k <= over <= 1 << 21):
        t = t.detach().contiguous()
        over = k
    return t, over if n > 1 else k


def _same_rows(weights):
    """The same of every expert's matrix, all with one stride: tensors, addresses, stride."""
    if len(weights) == 1 and weights[0].dim() == 3:
        t = weights[0]
        (_, n, k), (_, over, along) = t.size(), t.stride()
        if (k > 1 and along != 1) or (n > 1 and not k <= over <= 1 << 21):
            t = t.detach().contiguous()
            over = k
        base, step = t.data_ptr(), t.stride(0) * t.element_size()
        return [t], [base + i * step for i in range(t.shape[0])], over if n > 1 else k
    n, k = weights[0].size()
    first = weights[0].stride()
    if (first[1] == 1 or k == 1) and (n == 1 or k <= first[0] <= 1 << 21) and all(w.stride() == first for w in weights):
        return weights, [w.data_ptr() for w in weights], first[0] if n > 1 else k
    laid = [w.detach().contiguous() for w in weights]
    return laid, [w.data_ptr() for w in laid], k


def _table(values):
    return (ctypes.c_uint64 * len(values))(*values)


def _refuse(x, counts, weights) -> None:
    """Raises for the first argument that is not as it has to be."""
    if not isinstance(x, torch.Tensor):
        raise TypeError("x is no tensor")
    device = x.device
    on_device("x", x, device)
    dtype_code(x, "x", (torch.bfloat16, torch.float16))
    if x.dim() != 2:
        raise ValueError(f"x is {tuple(x.shape)}: [rows, n_in] is wanted")
    on_device("counts", counts, device)
    if counts.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"counts is {counts.dtype}: torch.int32 or torch.int64 is wanted")
    for i, w in enumerate(weights):
        on_device(f"weight {i}", w, device)
        if w.dtype != x.dtype:
            raise TypeError(f"weight {i} is {w.dtype}, x {x.dtype}")
        if w.dim() != (3 if len(weights) == 1 and w.dim() == 3 else 2):
            raise ValueError(f"weight {i} has {w.dim()} dimensions: a matrix for every expert, or all of them stacked, is wanted")
        if w.shape[-1] != x.shape[1] or w.shape[-2:] != weights[0].shape[-2:]:
            raise ValueError(f"weight {i} is {tuple(w.shape[-2:])}: [{weights[0].shape[-2]}, {x.shape[1]}] is wanted")


class _Call:
    """The checked arguments of one product, and the record that the native calls take.

    ``weights``: one tensor [experts, n_out, n_in], or one matrix [n_out, n_in] for every expert."""

    def __init__(self, x, counts, weights):
        stacked = len(weights) == 1 and isinstance(weights[0], torch.Tensor) and weights[0].dim() == 3
        if not (isinstance(x, torch.Tensor) and x.is_cuda and x.dtype in (torch.bfloat16, torch.float16) and x.dim() == 2 and
                isinstance(weights[0], torch.Tensor)):
            _refuse(x, counts, weights)
        device, dtype, size = x.device, x.dtype, weights[0].size()
        for w in weights:  # one by one only where something is wrong
            if not (isinstance(w, torch.Tensor) and w.dtype is dtype and w.device == device and w.size() == size):
                _refuse(x, counts, weights)
        if not (isinstance(counts, torch.Tensor) and counts.device == device and counts.dtype in (torch.int32, torch.int64) and
                len(size) == (3 if stacked else 2) and size[-1] == x.size(1)):
            _refuse(x, counts, weights)
        experts = size[0] if stacked else len(weights)
        if not 1 <= experts <= _native.EMRS_EXPERTS_MAX:
            raise ValueError(f"{experts} experts: 1 to {_native.EMRS_EXPERTS_MAX} are wanted")
        if counts.shape != (experts,):
            raise ValueError(f"counts is {tuple(counts.shape)}: [{experts}] is wanted")
        n_out, n_in = size[-2:]
        if not n_in or not n_out:
            raise ValueError(f"weights of {n_out} x {n_in}: no side may be 0")
        self.x, x_stride = _rows(x)
        self.counts = counts if counts.is_contiguous() else counts.contiguous()
        self.weights, addresses, weight_stride = _same_rows(weights)
        self.device, self.dtype, self.experts, self.shape, self.size, self.n_out = device, dtype, experts, x.size(), size, n_out
        self._table = _table(addresses)
        self.record = _native.Experts(DTYPE_CODES[dtype], experts, x.shape[0], n_in, n_out, self.counts.data_ptr(), counts.element_size(), 0,
                                      self.x.data_ptr(), x_stride, ctypes.addressof(self._table), weight_stride)

    def again(self, x, counts, weights) -> "_Call":
        """The same call on tensors that autograd hands back: itself where they are where they were, and checked anew where not."""
        if lies(x, counts, *weights) != self.lies:
            return _Call(x, counts, weights)
        call = object.__new__(_Call)
        call.__dict__.update(self.__dict__)
        call.record = _native.Experts.from_buffer_copy(self.record)
        return call

    def release(self) -> None:
        """What is left knows where its tensors were, and does not keep them."""
        self.lies = lies(self.x, self.counts, *self.weights)
        self.x = self.counts = self.weights = None

    def _run(self, call, backward):
        a = self.record
        size = _native.experts_workspace(a, backward)
        if size:
            scratch = workspace(size, self.device)
            a.workspace, a.workspace_bytes = scratch.data_ptr(), scratch.numel()
        run_on(self.device, call, a)

    def forward(self) -> torch.Tensor:
        y = torch.empty((self.shape[0], self.n_out), dtype=self.dtype, device=self.device)
        if self.shape[0]:
            self.record.y = y.data_ptr()
            self._run(_native.experts_forward, False)
        return y

    def backward(self, grad_y, want_x, want_weights):
        """``(grad_x, gradients of the weights)``; each may be None."""
        a = self.record
        if grad_y.size() != (self.shape[0], self.n_out):
            raise ValueError(f"a gradient of {tuple(grad_y.shape)} for {self.shape[0]} rows of {self.n_out}")
        rows, a.grad_y_stride = _rows(grad_y if grad_y.dtype is self.dtype else grad_y.to(self.dtype))
        a.grad_y, a.y = rows.data_ptr(), None
        gx = torch.empty(self.shape, dtype=self.dtype, device=self.device) if want_x else None
        gw = None
        a.grad_x = None if gx is None else gx.data_ptr()
        if want_weights:
            if len(self.size) == 3:
                gw = [torch.empty(self.size, dtype=self.dtype, device=self.device)]
                step = gw[0].element_size() * self.n_out * self.shape[1]
                table = _table([gw[0].data_ptr() + i * step for i in range(self.experts)])
            else:
                # One allocation: that of each for itself is most of a small call's host time.
                gw = torch.empty((self.experts, *self.size), dtype=self.dtype, device=self.device).unbind(0)
                table = _table([g.data_ptr() for g in gw])
            a.grad_weights = ctypes.addressof(table)
        if gw or (want_x and self.shape[0]):
            self._run(_native.experts_backward, True)
        return gx, gw


class _ExpertLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, counts, *weights):
        call = _Call(x, counts, weights)
        y = call.forward()
        # What the kernels read: the inputs, or the copies that had to be made of them.  The graph alone keeps them.
        ctx.save_for_backward(call.x, call.counts, *call.weights)
        ctx.call = call
        call.release()
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y):
        x, counts, *weights = ctx.saved_tensors  # raises where one was changed in place
        need = ctx.needs_input_grad
        gx, gw = ctx.call.again(x, counts, weights).backward(grad_y, need[0], any(need[2:]))
        return (gx, None, *((g if want else None for g, want in zip(gw, need[2:])) if gw else [None] * len(weights)))


def expert_linear(x: torch.Tensor, weights: Weights, counts: torch.Tensor) -> torch.Tensor:
    """``y`` [rows, n_out] with ``y[t] = weights[e] @ x[t]`` for the rows t of expert e.

    ``x`` [rows, n_in] (bf16 or fp16) has its rows by expert: the first ``counts[0]`` are expert 0's, and so on.
    ``counts`` [experts] (int32 or int64) is on ``x``'s device, and nothing waits for it.  Rows behind the last
    expert's belong to none: they give zeros, and get zero gradients.  Counts below 0 count as 0, and where they sum to
    more than there are rows, rows end first.

    ``weights``: one matrix [n_out, n_in] for every expert (1 to 256), as a state holds them, or a tensor
    [experts, n_out, n_in]; of ``x``'s type.  Differentiable once, to ``x`` and to every matrix (whose gradients share
    one allocation); an expert without rows has a gradient of zeros.  Rows that lie off 16 bytes, or whose length is no multiple of 8, are copied first."""
    weights = [weights] if isinstance(weights, torch.Tensor) else list(weights)
    if not weights:
        raise ValueError("no weights are given")
    refuse_tangents(x, weights)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (x, *weights)):
        return _ExpertLinear.apply(x, counts, *weights)
    return _Call(x, counts, weights).forward()
