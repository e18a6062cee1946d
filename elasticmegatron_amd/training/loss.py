"""Cross entropy over a large vocabulary, from hidden states and the output layer's weight.

    x_tv = hidden_t . weight_v,  lse_t = log sum_v exp(x_tv),  loss_t = lse_t - x_t,target_t

over the vocabulary rows v < ``vocab_size``.  The logits are never kept: the forward pass reduces them as
they are computed, and the backward pass computes them again in pieces of the vocabulary.  The weight is
one tensor or the consecutive vocabulary shards of tensor parallelism, as a state's bf16 arena holds them;
rows at and past ``vocab_size`` are the padding of the vocabulary and count nowhere.
"""

from __future__ import annotations

import ctypes
from typing import List, Optional, Sequence, Tuple, Union

import torch

from .. import _native
from ._common import dtype_code, on_device, refuse_tangents, run_on, workspace

Weight = Union[torch.Tensor, Sequence[torch.Tensor]]


def _rows(t: torch.Tensor):
    """``t`` [n, h] with unit column stride and rows that do not overlap; its sizes and strides."""
    size, stride = t.size(), t.stride()
    (n, h), (over, along) = size, stride
    if (h > 1 and along != 1) or (n > 1 and not h <= over <= 1 << 21):
        t = t.detach().contiguous()
        stride = t.stride()
    return t, size, stride


def _room_for(t: torch.Tensor) -> torch.Tensor:
    """A contiguous gradient of ``t``."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.size(), dtype=t.dtype, device=t.device)


def _table(values):
    return (ctypes.c_uint64 * len(values))(*values)


def _refuse(shards, device, dtype, h) -> None:
    """Raises for the first shard that is not as it has to be."""
    for i, w in enumerate(shards):
        on_device(f"weight shard {i}", w, device)
        if w.dtype != dtype:
            raise TypeError(f"weight shard {i} is {w.dtype}, hidden {dtype}")
        if w.dim() != 2 or w.shape[1] != h:
            raise ValueError(f"weight shard {i} is {tuple(w.shape)}: [rows, {h}] is wanted")


class _Call:
    """The checked arguments of one loss, and the record that the native calls take."""

    def __init__(self, hidden, weight, target, vocab_start, vocab_size, ignore_index):
        shards = [weight] if isinstance(weight, torch.Tensor) else list(weight)
        if not 1 <= len(shards) <= _native.EMRS_LOSS_MAX_SHARDS:
            raise ValueError(f"{len(shards)} vocabulary shards: 1 to {_native.EMRS_LOSS_MAX_SHARDS} are wanted")
        if not isinstance(hidden, torch.Tensor):
            raise TypeError("hidden is no tensor")
        refuse_tangents(hidden, shards)
        self.device = hidden.device
        on_device("hidden", hidden, self.device)
        on_device("target", target, self.device)
        code = dtype_code(hidden, "hidden", (torch.bfloat16, torch.float16))
        if target.dtype != torch.int64:
            raise TypeError(f"target is {target.dtype}: torch.int64 is wanted")
        if hidden.dim() < 1 or target.shape != hidden.shape[:-1]:
            raise ValueError(f"target {tuple(target.shape)} does not fit hidden {tuple(hidden.shape)}")
        h, device, dtype = hidden.size(-1), self.device, hidden.dtype
        laid, pointers, strides, rows, lie = [], [], [], [], []
        for w in shards:  # one by one only where something is wrong: this is most of a small loss's host time
            if not (isinstance(w, torch.Tensor) and w.dtype is dtype and w.device == device and w.dim() == 2):
                _refuse(shards, device, dtype, h)
            w, size, stride = _rows(w)
            if size[1] != h:
                _refuse(shards, device, dtype, h)
            laid.append(w), pointers.append(w.data_ptr()), strides.append(stride[0]), rows.append(size[0]), lie.append((size, stride))
        if vocab_start < 0:
            raise ValueError("vocab_start is negative")
        if vocab_size is None:
            vocab_size = vocab_start + sum(rows)
        if vocab_size < 0:
            raise ValueError("vocab_size is negative")
        self.hidden, size, stride = _rows(hidden if hidden.dim() == 2 else hidden.detach().reshape(-1, h))
        self.shards, self.shape, self.rows = laid, target.size(), sum(rows)
        self.target = target if target.dim() == 1 and target.is_contiguous() else target.reshape(-1).contiguous()
        self._lie, self._dtype, count = [*lie, (size, stride)], dtype, len(laid)
        self._tables = (_table([*pointers, *strides, *rows]),)
        at = ctypes.addressof(self._tables[0])
        self.record = _native.Loss(code, count, size[0], h, self.hidden.data_ptr(), stride[0], at, at + 8 * count, at + 16 * count,
                                   vocab_start, vocab_size, self.target.data_ptr(), ignore_index)

    def forward(self, with_loss: bool) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
        """``(lse, target logits, losses or None)``, the losses in the target's shape."""
        a, t = self.record, self.target.numel()
        out = torch.empty((2, t), dtype=torch.float32, device=self.device)
        loss = torch.empty(self.shape, dtype=torch.float32, device=self.device) if with_loss else None
        if t:
            at = out.data_ptr()
            a.lse, a.target_logit, a.loss = at, at + 4 * t, loss.data_ptr() if with_loss else None
            scratch = workspace(_native.loss_workspace(a, False), self.device)
            a.workspace, a.workspace_bytes = scratch.data_ptr(), scratch.numel()
            run_on(self.device, _native.loss_forward, a)
        lse, logit = out.unbind()
        return lse, logit, loss

    def again(self, hidden, target, shards) -> "_Call":
        """The same call on tensors that autograd hands back: at their own addresses, and checked anew where they
        do not lie as the first did."""
        a, device = self.record, self.device
        lie = [(t.size(), t.stride()) for t in shards if t.dtype is self._dtype and t.device == device]
        lie.append((hidden.size(), hidden.stride()))
        if not (lie == self._lie and hidden.dtype is self._dtype and hidden.device == device and target.dtype is torch.int64 and
                target.device == device and target.size() == (a.tokens,) and target.is_contiguous()):
            return _Call(hidden, shards, target, a.vocab_start, a.vocab_size, a.ignore_index)
        call = object.__new__(_Call)
        call.device, call.rows, call.hidden, call.target, call.shards = device, self.rows, hidden, target, shards
        call._tables = (_table([w.data_ptr() for w in shards]), *self._tables)
        a = call.record = _native.Loss.from_buffer_copy(a)
        a.hidden, a.target, a.weights = hidden.data_ptr(), target.data_ptr(), ctypes.addressof(call._tables[0])
        return call

    def release(self) -> None:
        self.hidden = self.target = self.shards = None

    def backward(self, lse, grad_loss, want_hidden: bool, want_weights: Sequence[bool]):
        a = self.record
        gh = _room_for(self.hidden) if want_hidden else None
        gw = [_room_for(w) if want else None for w, want in zip(self.shards, want_weights)]
        if not a.tokens or not self.rows:  # sums over nothing
            for g in (gh, *gw):
                if g is not None:
                    g.zero_()
            return gh, gw
        table = _table([0 if g is None else g.data_ptr() for g in gw])
        a.lse, a.grad_loss = lse.data_ptr(), grad_loss.data_ptr()
        a.grad_hidden = None if gh is None else gh.data_ptr()
        a.grad_weights = ctypes.addressof(table) if any(want_weights) else None
        scratch = workspace(_native.loss_workspace(a, True), self.device)
        a.workspace, a.workspace_bytes = scratch.data_ptr(), scratch.numel()
        run_on(self.device, _native.loss_backward, a)
        return gh, gw


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, target, vocab_size, ignore_index, *shards):
        call = _Call(hidden, shards, target, 0, vocab_size, ignore_index)
        lse, _, loss = call.forward(True)
        # What the kernels read: the inputs, or the copies that had to be made of them.  The graph alone keeps them.
        ctx.save_for_backward(call.hidden, call.target, lse, *call.shards)
        ctx.call, ctx.shape = call, hidden.size()
        call.release()
        return loss  # no view: users may scale it in place

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        hidden, target, lse, *shards = ctx.saved_tensors  # raises where one was changed in place
        call = ctx.call.again(hidden, target, shards)
        if not (lse.device == call.device and lse.is_contiguous()):
            on_device("lse", lse, call.device)
            lse = lse.contiguous()
        if grad_loss.dim() != 1 or grad_loss.dtype != torch.float32 or not grad_loss.is_contiguous():
            grad_loss = grad_loss.reshape(-1).to(torch.float32).contiguous()
        gh, gw = call.backward(lse, grad_loss, ctx.needs_input_grad[0], ctx.needs_input_grad[4:])
        return (gh if gh is None or len(ctx.shape) == 2 else gh.view(ctx.shape), None, None, None, *gw)


def linear_cross_entropy(hidden: torch.Tensor, weight: Weight, target: torch.Tensor, *, vocab_size: Optional[int] = None,
                         ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """The loss of every token of ``hidden`` [..., h] (bf16 or fp16) against ``weight`` (one tensor [V, h]
    or its consecutive vocabulary shards, of the same type) at ``target`` [...] (int64).

    ``vocab_size``: rows of the vocabulary that count; the rows from there on are padding, which may hold
    anything and gets zero gradients.  ``ignore_index``: tokens of this target have loss 0 and add nothing
    to any gradient, whatever their hidden state holds.  A target outside the vocabulary has loss inf.
    ``reduction``: ``"none"`` (fp32, the shape of ``target``), ``"sum"``, or ``"mean"`` over the tokens that
    count (NaN where none does).  Differentiable once, to ``hidden`` and to every shard.

    A token's gradient to ``hidden`` is as exact whatever the other tokens' loss counts for.  Gradients to the shards
    sum over tokens: what one adds there keeps fewer bits from 2^-27 of the largest |gradient of a loss| times
    |hidden| on, and nothing below 2^-38.
    """
    if reduction not in ("none", "sum", "mean"):
        raise ValueError(f"reduction {reduction!r}: 'none', 'sum' or 'mean' is wanted")
    shards = [weight] if isinstance(weight, torch.Tensor) else list(weight)
    refuse_tangents(hidden, shards)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (hidden, *shards)):
        loss = _LinearCrossEntropy.apply(hidden, target, vocab_size, ignore_index, *shards)
    else:
        loss = _Call(hidden, shards, target, 0, vocab_size, ignore_index).forward(True)[2]
    if reduction == "none":
        return loss
    total = loss.sum()
    return total if reduction == "sum" else total / (target != ignore_index).sum()


def vocab_statistics(hidden: torch.Tensor, weight: Weight, target: torch.Tensor, *, vocab_start: int = 0,
                     vocab_size: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(lse, target_logit)`` over the vocabulary rows that this process holds, the first of them row
    ``vocab_start`` of the vocabulary: fp32, the shape of ``target``.  Where the target's row is elsewhere,
    ``target_logit`` is -inf; where no row counts, so is ``lse``."""
    lse, logit, _ = _Call(hidden, weight, target, vocab_start, vocab_size, -100).forward(False)
    return lse.view(target.shape), logit.view(target.shape)


def merge_vocab_statistics(lse: torch.Tensor, target_logit: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(lse, target_logit)`` of the whole vocabulary from those of every process, stacked along dim 0.
    The loss is their difference; the merged ``lse`` is what :func:`vocab_gradients` takes."""
    return torch.logsumexp(lse, 0), target_logit.amax(0)


def vocab_gradients(hidden: torch.Tensor, weight: Weight, target: torch.Tensor, lse: torch.Tensor, grad_loss: torch.Tensor, *,
                    vocab_start: int = 0, vocab_size: Optional[int] = None,
                    ignore_index: int = -100) -> Tuple[torch.Tensor, List[torch.Tensor]]:
    """``(grad_hidden, grad_weights)`` from the rows that this process holds: its share of the gradient to
    ``hidden`` (the whole is the sum over the processes) and the gradients of its own shards.

    ``lse`` is of the whole vocabulary; ``grad_loss`` is the loss's gradient for each token."""
    refuse_tangents(lse, grad_loss)
    call = _Call(hidden, weight, target, vocab_start, vocab_size, ignore_index)
    for what, t in (("lse", lse), ("grad_loss", grad_loss)):
        on_device(what, t, call.device)
        if t.shape != target.shape:
            raise ValueError(f"{what} {tuple(t.shape)} does not fit target {tuple(target.shape)}")
    lse, grad_loss = (t.detach().reshape(-1).to(torch.float32).contiguous() for t in (lse, grad_loss))
    gh, gw = call.backward(lse, grad_loss, True, [True] * len(call.shards))
    return gh.view(hidden.shape), gw
