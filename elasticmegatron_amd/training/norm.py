"""The norm before a block, and what joins the block behind it to the residual stream.

    stream = residual_scale residual + gate n(branch),  normed = stream / rms(stream) weight

with n(b) = b / rms(b) branch_weight, or b itself, and rms(x) = sqrt(mean x^2 + eps) over a token's channels.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from .. import _native
from ._common import DTYPE_CODES, dtype_code, lies, on_device, refuse_tangents, run_on, workspace


def _rows(t: torch.Tensor, h: int):
    """``t`` as rows [n, h] with unit column stride that do not overlap, and the stride between them."""
    if t.dim() != 2:
        t = t.detach().reshape(-1, h)
    (n, _), (over, along) = t.size(), t.stride()
    if n <= 1 and (along == 1 or h == 1):
        return t, h
    if (along != 1 and h > 1) or over < h:
        t = t.detach().contiguous()
        over = h
    return t, over


def _vector(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.detach().contiguous()


def _check(residual, branch, gate, branch_weight, weight) -> int:
    """Raises for the first argument that is not as it has to be; the kind of gate."""
    if not isinstance(residual, torch.Tensor):
        raise TypeError("residual is no tensor")
    device = residual.device
    on_device("residual", residual, device)
    dtype_code(residual, "residual")
    if residual.dim() < 1 or not 1 <= residual.shape[-1] <= _native.EMRS_NORM_MAX_HIDDEN:
        raise ValueError(f"residual is {tuple(residual.shape)}: [..., h] with h from 1 to {_native.EMRS_NORM_MAX_HIDDEN} is wanted")
    size, first = residual.size(), None
    vector = size[-1:]
    for what, t in (("branch", branch), ("weight", weight), ("branch_weight", branch_weight), ("gate", gate)):
        if t is None:
            continue
        if not (isinstance(t, torch.Tensor) and t.device == device):
            on_device(what, t, device)
        first = first or (what, t.dtype)
        if t.dtype != first[1] or t.dtype not in (torch.bfloat16, torch.float16):
            dtype_code(t, what, (torch.bfloat16, torch.float16))
            raise TypeError(f"{what} is {t.dtype}, {first[0]} {first[1]}")
        if what == "branch" and t.size() != size:
            raise ValueError(f"branch {tuple(t.shape)} does not fit residual {tuple(size)}")
        if what in ("weight", "branch_weight") and t.size() != vector:
            raise ValueError(f"{what} is {tuple(t.shape)}: [{size[-1]}] is wanted")
    if first is None:
        raise ValueError("neither a branch nor a weight is given")
    if residual.dtype not in (torch.float32, first[1]):
        raise TypeError(f"residual is {residual.dtype}: torch.float32 or {first[0]}'s {first[1]} is wanted")
    if gate is None:
        return _native.EMRS_NORM_GATE_NONE
    if branch is None:
        raise ValueError("a gate without a branch")
    if gate.size() == size:
        return _native.EMRS_NORM_GATE_TOKEN
    if gate.size() != vector:
        raise ValueError(f"gate is {tuple(gate.shape)}: [{size[-1]}] or branch's {tuple(size)} is wanted")
    return _native.EMRS_NORM_GATE_CHANNEL


def _address(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _record(residual, branch, gate, branch_weight, weight, scale, eps):
    """The record with what both passes read, and those tensors: rows and vectors as the kernels take them."""
    kind = _check(residual, branch, gate, branch_weight, weight)
    h = residual.shape[-1]
    a = _native.Norm(DTYPE_CODES[(weight if branch is None else branch).dtype], DTYPE_CODES[residual.dtype], kind, 0, residual.numel() // h, h)
    a.residual_scale, a.eps = scale, eps
    if branch is not None:
        branch, a.branch_stride = _rows(branch, h)
        a.branch = branch.data_ptr()
        if gate is not None:
            gate, a.gate_stride = _rows(gate, h) if kind == _native.EMRS_NORM_GATE_TOKEN else (_vector(gate), h)
            a.gate = gate.data_ptr()
        if branch_weight is not None:
            branch_weight = _vector(branch_weight)
            a.branch_weight = branch_weight.data_ptr()
    if weight is not None:
        weight = _vector(weight)
        a.weight = weight.data_ptr()
    return a, (branch, gate, branch_weight, weight)


def _forward(residual, branch, gate, branch_weight, weight, scale, eps, statistics):
    """``(stream or None, normed or None, statistics or None, the record, the tensors that it points to)``."""
    a, read = _record(residual, branch, gate, branch_weight, weight, scale, eps)
    size, device, tokens = residual.size(), residual.device, a.tokens
    stream = None if branch is None else torch.empty(size, dtype=residual.dtype, device=device)
    normed = None if weight is None else torch.empty(size, dtype=weight.dtype, device=device)
    rms = torch.empty((2, tokens), dtype=torch.float32, device=device) if statistics else None
    if tokens:
        rows, a.residual_stride = _rows(residual, a.hidden)
        a.residual, a.stream, a.normed = rows.data_ptr(), _address(stream), _address(normed)
        if statistics:
            a.stream_rms = rms.data_ptr()
            a.branch_rms = a.stream_rms + 4 * tokens
        run_on(device, _native.norm_forward, a)
    return stream, normed, rms, a, read


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, branch, gate, branch_weight, weight, scale, eps):
        stream, normed, rms, a, read = _forward(residual, branch, gate, branch_weight, weight, scale, eps, True)
        # What the kernels read: the inputs, or the copies that had to be made of them.
        saved = (residual if stream is None else stream, *read, rms)
        ctx.save_for_backward(*saved)
        ctx.record, ctx.lies = a, lies(*saved)
        ctx.likes = [None if t is None else t.size() for t in (residual, branch, gate, branch_weight, weight)]
        ctx.set_materialize_grads(False)
        if stream is None:
            return normed
        return stream if normed is None else (stream, normed)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        saved = ctx.saved_tensors  # raises where one was changed in place
        stream, branch, gate, branch_weight, weight, rms = saved
        a, likes, need = ctx.record, ctx.likes, ctx.needs_input_grad
        grad_stream = None if branch is None else grads[0]
        grad_normed = None if weight is None else grads[-1]
        if grad_stream is None and grad_normed is None:
            return (None,) * 7
        device, shape, h = stream.device, likes[0], likes[0][-1]
        if lies(*saved) == ctx.lies:
            a = _native.Norm.from_buffer_copy(a)
        else:  # hooks on saved tensors handed back others
            on_device("the statistics", rms, device)
            if rms.size() != (2, a.tokens) or rms.dtype != torch.float32:
                raise ValueError("the saved statistics are not those of the forward pass")
            rms = rms.contiguous()
            back = [None if t is None else t.reshape(like) for t, like in zip((stream, branch, gate, branch_weight, weight), likes)]
            a, (branch, gate, branch_weight, weight) = _record(*back, a.residual_scale, a.eps)
            stream = back[0]
        tokens, dtype = a.tokens, (weight if branch is None else branch).dtype
        # With nothing between them, residual and branch have one gradient, as those of a sum have.
        one = need[0] and need[1] and gate is None and branch_weight is None and a.residual_scale == 1.0 and stream.dtype == dtype
        sums = need[3] or (need[4] and grad_normed is not None) or (need[2] and a.gate_kind == _native.EMRS_NORM_GATE_CHANNEL)
        gr = torch.empty(shape, dtype=stream.dtype, device=device) if need[0] else None
        gb = torch.empty(shape, dtype=dtype, device=device) if need[1] and not one else None
        gg = torch.empty(likes[2], dtype=dtype, device=device) if need[2] else None
        gbw = torch.empty(likes[3], dtype=dtype, device=device) if need[3] else None
        gw = torch.empty(likes[4], dtype=dtype, device=device) if need[4] and grad_normed is not None else None
        if tokens:
            keep = []
            a.stream = a.grad_stream = a.grad_normed = a.normed = None
            if grad_normed is not None:
                rows, a.stream_stride = _rows(stream, h)
                if not (grad_normed.dtype is dtype and grad_normed.is_contiguous()):
                    grad_normed = grad_normed.to(dtype).contiguous()
                keep += [rows, grad_normed]
                a.stream, a.grad_normed = rows.data_ptr(), grad_normed.data_ptr()
            if grad_stream is not None:
                if not (grad_stream.dtype is stream.dtype and grad_stream.is_contiguous()):
                    grad_stream = grad_stream.to(stream.dtype).contiguous()
                a.grad_stream = grad_stream.data_ptr()
            a.stream_rms = rms.data_ptr()
            a.branch_rms = a.stream_rms + 4 * tokens
            a.grad_residual, a.grad_branch, a.grad_gate = _address(gr), _address(gb), _address(gg)
            a.grad_branch_weight, a.grad_weight = _address(gbw), _address(gw)
            if sums:
                scratch = workspace(_native.norm_workspace(a), device)
                a.workspace, a.workspace_bytes = scratch.data_ptr(), scratch.numel()
            run_on(device, _native.norm_backward, a)
        else:
            for g in (gr, gb, gg, gbw, gw):
                if g is not None:
                    g.zero_()
        return gr, gr if one else gb, gg, gbw, gw, None, None


def _call(residual, branch, gate, branch_weight, weight, scale, eps):
    tensors = (residual, branch, gate, branch_weight, weight)
    refuse_tangents(*tensors)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors):
        return _ResidualNorm.apply(*tensors, scale, eps)
    stream, normed = _forward(*tensors, scale, eps, False)[:2]
    if stream is None:
        return normed
    return stream if normed is None else (stream, normed)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-5) -> torch.Tensor:
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension of ``x`` [..., h], of ``weight``'s type.

    ``weight`` [h] is bf16 or fp16, ``x`` of its type or fp32, h up to 16384.  Differentiable once, to both."""
    if weight is None:
        raise TypeError("weight is no tensor")
    return _call(x, None, None, None, weight, 1.0, eps)


def residual_norm(residual: torch.Tensor, branch: torch.Tensor, weight: Optional[torch.Tensor] = None, *,
                  branch_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0,
                  eps: float = 1e-5) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``(stream, normed)``: what a block's output ``branch`` [..., h] makes of the ``residual`` stream, and the norm
    that the next block reads, in one pass:

        stream = residual_scale residual + gate n(branch)       (``gate`` given; else n(branch))
        n(b) = b / sqrt(mean(b^2) + eps) branch_weight          (``branch_weight`` given; else b)
        normed = stream / sqrt(mean(stream^2) + eps) weight     (``weight`` given; else only stream is returned)

    ``branch``, the weights [h] and the gate are bf16 or fp16, of one type, and so is ``normed``; ``residual``, and with
    it ``stream``, may be fp32.  ``gate`` is [h], or of ``branch``'s shape.  h goes up to 16384.  Differentiable once,
    to all of them; where nothing stands between a sum and its two terms, these share one gradient tensor."""
    if branch is None:
        raise TypeError("branch is no tensor")
    return _call(residual, branch, gate, branch_weight, weight, float(residual_scale), eps)
