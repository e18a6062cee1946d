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
    if t.is_contiguous():
        return t, h
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


def _refuse(residual, branch, gate, branch_weight, weight) -> None:
    """Raises for the first argument that is not as it has to be."""
    if not isinstance(residual, torch.Tensor):
        raise TypeError("residual is no tensor")
    device = residual.device
    on_device("residual", residual, device)
    dtype_code(residual, "residual")
    if residual.dim() < 1 or not 1 <= residual.shape[-1] <= _native.EMRS_NORM_MAX_HIDDEN:
        raise ValueError(f"residual is {tuple(residual.shape)}: [..., h] with h from 1 to {_native.EMRS_NORM_MAX_HIDDEN} is wanted")
    size, first = residual.size(), None
    for what, t in (("branch", branch), ("weight", weight), ("branch_weight", branch_weight), ("gate", gate)):
        if t is None:
            continue
        on_device(what, t, device)
        first = first or (what, t.dtype)
        dtype_code(t, what, (torch.bfloat16, torch.float16))
        if t.dtype != first[1]:
            raise TypeError(f"{what} is {t.dtype}, {first[0]} {first[1]}")
        if what == "branch" and t.size() != size:
            raise ValueError(f"branch {tuple(t.shape)} does not fit residual {tuple(size)}")
        if what in ("weight", "branch_weight") and t.size() != size[-1:]:
            raise ValueError(f"{what} is {tuple(t.shape)}: [{size[-1]}] is wanted")
    if first is None:
        raise ValueError("neither a branch nor a weight is given")
    if residual.dtype not in (torch.float32, first[1]):
        raise TypeError(f"residual is {residual.dtype}: torch.float32 or {first[0]}'s {first[1]} is wanted")
    if gate is not None and branch is None:
        raise ValueError("a gate without a branch")
    if gate is not None and gate.size() not in (size, size[-1:]):
        raise ValueError(f"gate is {tuple(gate.shape)}: [{size[-1]}] or branch's {tuple(size)} is wanted")


_HALVES = (torch.bfloat16, torch.float16)


def _fits(t, device, dtype, size) -> bool:
    return isinstance(t, torch.Tensor) and t.dtype is dtype and t.device == device and t.size() == size


def _record(residual, branch, gate, branch_weight, weight, scale, eps):
    """The record with what both passes read, and those tensors: rows and vectors as the kernels take them.

    Small calls are host time for the most part: what is right is found at once, and what is not, one by one."""
    model = weight if branch is None else branch
    if not (isinstance(residual, torch.Tensor) and isinstance(model, torch.Tensor) and residual.is_cuda and residual.dim()):
        _refuse(residual, branch, gate, branch_weight, weight)
    device, size, dtype = residual.device, residual.size(), model.dtype
    h, vector = size[-1], size[-1:]
    if not (dtype in _HALVES and (residual.dtype is dtype or residual.dtype is torch.float32) and 1 <= h <= _native.EMRS_NORM_MAX_HIDDEN and
            (branch is None or _fits(branch, device, dtype, size)) and (weight is None or _fits(weight, device, dtype, vector)) and
            (branch_weight is None or _fits(branch_weight, device, dtype, vector)) and
            (gate is None or branch is not None and (_fits(gate, device, dtype, size) or _fits(gate, device, dtype, vector)))):
        _refuse(residual, branch, gate, branch_weight, weight)
    a = _native.Norm(DTYPE_CODES[dtype], DTYPE_CODES[residual.dtype], _native.EMRS_NORM_GATE_NONE, 0, residual.numel() // h, h)
    a.residual_scale, a.eps = scale, eps
    if branch is not None:
        branch, a.branch_stride = _rows(branch, h)
        a.branch = branch.data_ptr()
        if gate is not None:
            if gate.size() == size:
                a.gate_kind, (gate, a.gate_stride) = _native.EMRS_NORM_GATE_TOKEN, _rows(gate, h)
            else:
                a.gate_kind, gate = _native.EMRS_NORM_GATE_CHANNEL, _vector(gate)
            a.gate = gate.data_ptr()
        if branch_weight is not None:
            branch_weight = _vector(branch_weight)
            a.branch_weight = branch_weight.data_ptr()
    if weight is not None:
        weight = _vector(weight)
        a.weight = weight.data_ptr()
    return a, branch, gate, branch_weight, weight


def _forward(residual, branch, gate, branch_weight, weight, scale, eps, statistics):
    """``(stream or None, normed or None, statistics or None, the record, what backward reads of the others)``."""
    a, rows, gate, branch_weight, weight = _record(residual, branch, gate, branch_weight, weight, scale, eps)
    size, device, tokens = residual.size(), residual.device, a.tokens
    stream = normed = rms = None
    if branch is not None:
        stream = torch.empty(size, dtype=residual.dtype, device=device)
        a.stream = stream.data_ptr()
    if weight is not None:
        normed = torch.empty(size, dtype=weight.dtype, device=device)
        a.normed = normed.data_ptr()
    if statistics:
        rms = torch.empty((2, tokens), dtype=torch.float32, device=device)
        a.stream_rms = at = rms.data_ptr()
        a.branch_rms = at + 4 * tokens
    if tokens:
        flat, a.residual_stride = _rows(residual, a.hidden)
        a.residual = flat.data_ptr()
        run_on(device, _native.norm_forward, a)
    # With nothing between the branch and the stream, backward does not read it, and the graph does not keep it.
    if gate is None and branch_weight is None:
        rows = a.branch = None
    return stream, normed, rms, a, (rows, gate, branch_weight, weight)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, branch, gate, branch_weight, weight, scale, eps):
        # Only a norm has statistics, and only the gradient of that before the next block reads the stream.
        normalises = weight is not None or branch_weight is not None
        stream, normed, rms, a, read = _forward(residual, branch, gate, branch_weight, weight, scale, eps, normalises)
        # What the kernels read: the inputs, or the copies that had to be made of them.
        saved = [t for t in ((residual if stream is None else stream) if weight is not None else None, rms, *read) if t is not None]
        ctx.save_for_backward(*saved)
        ctx.record, ctx.lies, ctx.has, ctx.size, ctx.device = a, lies(*saved), [t is not None for t in read], residual.size(), residual.device
        ctx.set_materialize_grads(False)
        if stream is None:
            return normed
        return stream if normed is None else (stream, normed)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        saved = ctx.saved_tensors  # raises where one was changed in place
        need, size, has = ctx.needs_input_grad, ctx.size, ctx.has
        # Without a branch there is no stream to be differentiated to, without a weight no norm.
        grad_normed = grads[-1] if has[3] else None
        grad_stream = grads[0] if len(grads) > 1 or not has[3] else None
        if grad_stream is None and grad_normed is None:
            return (None,) * 7
        if lies(*saved) == ctx.lies:
            a = _native.Norm.from_buffer_copy(ctx.record)
        else:
            a, saved = _again(ctx, saved)
        device, tokens, h, dtype, stream_dtype = ctx.device, a.tokens, size[-1], _DTYPES[a.dtype], _DTYPES[a.residual_dtype]
        out = torch.empty
        # With nothing between them, residual and branch have one gradient, as those of a sum have.
        one = need[0] and need[1] and not has[0] and a.residual_scale == 1.0 and stream_dtype is dtype
        gr = out(size, dtype=stream_dtype, device=device) if need[0] else None
        gb = out(size, dtype=dtype, device=device) if need[1] and not one else None
        gg = gbw = gw = None
        if need[2]:
            gg = out(size if a.gate_kind == _native.EMRS_NORM_GATE_TOKEN else size[-1:], dtype=dtype, device=device)
        if need[3]:
            gbw = out(size[-1:], dtype=dtype, device=device)
        if need[4] and grad_normed is not None:
            gw = out(size[-1:], dtype=dtype, device=device)
        if tokens:
            a.stream = a.normed = None
            if grad_normed is not None:
                rows, a.stream_stride = _rows(saved[0], h)
                if not (grad_normed.dtype is dtype and grad_normed.is_contiguous()):
                    grad_normed = grad_normed.to(dtype).contiguous()
                a.stream, a.grad_normed = rows.data_ptr(), grad_normed.data_ptr()
            if grad_stream is not None:
                if not (grad_stream.dtype is stream_dtype and grad_stream.is_contiguous()):
                    grad_stream = grad_stream.to(stream_dtype).contiguous()
                a.grad_stream = grad_stream.data_ptr()
            if gr is not None:
                a.grad_residual = gr.data_ptr()
            if gb is not None:
                a.grad_branch = gb.data_ptr()
            if gg is not None:
                a.grad_gate = gg.data_ptr()
            if gbw is not None:
                a.grad_branch_weight = gbw.data_ptr()
            if gw is not None:
                a.grad_weight = gw.data_ptr()
            if gw is not None or gbw is not None or (gg is not None and a.gate_kind == _native.EMRS_NORM_GATE_CHANNEL):
                scratch = workspace(_native.norm_workspace(a), device)
                a.workspace, a.workspace_bytes = scratch.data_ptr(), scratch.numel()
            run_on(device, _native.norm_backward, a)
        else:
            for g in (gr, gb, gg, gbw, gw):
                if g is not None:
                    g.zero_()
        return gr, gr if one else gb, gg, gbw, gw, None, None


_DTYPES = {code: dtype for dtype, code in DTYPE_CODES.items()}


def _again(ctx, saved):
    """The record anew, for tensors that hooks on saved tensors handed back; and those tensors."""
    a, size, rest = ctx.record, ctx.size, iter(saved)
    kept = [next(rest) if has else None for has in (ctx.has[3], ctx.has[2] or ctx.has[3], *ctx.has)]
    stream, rms, branch, gate, branch_weight, weight = kept
    for what, t in zip(("the stream", "the statistics", "the branch", "the gate", "the branch's weight", "the weight"), kept):
        if t is not None:
            on_device(what, t, ctx.device)
    if rms is not None and (rms.size() != (2, a.tokens) or rms.dtype != torch.float32):
        raise ValueError("the saved tensors are not those of the forward pass")
    if stream is not None and (stream.numel() != size.numel() or stream.dtype != _DTYPES[a.residual_dtype]):
        raise ValueError("the saved tensors are not those of the forward pass")
    # Where the stream is not read, one element stands for its shape.
    stream = torch.empty((), dtype=_DTYPES[a.residual_dtype], device=ctx.device).expand(size) if stream is None else stream.reshape(size)
    branch = None if branch is None else branch.reshape(size)
    if gate is not None:
        gate = gate.reshape(size if a.gate_kind == _native.EMRS_NORM_GATE_TOKEN else size[-1:])
    b, *others = _record(stream, branch, gate, branch_weight, weight, a.residual_scale, a.eps)
    if b.dtype != a.dtype:
        raise ValueError("the saved tensors are not those of the forward pass")
    b.gate_kind = a.gate_kind
    if rms is not None:
        rms = rms.contiguous()
        b.stream_rms = rms.data_ptr()
        b.branch_rms = b.stream_rms + 4 * a.tokens
    return b, [t for t in (stream, rms, *others) if t is not None]


def _wants_gradient(t) -> bool:
    return isinstance(t, torch.Tensor) and t.requires_grad


def _call(residual, branch, gate, branch_weight, weight, scale, eps):
    refuse_tangents(residual, branch, gate, branch_weight, weight)
    if torch.is_grad_enabled() and (_wants_gradient(residual) or _wants_gradient(branch) or _wants_gradient(weight) or _wants_gradient(gate) or
                                    _wants_gradient(branch_weight)):
        return _ResidualNorm.apply(residual, branch, gate, branch_weight, weight, scale, eps)
    stream, normed = _forward(residual, branch, gate, branch_weight, weight, scale, eps, False)[:2]
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
