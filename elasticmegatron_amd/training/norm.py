"""The norm before a block, and what joins the block behind it to the residual stream.

    stream = residual_scale residual + gate n(branch),  normed = stream / rms(stream) weight

with n(b) = b / rms(b) branch_weight, or b itself, and rms(x) = sqrt(mean x^2 + eps) over a token's channels.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from .. import _native
from ._common import DTYPE_CODES, dtype_code, on_device, refuse_tangents, run_on, workspace


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
    h, first = residual.shape[-1], None
    for what, t in (("branch", branch), ("weight", weight), ("branch_weight", branch_weight), ("gate", gate)):
        if t is None:
            continue
        on_device(what, t, device)
        first = first or (what, t.dtype)
        dtype_code(t, what, (torch.bfloat16, torch.float16))
        if t.dtype != first[1]:
            raise TypeError(f"{what} is {t.dtype}, {first[0]} {first[1]}")
        if what == "branch" and t.shape != residual.shape:
            raise ValueError(f"branch {tuple(t.shape)} does not fit residual {tuple(residual.shape)}")
        if what in ("weight", "branch_weight") and t.shape != (h,):
            raise ValueError(f"{what} is {tuple(t.shape)}: [{h}] is wanted")
    if first is None:
        raise ValueError("neither a branch nor a weight is given")
    if residual.dtype not in (torch.float32, first[1]):
        raise TypeError(f"residual is {residual.dtype}: torch.float32 or {first[0]}'s {first[1]} is wanted")
    if gate is None:
        return _native.EMRS_NORM_GATE_NONE
    if branch is None:
        raise ValueError("a gate without a branch")
    if gate.shape == branch.shape:
        return _native.EMRS_NORM_GATE_TOKEN
    if gate.shape != (h,):
        raise ValueError(f"gate is {tuple(gate.shape)}: [{h}] or branch's {tuple(branch.shape)} is wanted")
    return _native.EMRS_NORM_GATE_CHANNEL


def _address(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _record(kind, stream_dtype, dtype, tokens, h, branch, gate, branch_weight, weight, scale, eps):
    """The record with what both passes read; the tensors that it points to."""
    a = _native.Norm()
    a.dtype, a.residual_dtype, a.gate_kind = DTYPE_CODES[dtype], DTYPE_CODES[stream_dtype], kind
    a.tokens, a.hidden, a.residual_scale, a.eps = tokens, h, scale, eps
    keep = []
    if branch is not None:
        rows, a.branch_stride = _rows(branch, h)
        a.branch = rows.data_ptr()
        keep.append(rows)
        if gate is not None:
            rows, a.gate_stride = _rows(gate, h) if kind == _native.EMRS_NORM_GATE_TOKEN else (_vector(gate), h)
            a.gate = rows.data_ptr()
            keep.append(rows)
        if branch_weight is not None:
            rows = _vector(branch_weight)
            a.branch_weight = rows.data_ptr()
            keep.append(rows)
    if weight is not None:
        rows = _vector(weight)
        a.weight = rows.data_ptr()
        keep.append(rows)
    return a, keep


def _forward(residual, branch, gate, branch_weight, weight, scale, eps, statistics):
    """``(stream or None, normed or None, statistics or None, kind of gate)``."""
    kind = _check(residual, branch, gate, branch_weight, weight)
    h, dtype, device = residual.shape[-1], (weight if branch is None else branch).dtype, residual.device
    tokens = residual.numel() // h
    stream = None if branch is None else torch.empty(residual.size(), dtype=residual.dtype, device=device)
    normed = None if weight is None else torch.empty(residual.size(), dtype=dtype, device=device)
    rms = torch.empty((2, tokens), dtype=torch.float32, device=device) if statistics else None
    if tokens:
        a, keep = _record(kind, residual.dtype, dtype, tokens, h, branch, gate, branch_weight, weight, scale, eps)
        rows, a.residual_stride = _rows(residual, h)
        a.residual, a.stream, a.normed = rows.data_ptr(), _address(stream), _address(normed)
        if statistics:
            a.stream_rms = rms.data_ptr()
            a.branch_rms = a.stream_rms + 4 * tokens
        run_on(device, _native.norm_forward, a)
    return stream, normed, rms, kind


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, branch, gate, branch_weight, weight, scale, eps):
        stream, normed, rms, ctx.kind = _forward(residual, branch, gate, branch_weight, weight, scale, eps, True)
        ctx.save_for_backward(residual if stream is None else stream, branch, gate, branch_weight, weight, rms)
        ctx.scale, ctx.eps = scale, eps
        ctx.set_materialize_grads(False)
        if stream is None:
            return normed
        return stream if normed is None else (stream, normed)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        stream, branch, gate, branch_weight, weight, rms = ctx.saved_tensors  # raises where one was changed in place
        _check(stream, branch, gate, branch_weight, weight)  # hooks on saved tensors may hand back others
        on_device("the statistics", rms, stream.device)
        grad_stream = None if branch is None else grads[0]
        grad_normed = None if weight is None else grads[-1]
        need = ctx.needs_input_grad
        if grad_stream is None and grad_normed is None:
            return (None,) * 7
        shape, h, device = stream.size(), stream.shape[-1], stream.device
        dtype, tokens = (weight if branch is None else branch).dtype, stream.numel() // stream.shape[-1]
        room = lambda t: torch.empty(t.size(), dtype=t.dtype, device=device)  # noqa: E731
        # With nothing between them, residual and branch have one gradient, as those of a sum have.
        one = need[0] and need[1] and gate is None and branch_weight is None and ctx.scale == 1.0 and stream.dtype == dtype
        out = {
            "grad_residual": torch.empty(shape, dtype=stream.dtype, device=device) if need[0] else None,
            "grad_branch": room(branch) if need[1] and not one else None,
            "grad_gate": room(gate) if need[2] else None,
            "grad_branch_weight": room(branch_weight) if need[3] else None,
            "grad_weight": room(weight) if need[4] and grad_normed is not None else None,
        }
        if not tokens:
            for g in out.values():
                if g is not None:
                    g.zero_()
        else:
            a, keep = _record(ctx.kind, stream.dtype, dtype, tokens, h, branch, gate, branch_weight, weight, ctx.scale, ctx.eps)
            if grad_normed is not None:
                rows, a.stream_stride = _rows(stream, h)
                keep += [rows, grad_normed.to(dtype).contiguous()]
                a.stream, a.grad_normed = rows.data_ptr(), keep[-1].data_ptr()
            if grad_stream is not None:
                keep.append(grad_stream.to(stream.dtype).contiguous())
                a.grad_stream = keep[-1].data_ptr()
            rms = rms.contiguous()
            a.stream_rms = rms.data_ptr()
            a.branch_rms = a.stream_rms + 4 * tokens
            for name, g in out.items():
                setattr(a, name, _address(g))
            if out["grad_weight"] is not None or out["grad_branch_weight"] is not None or out["grad_gate"] is not None:
                scratch = workspace(_native.norm_workspace(a), device)
                a.workspace, a.workspace_bytes = scratch.data_ptr(), scratch.numel()
            run_on(device, _native.norm_backward, a)
        if one:
            out["grad_branch"] = out["grad_residual"]
        return out["grad_residual"], out["grad_branch"], out["grad_gate"], out["grad_branch_weight"], out["grad_weight"], None, None


def _call(residual, branch, gate, branch_weight, weight, scale, eps):
    tensors = (residual, branch, gate, branch_weight, weight)
    refuse_tangents(*tensors)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors):
        return _ResidualNorm.apply(*tensors, scale, eps)
    stream, normed, _, _ = _forward(*tensors, scale, eps, False)
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
