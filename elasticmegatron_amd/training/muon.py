"""Newton-Schulz orthogonalisation, and the Muon update of weight matrices.

    X = U / (|U|_F + eps);  steps times:  A = X X^T,  X = a X + (b A + c A A) X

leaves U's singular vectors and brings its singular values near 1.  Muon takes U from the momentum of
the gradients and steps along X, whose entries it scales to the size of AdamW's updates.
"""

from __future__ import annotations

import ctypes
import math
from typing import List, Optional, Sequence, Tuple, Union

import torch

from .. import _native
from ._common import dtype_code, on_device, stream_of, workspace

Matrices = Union[torch.Tensor, Sequence[torch.Tensor]]

# a, b, c: the quintic whose slope at 0 is steep, so that five steps bring singular values from 0.002 of
# the norm on into [0.7, 1.2].
MUON_COEFFICIENTS = (3.4445, -4.7750, 2.0315)

# One native call works on as many matrices as fit this much workspace (and on one at least).
WORKSPACE_BYTES = 8 << 30


def _matrices(what: str, m: Matrices) -> List[torch.Tensor]:
    if isinstance(m, torch.Tensor):
        if m.dim() not in (2, 3):
            raise ValueError(f"{what} has {m.dim()} dimensions: a matrix, or a stack of matrices, is wanted")
        return [m] if m.dim() == 2 else list(m.unbind(0))
    return list(m)


def _check(what: str, ms: List[torch.Tensor], count: int, shape, device, dtype=None) -> None:
    if len(ms) != count:
        raise ValueError(f"{what} holds {len(ms)} matrices, the others {count}")
    for t in ms:
        on_device(what, t, device)
        if t.shape != shape or t.dim() != 2:
            raise ValueError(f"{what} is {tuple(t.shape)}: {tuple(shape)} is wanted, for all matrices of a call")
        if dtype is not None and t.dtype != dtype:
            raise TypeError(f"{what} is {t.dtype}: {dtype} is wanted")
        if t.dtype != ms[0].dtype:
            raise TypeError(f"{what} holds matrices of several types")


def _in_rows(t: torch.Tensor) -> bool:
    rows, cols = t.shape
    return (cols == 1 or t.stride(1) == 1) and (rows == 1 or t.stride(0) >= cols)


def _coefficients(c, steps: int):
    rows = [tuple(c)] * steps if len(c) == 3 and not hasattr(c[0], "__len__") else [tuple(r) for r in c]
    if not 1 <= steps <= _native.EMRS_MUON_MAX_STEPS:
        raise ValueError(f"{steps} steps: 1 to {_native.EMRS_MUON_MAX_STEPS} are wanted")
    if len(rows) != steps or any(len(r) != 3 for r in rows):
        raise ValueError("coefficients are (a, b, c), or one such triple for each step")
    return (ctypes.c_float * (3 * steps))(*(float(x) for r in rows for x in r))


class _Stack:
    """Matrices of one kind: their addresses and the row stride that they share."""

    def __init__(self, what: str, ms: Optional[List[torch.Tensor]], copy: bool):
        self.ms = ms
        if ms is None:
            return
        strides = {t.stride(0) for t in ms}
        if not all(map(_in_rows, ms)) or (len(strides) > 1 and ms[0].shape[0] > 1):
            if not copy:
                raise ValueError(f"{what} is written in place: unit column stride and one row stride are wanted")
            self.ms = [t.contiguous() for t in ms]
        self.stride = self.ms[0].stride(0)

    def table(self, lo: int, hi: int):
        return None if self.ms is None else (ctypes.c_uint64 * (hi - lo))(*(t.data_ptr() for t in self.ms[lo:hi]))


def _run(grad, momentum, main, image, out, *, steps, coefficients, eps, mu, nesterov, decay, rate) -> None:
    """One native call for as many matrices as its workspace allows, until all are done."""
    device, (rows, cols) = grad.ms[0].device, grad.ms[0].shape
    a = _native.Muon()
    a.grad_dtype = dtype_code(grad.ms[0], "grad")
    a.rows, a.cols, a.steps, a.nesterov = rows, cols, steps, int(nesterov)
    a.coefficients = ctypes.addressof(coefficients)
    a.mu, a.eps, a.decay, a.rate = mu, eps, decay, rate
    a.count = 1
    count = len(grad.ms)
    at_once = min(count, _native.EMRS_MUON_MAX_MATRICES, max(1, WORKSPACE_BYTES // _native.muon_workspace(a)))
    a.count = at_once
    scratch = workspace(_native.muon_workspace(a), device)
    a.workspace, a.workspace_bytes = scratch.data_ptr(), scratch.numel()
    kinds = [("grad", grad), ("momentum", momentum), ("main", main), ("image", image), ("out", out)]
    for lo in range(0, count, at_once):
        hi = min(count, lo + at_once)
        a.count = hi - lo
        tables = [s.table(lo, hi) for _, s in kinds]
        for (name, s), t in zip(kinds, tables):
            setattr(a, name, None if t is None else ctypes.addressof(t))
            if t is not None:
                setattr(a, name + "_stride", s.stride)
        with torch.cuda.device(device):
            _native.muon_step(a, stream_of(device))


def _head(grad: Matrices):
    g = _matrices("grad", grad)
    if not g:
        return g, None, None
    if not isinstance(g[0], torch.Tensor):
        raise TypeError("grad is no tensor")
    _check("grad", g, len(g), g[0].shape, g[0].device)
    dtype_code(g[0], "grad")
    return g, g[0].shape, g[0].device


def orthogonalise(matrices: Matrices, *, steps: int = 5, coefficients=MUON_COEFFICIENTS,
                  eps: float = 1e-7) -> Union[torch.Tensor, List[torch.Tensor]]:
    """``matrices`` (fp32, bf16 or fp16; one matrix, a stack [n, rows, cols], or a sequence of matrices of
    one shape) with their singular values brought near 1: bf16, of the same form.

    ``coefficients``: (a, b, c), or one such triple for each step; they have to keep singular values in
    [0, 1] bounded.  A matrix of zeros stays zeros.
    """
    g, shape, device = _head(matrices)
    coefficients = _coefficients(coefficients, steps)
    stacked = torch.empty((len(g), *(shape or (0, 0))), dtype=torch.bfloat16, device=device)
    if g and shape.numel():
        _run(_Stack("matrices", [t.detach() for t in g], True), _Stack("", None, True), _Stack("", None, True),
             _Stack("", None, True), _Stack("out", list(stacked.unbind(0)), False), steps=steps, coefficients=coefficients, eps=eps,
             mu=0.0, nesterov=False, decay=0.0, rate=0.0)
    if isinstance(matrices, torch.Tensor):
        return stacked.view(matrices.shape)
    return list(stacked.unbind(0))


@torch.no_grad()
def muon_step(main: Matrices, momentum_buffer: Matrices, grad: Matrices, *, model: Optional[Matrices] = None, lr: float,
              momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0, rms_scale: float = 0.2, steps: int = 5,
              coefficients: Tuple = MUON_COEFFICIENTS, eps: float = 1e-7) -> None:
    """One Muon update, in place, of matrices of one shape (each argument one matrix, a stack
    [n, rows, cols], or a sequence of matrices):

        momentum_buffer = momentum * momentum_buffer + grad
        U = grad + momentum * momentum_buffer   (``nesterov``; else momentum_buffer)
        main = main * (1 - lr * weight_decay) - lr * rms_scale * sqrt(max(rows, cols)) * orthogonalise(U)
        model = main as bf16                    (``model`` given)

    ``main`` and ``momentum_buffer`` are fp32 (a state's main and exp_avg), ``grad`` fp32, bf16 or fp16.
    Entries of an orthogonal matrix are 1 / sqrt(max(rows, cols)), so an update's are about
    ``lr * rms_scale``, as AdamW's are with 0.2.  A matrix is taken as it is given: one that tensor
    parallelism or a distributed optimizer has cut is to be gathered first.
    """
    g, shape, device = _head(grad)
    w, b = _matrices("main", main), _matrices("momentum_buffer", momentum_buffer)
    img = None if model is None else _matrices("model", model)
    coefficients = _coefficients(coefficients, steps)
    if not g and not w and not b and not img:
        return
    if not g:
        raise ValueError("grad holds no matrices")
    _check("main", w, len(g), shape, device, torch.float32)
    _check("momentum_buffer", b, len(g), shape, device, torch.float32)
    if img is not None:
        _check("model", img, len(g), shape, device, torch.bfloat16)
    if not shape.numel():
        return
    _run(_Stack("grad", g, True), _Stack("momentum_buffer", b, False), _Stack("main", w, False), _Stack("model", img, False),
         _Stack("", None, False), steps=steps, coefficients=coefficients, eps=eps, mu=momentum, nesterov=nesterov,
         decay=lr * weight_decay, rate=lr * rms_scale * math.sqrt(max(shape)))
