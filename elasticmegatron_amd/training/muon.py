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
from ._common import dtype_code, on_device, refuse_tangents, run_on, workspace, written
from ._overlap import first_conflict, rows_of

Matrices = Union[torch.Tensor, Sequence[torch.Tensor]]

# a, b, c: the quintic whose slope at 0 is steep, so that five steps bring singular values from 0.002 of
# the norm on into [0.7, 1.2].
MUON_COEFFICIENTS = (3.4445, -4.7750, 2.0315)

# One native call works on as many matrices as fit this much workspace (and on one at least).
WORKSPACE_BYTES = 8 << 30


class _Stack:
    """Matrices of one kind and one shape: their addresses and the row stride that they share."""

    def __init__(self, what: str, m: Matrices):
        self.what = what
        if isinstance(m, torch.Tensor):
            if m.dim() not in (2, 3):
                raise ValueError(f"{what} has {m.dim()} dimensions: a matrix, or a stack of matrices, is wanted")
            self.tensors, self.count = [m], 1 if m.dim() == 2 else m.shape[0]
        else:
            self.tensors = list(m)
            self.count = len(self.tensors)
            for t in self.tensors:
                if not isinstance(t, torch.Tensor):
                    raise TypeError(f"{what} is no tensor")
                if t.dim() != 2:
                    raise ValueError(f"{what} has a member of {t.dim()} dimensions: matrices are wanted")
        refuse_tangents(self.tensors)
        if self.count:
            self.shape = self.tensors[0].shape[-2:]
            self.dtype, self.device = self.tensors[0].dtype, self.tensors[0].device

    def check(self, count: int, shape, device, dtype=None) -> None:
        """Raises unless there are `count` matrices of that shape, on that device and of one type."""
        if self.count != count:
            raise ValueError(f"{self.what} holds {self.count} matrices, the others {count}")
        for t in self.tensors:
            on_device(self.what, t, device)
            if t.shape[-2:] != shape:
                raise ValueError(f"{self.what} is {tuple(t.shape[-2:])}: {tuple(shape)} is wanted, for all matrices of a call")
            if dtype is not None and t.dtype != dtype:
                raise TypeError(f"{self.what} is {t.dtype}: {dtype} is wanted")
            if t.dtype != self.dtype:
                raise TypeError(f"{self.what} holds matrices of several types")

    def lay_out(self, copy: bool) -> None:
        """Addresses and the row stride; matrices that lie otherwise are copied, or refused."""
        rows, cols = self.shape
        strides = {t.stride(-2) for t in self.tensors}
        if any((cols > 1 and t.stride(-1) != 1) or (rows > 1 and t.stride(-2) < cols) for t in self.tensors) or (len(strides) > 1 and rows > 1):
            if not copy:
                raise ValueError(f"{self.what} is written in place: unit column stride and one row stride are wanted")
            self.tensors = [t.contiguous() for t in self.tensors]
        self.stride = self.tensors[0].stride(-2)
        if len(self.tensors) == 1 and self.tensors[0].dim() == 3:
            t = self.tensors[0]
            step = t.stride(0) * t.element_size()
            base = t.data_ptr()
            self.addresses = [base + i * step for i in range(self.count)]
        else:
            self.addresses = [t.data_ptr() for t in self.tensors]

    def in_memory(self, written: bool):
        rows, cols = self.shape
        size = self.tensors[0].element_size()
        stride = (self.stride if rows > 1 else cols) * size
        return [rows_of(base, rows, stride, cols * size, self.what, i, written) for i, base in enumerate(self.addresses)]

    def table(self, lo: int, hi: int):
        return (ctypes.c_uint64 * (hi - lo))(*self.addresses[lo:hi])


def _coefficients(c, steps: int):
    rows = [tuple(c)] * steps if len(c) == 3 and not hasattr(c[0], "__len__") else [tuple(r) for r in c]
    if not 1 <= steps <= _native.EMRS_MUON_MAX_STEPS:
        raise ValueError(f"{steps} steps: 1 to {_native.EMRS_MUON_MAX_STEPS} are wanted")
    if len(rows) != steps or any(len(r) != 3 for r in rows):
        raise ValueError("coefficients are (a, b, c), or one such triple for each step")
    return (ctypes.c_float * (3 * steps))(*(float(x) for r in rows for x in r))


def _run(kinds, *, steps, coefficients, eps, mu, nesterov, decay, rate) -> None:
    """One native call for as many matrices as its workspace allows, until all are done."""
    grad = kinds["grad"]
    for name, k in kinds.items():
        k.lay_out(copy=name == "grad")
    if "main" in kinds:  # matrices are worked on side by side
        conflict = first_conflict(m for name, k in kinds.items() for m in k.in_memory(name != "grad"))
        if conflict:
            a, b = conflict
            raise ValueError(f"{a.what} [{a.index}] and {b.what} [{b.index}] share memory, which is written in place")
    a = _native.Muon()
    a.grad_dtype = dtype_code(grad.tensors[0], "grad")
    a.rows, a.cols, a.steps, a.nesterov = *grad.shape, steps, int(nesterov)
    a.coefficients = ctypes.addressof(coefficients)
    a.mu, a.eps, a.decay, a.rate = mu, eps, decay, rate
    a.count = 1
    at_once, size = grad.count, 0
    if grad.count > 1:
        at_once = min(grad.count, _native.EMRS_MUON_MAX_MATRICES, max(1, WORKSPACE_BYTES // _native.muon_workspace(a)))
        a.count = at_once
    size = _native.muon_workspace(a)
    scratch = workspace(size, grad.device)
    a.workspace, a.workspace_bytes = scratch.data_ptr(), scratch.numel()
    written(*(t for name, k in kinds.items() if name != "grad" for t in k.tensors))
    for lo in range(0, grad.count, at_once):
        hi = min(grad.count, lo + at_once)
        a.count = hi - lo
        tables = {name: k.table(lo, hi) for name, k in kinds.items()}
        for name, t in tables.items():
            setattr(a, name, ctypes.addressof(t))
            setattr(a, name + "_stride", kinds[name].stride)
        run_on(grad.device, _native.muon_step, a)


@torch.no_grad()
def orthogonalise(matrices: Matrices, *, steps: int = 5, coefficients=MUON_COEFFICIENTS,
                  eps: float = 1e-7) -> Union[torch.Tensor, List[torch.Tensor]]:
    """``matrices`` (fp32, bf16 or fp16; one matrix, a stack [n, rows, cols], or a sequence of matrices of
    one shape) with their singular values brought near 1: bf16, of the same form.

    ``coefficients``: (a, b, c), or one such triple for each step; they have to keep singular values in
    [0, 1] bounded.  A matrix of zeros stays zeros.
    """
    g = _Stack("matrices", matrices)
    coefficients = _coefficients(coefficients, steps)
    single = isinstance(matrices, torch.Tensor)
    if g.count:
        g.check(g.count, g.shape, g.device)
        dtype_code(g.tensors[0], "matrices")
        out = torch.empty((g.count, *g.shape), dtype=torch.bfloat16, device=g.device)
        if g.shape.numel():
            _run({"grad": g, "out": _Stack("out", out)}, steps=steps, coefficients=coefficients, eps=eps, mu=0.0, nesterov=False,
                 decay=0.0, rate=0.0)
        return out.view(matrices.shape) if single else list(out.unbind(0))
    return torch.empty(matrices.shape, dtype=torch.bfloat16, device=matrices.device) if single else []


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
    ``lr * rms_scale``, as AdamW's are with 0.2.  No two matrices may share memory that is written (a tied one is
    listed once); ``grad`` may be that of its own ``main`` or ``model``.  A matrix is taken as it is given: one that tensor
    parallelism or a distributed optimizer has cut is to be gathered first.
    """
    g, w, b = _Stack("grad", grad), _Stack("main", main), _Stack("momentum_buffer", momentum_buffer)
    img = None if model is None else _Stack("model", model)
    coefficients = _coefficients(coefficients, steps)
    if not g.count:
        if w.count or b.count or (img is not None and img.count):
            raise ValueError("grad holds no matrices")
        return
    g.check(g.count, g.shape, g.device)
    dtype_code(g.tensors[0], "grad")
    w.check(g.count, g.shape, g.device, torch.float32)
    b.check(g.count, g.shape, g.device, torch.float32)
    kinds = {"grad": g, "momentum": b, "main": w}
    if img is not None:
        img.check(g.count, g.shape, g.device, torch.bfloat16)
        kinds["image"] = img
    if g.shape.numel():
        _run(kinds, steps=steps, coefficients=coefficients, eps=eps, mu=momentum, nesterov=nesterov, decay=lr * weight_decay,
             rate=lr * rms_scale * math.sqrt(max(g.shape)))
