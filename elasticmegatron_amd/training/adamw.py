"""The AdamW update of a flat run of a state's elements."""

from __future__ import annotations

from typing import Optional

import torch

from .. import _native
from ._common import DTYPE_CODES, dtype_code, on_device, refuse_tangents, run_on, written


def adamw_step(main: torch.Tensor, exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor, grad: torch.Tensor, *,
               model: Optional[torch.Tensor] = None, lr: float, beta1: float = 0.9, beta2: float = 0.95, eps: float = 1e-8,
               weight_decay: float = 0.0, step: int) -> None:
    """One AdamW update, in place:

        exp_avg = beta1 exp_avg + (1 - beta1) grad,  exp_avg_sq = beta2 exp_avg_sq + (1 - beta2) grad^2
        main = main (1 - lr weight_decay) - lr (exp_avg / (1 - beta1^step)) / (sqrt(exp_avg_sq / (1 - beta2^step)) + eps)
        model = main as bf16   (``model`` given)

    ``main``, ``exp_avg`` and ``exp_avg_sq`` are fp32, ``grad`` fp32, bf16 or fp16, all contiguous and of one
    size: a parameter's, a rank's shard of it, or a whole arena.  Shapes may differ as views of one flat run do; a
    ``grad`` with ``main``'s sides in another order is refused.  ``step`` counts from 1.
    """
    refuse_tangents(main, exp_avg, exp_avg_sq, grad, model)
    n = main.numel() if isinstance(main, torch.Tensor) else 0
    for t in (main, exp_avg, exp_avg_sq):
        if not (isinstance(t, torch.Tensor) and t.dtype is torch.float32 and t.is_cuda and t.numel() == n and t.is_contiguous()):
            _refuse(main, exp_avg, exp_avg_sq, grad, model)
    if not (isinstance(grad, torch.Tensor) and grad.dtype in DTYPE_CODES and grad.is_cuda and grad.numel() == n):
        _refuse(main, exp_avg, exp_avg_sq, grad, model)
    if grad.size() != main.size() and _turned(grad.size(), main.size()):
        raise ValueError(f"grad is {tuple(grad.size())}, main {tuple(main.size())}: its elements are in another order")
    if model is not None and not (isinstance(model, torch.Tensor) and model.dtype is torch.bfloat16 and model.is_cuda and
                                  model.numel() == n and model.is_contiguous()):
        _refuse(main, exp_avg, exp_avg_sq, grad, model)
    device = main.device
    if not (exp_avg.device == device == exp_avg_sq.device and grad.device == device and (model is None or model.device == device)):
        _refuse(main, exp_avg, exp_avg_sq, grad, model)
    if not 1 <= step < 1 << 32:
        raise ValueError("step counts from 1")
    grad = grad.detach().contiguous()
    a = _native.AdamW(n, main.data_ptr(), exp_avg.data_ptr(), exp_avg_sq.data_ptr(), grad.data_ptr(), DTYPE_CODES[grad.dtype], step,
                      None if model is None else model.data_ptr(), lr, beta1, beta2, eps, weight_decay)
    written(*((main, exp_avg, exp_avg_sq) if model is None else (main, exp_avg, exp_avg_sq, model)))
    run_on(device, _native.adamw_step, a)


def _turned(a, b) -> bool:
    """Whether ``a`` has the sides of ``b`` in another order: a transposed tensor, no flat run of the same one."""
    a, b = ([n for n in x if n != 1] for x in (a, b))
    return a != b and sorted(a) == sorted(b)


def _refuse(main, exp_avg, exp_avg_sq, grad, model) -> None:
    """Raises for the first argument that is not as it has to be."""
    for what, t, dtype in (("main", main, torch.float32), ("exp_avg", exp_avg, torch.float32),
                           ("exp_avg_sq", exp_avg_sq, torch.float32), ("grad", grad, None), ("model", model, torch.bfloat16)):
        if t is None and what == "model":
            continue
        on_device(what, t, main.device if isinstance(main, torch.Tensor) else None)
        if dtype is not None and t.dtype != dtype:
            raise TypeError(f"{what} is {t.dtype}: {dtype} is wanted")
        if t.numel() != main.numel():
            raise ValueError(f"{what} has {t.numel()} elements, main {main.numel()}")
        if what != "grad" and not t.is_contiguous():
            raise ValueError(f"{what} is written in place: a contiguous tensor is wanted")
    dtype_code(grad, "grad")
