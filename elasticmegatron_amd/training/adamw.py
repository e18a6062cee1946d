"""The AdamW update of a flat run of a state's elements."""

from __future__ import annotations

from typing import Optional

import torch

from .. import _native
from ._common import dtype_code, on_device, run_on


@torch.no_grad()
def adamw_step(main: torch.Tensor, exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor, grad: torch.Tensor, *,
               model: Optional[torch.Tensor] = None, lr: float, beta1: float = 0.9, beta2: float = 0.95, eps: float = 1e-8,
               weight_decay: float = 0.0, step: int) -> None:
    """One AdamW update, in place:

        exp_avg = beta1 exp_avg + (1 - beta1) grad,  exp_avg_sq = beta2 exp_avg_sq + (1 - beta2) grad^2
        main = main (1 - lr weight_decay) - lr (exp_avg / (1 - beta1^step)) / (sqrt(exp_avg_sq / (1 - beta2^step)) + eps)
        model = main as bf16   (``model`` given)

    ``main``, ``exp_avg`` and ``exp_avg_sq`` are fp32, ``grad`` fp32, bf16 or fp16, all contiguous and of one
    size: a parameter's, a rank's shard of it, or a whole arena.  ``step`` counts from 1.
    """
    if not isinstance(main, torch.Tensor):
        raise TypeError("main is no tensor")
    n, device = main.numel(), main.device
    for what, t, dtype in (("main", main, torch.float32), ("exp_avg", exp_avg, torch.float32),
                           ("exp_avg_sq", exp_avg_sq, torch.float32), ("grad", grad, None), ("model", model, torch.bfloat16)):
        if t is None and what == "model":
            continue
        on_device(what, t, device)
        if dtype is not None and t.dtype != dtype:
            raise TypeError(f"{what} is {t.dtype}: {dtype} is wanted")
        if t.numel() != n:
            raise ValueError(f"{what} has {t.numel()} elements, main {n}")
        if not t.is_contiguous():
            if what != "grad":
                raise ValueError(f"{what} is written in place: a contiguous tensor is wanted")
            grad = t.contiguous()
    if not 1 <= step < 1 << 32:
        raise ValueError("step counts from 1")
    a = _native.AdamW()
    a.n, a.grad_dtype, a.step = n, dtype_code(grad, "grad"), step
    a.main, a.exp_avg, a.exp_avg_sq, a.grad = (t.data_ptr() for t in (main, exp_avg, exp_avg_sq, grad))
    a.image = None if model is None else model.data_ptr()
    a.lr, a.beta1, a.beta2, a.eps, a.weight_decay = lr, beta1, beta2, eps, weight_decay
    run_on(device, _native.adamw_step, a)
