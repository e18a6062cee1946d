"""What the operators share: types, devices and workspaces."""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from .. import _native

DTYPE_CODES = {torch.float32: _native.EMRS_FP32, torch.bfloat16: _native.EMRS_BF16, torch.float16: _native.EMRS_FP16}


def dtype_code(t: torch.Tensor, what: str, allowed=tuple(DTYPE_CODES)) -> int:
    if t.dtype not in allowed:
        raise TypeError(f"{what} is {t.dtype}: one of {', '.join(str(d) for d in allowed)} is wanted")
    return DTYPE_CODES[t.dtype]


def on_device(what: str, t: torch.Tensor, device: torch.device) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} is no tensor")
    if not t.is_cuda:
        raise ValueError(f"{what} is on {t.device}: a GPU is wanted")
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, the others on {device}")


def refuse_tangents(*arguments) -> None:
    """Raises where a tensor, alone or in a sequence, carries a forward-mode tangent: no operator here has such a
    derivative, and a kernel that reads the tensor's memory would drop it."""
    if forward_ad._current_level < 0:  # none is being taken
        return
    for t in arguments:
        if isinstance(t, (list, tuple)):
            refuse_tangents(*t)
        elif isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("the operators of a training step have no forward-mode derivatives")


def lies(*tensors) -> tuple:
    """Where tensors (or None) are and how: what a record of their addresses holds good for."""
    return tuple([None if t is None else (t.data_ptr(), t.size(), t.stride(), t.dtype) for t in tensors])


def workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    """Scratch of one call.  The caching allocator's blocks lie on 512 bytes, and one that is freed after the
    call is reused by later work of the same stream only."""
    return torch.empty(max(1, nbytes), dtype=torch.uint8, device=device)


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


# The same without a Stream object on the way, where torch has it: 2 us less a call.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def written(*tensors: torch.Tensor) -> None:
    """Counts ``tensors`` as changed in place, which kernels behind an address do not do by themselves: a graph
    that saved one of them, or an arena that it is a view of, then refuses to run backward."""
    torch.autograd.graph.increment_version(tensors)


def run_on(device: torch.device, call, record) -> None:
    """``call(record, stream)`` with ``device`` current, on its current stream."""
    stream = _raw_stream(device.index) if _raw_stream is not None else _stream(device)
    if torch.cuda.current_device() == device.index:
        call(record, stream)
    else:
        with torch.cuda.device(device):
            call(record, stream)
