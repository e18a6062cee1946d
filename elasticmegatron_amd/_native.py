"""ctypes binding of libemrs (include/emrs.h).

The library is built in-tree by ``__graft_entry__.build()`` (or
``python -m elasticmegatron_amd.build``) into
``elasticmegatron_amd/csrc/libemrs.so``.  There is no fallback: when the
library is missing every entry point raises.
"""

from __future__ import annotations

import array
import ctypes
import os
from typing import Optional, Sequence

import numpy as np

from .resharding.layout import PIECE_DTYPE, SEGMENT_DTYPE

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "csrc", "libemrs.so")

EMRS_OK = 0
ERRORS = {
    -1: "EMRS_ERR_INVALID_ARGUMENT",
    -2: "EMRS_ERR_OUT_OF_BOUNDS",
    -3: "EMRS_ERR_MISALIGNED",
    -4: "EMRS_ERR_OVERLAP",
    -5: "EMRS_ERR_HIP",
    -6: "EMRS_ERR_NO_DEVICE",
    -7: "EMRS_ERR_TOO_MANY_BUFFERS",
    -8: "EMRS_ERR_ALIAS",
    -9: "EMRS_ERR_CAPTURE",
    -10: "EMRS_ERR_TOO_LARGE",
}
EMRS_PLAN_CHECK_DISJOINT = 1
EMRS_MAX_BUFFERS = 65535
EMRS_ARG_BUFFERS = 128  # buffers per side passed in kernel arguments (more use a device table)
EMRS_STATIC_SCRATCH_BYTES = 4 << 20  # device scratch of emrs_plan_compare_static

# Every function include/emrs.h declares.
EXPORTS = (
    "emrs_last_error", "emrs_abi_version", "emrs_device_count", "emrs_plan_create",
    "emrs_plan_stats_get", "emrs_plan_execute", "emrs_plan_destroy", "emrs_get_tuning",
    "emrs_set_tuning", "emrs_synth_fill", "emrs_synth_verify", "emrs_plan_compare", "emrs_xor_checksum",
    "emrs_plan_compare_static", "emrs_plan_prepare", "emrs_ipc_export", "emrs_ipc_open", "emrs_ipc_close",
    "emrs_ipc_open_count", "emrs_loss_workspace", "emrs_loss_forward", "emrs_loss_backward", "emrs_muon_workspace",
    "emrs_muon_step", "emrs_adamw_step", "emrs_norm_workspace", "emrs_norm_forward", "emrs_norm_backward",
    "emrs_experts_workspace", "emrs_experts_forward", "emrs_experts_backward",
    "emrs_attention_workspace", "emrs_attention_forward", "emrs_attention_backward",
)

# struct emrs_compare_stats
COMPARE_DTYPE = np.dtype([("elements", "<u8"), ("mismatches", "<u8"), ("nonfinite", "<u8"), ("reserved", "<u8"),
                          ("sum_sq_diff", "<f8"), ("sum_sq_expected", "<f8"), ("max_abs_diff", "<f4"),
                          ("max_rel_diff", "<f4"), ("reserved2", "<u8")])


class EmrsError(RuntimeError):
    def __init__(self, code: int, where: str, msg: str):
        super().__init__(f"{where}: {ERRORS.get(code, code)}: {msg}")
        self.code = code


class PlanStats(ctypes.Structure):
    _fields_ = [
        ("n_segments", ctypes.c_uint64), ("n_device_segments", ctypes.c_uint64),
        ("payload_bytes", ctypes.c_uint64), ("read_bytes", ctypes.c_uint64), ("vector_bytes", ctypes.c_uint64),
        ("scalar_bytes", ctypes.c_uint64), ("n_chunks", ctypes.c_uint64),
        ("n_src_bufs", ctypes.c_uint32), ("n_dst_bufs", ctypes.c_uint32),
    ]


class Tuning(ctypes.Structure):
    _fields_ = [("blocks_per_cu", ctypes.c_uint32), ("nontemporal", ctypes.c_uint32),
                ("xcd_remap", ctypes.c_uint32), ("run", ctypes.c_uint32), ("persistent", ctypes.c_uint32),
                ("lanes", ctypes.c_uint32), ("units", ctypes.c_uint32), ("buffer_ops", ctypes.c_uint32),
                ("chunk_index", ctypes.c_uint32), ("warm_tables", ctypes.c_uint32)]


class Loss(ctypes.Structure):
    """struct emrs_loss"""

    _fields_ = [("dtype", ctypes.c_uint32), ("n_shards", ctypes.c_uint32), ("tokens", ctypes.c_uint64),
                ("hidden_size", ctypes.c_uint64), ("hidden", ctypes.c_void_p), ("hidden_stride", ctypes.c_uint64),
                ("weights", ctypes.c_void_p), ("weight_strides", ctypes.c_void_p), ("shard_rows", ctypes.c_void_p),
                ("vocab_start", ctypes.c_uint64), ("vocab_size", ctypes.c_uint64), ("target", ctypes.c_void_p),
                ("ignore_index", ctypes.c_int64), ("lse", ctypes.c_void_p), ("target_logit", ctypes.c_void_p),
                ("loss", ctypes.c_void_p), ("grad_loss", ctypes.c_void_p), ("grad_hidden", ctypes.c_void_p),
                ("grad_weights", ctypes.c_void_p), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_uint64)]


class Muon(ctypes.Structure):
    """struct emrs_muon"""

    _fields_ = [("count", ctypes.c_uint32), ("grad_dtype", ctypes.c_uint32), ("rows", ctypes.c_uint64),
                ("cols", ctypes.c_uint64), ("grad", ctypes.c_void_p), ("momentum", ctypes.c_void_p),
                ("main", ctypes.c_void_p), ("image", ctypes.c_void_p), ("out", ctypes.c_void_p),
                ("grad_stride", ctypes.c_uint64), ("momentum_stride", ctypes.c_uint64),
                ("main_stride", ctypes.c_uint64), ("image_stride", ctypes.c_uint64), ("out_stride", ctypes.c_uint64),
                ("steps", ctypes.c_uint32), ("nesterov", ctypes.c_uint32), ("coefficients", ctypes.c_void_p),
                ("mu", ctypes.c_float), ("eps", ctypes.c_float), ("decay", ctypes.c_float), ("rate", ctypes.c_float),
                ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_uint64)]


class AdamW(ctypes.Structure):
    """struct emrs_adamw"""

    _fields_ = [("n", ctypes.c_uint64), ("main", ctypes.c_void_p), ("exp_avg", ctypes.c_void_p),
                ("exp_avg_sq", ctypes.c_void_p), ("grad", ctypes.c_void_p), ("grad_dtype", ctypes.c_uint32),
                ("step", ctypes.c_uint32), ("image", ctypes.c_void_p), ("lr", ctypes.c_double),
                ("beta1", ctypes.c_double), ("beta2", ctypes.c_double), ("eps", ctypes.c_double),
                ("weight_decay", ctypes.c_double)]


class Norm(ctypes.Structure):
    """struct emrs_norm"""

    _fields_ = [("dtype", ctypes.c_uint32), ("residual_dtype", ctypes.c_uint32), ("gate_kind", ctypes.c_uint32),
                ("reserved", ctypes.c_uint32), ("tokens", ctypes.c_uint64), ("hidden", ctypes.c_uint64),
                ("residual", ctypes.c_void_p), ("residual_stride", ctypes.c_uint64), ("branch", ctypes.c_void_p),
                ("branch_stride", ctypes.c_uint64), ("gate", ctypes.c_void_p), ("gate_stride", ctypes.c_uint64),
                ("branch_weight", ctypes.c_void_p), ("weight", ctypes.c_void_p), ("residual_scale", ctypes.c_float),
                ("eps", ctypes.c_float), ("stream", ctypes.c_void_p), ("stream_stride", ctypes.c_uint64),
                ("normed", ctypes.c_void_p), ("stream_rms", ctypes.c_void_p), ("branch_rms", ctypes.c_void_p),
                ("grad_stream", ctypes.c_void_p), ("grad_normed", ctypes.c_void_p), ("grad_residual", ctypes.c_void_p),
                ("grad_branch", ctypes.c_void_p), ("grad_gate", ctypes.c_void_p), ("grad_weight", ctypes.c_void_p),
                ("grad_branch_weight", ctypes.c_void_p), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_uint64)]


class Experts(ctypes.Structure):
    """struct emrs_experts"""

    _fields_ = [("dtype", ctypes.c_uint32), ("n_experts", ctypes.c_uint32), ("rows", ctypes.c_uint64),
                ("n_in", ctypes.c_uint64), ("n_out", ctypes.c_uint64), ("counts", ctypes.c_void_p),
                ("counts_bytes", ctypes.c_uint32), ("reserved", ctypes.c_uint32), ("x", ctypes.c_void_p),
                ("x_stride", ctypes.c_uint64), ("weights", ctypes.c_void_p), ("weight_stride", ctypes.c_uint64),
                ("y", ctypes.c_void_p), ("grad_y", ctypes.c_void_p), ("grad_y_stride", ctypes.c_uint64),
                ("grad_x", ctypes.c_void_p), ("grad_weights", ctypes.c_void_p), ("workspace", ctypes.c_void_p),
                ("workspace_bytes", ctypes.c_uint64)]


class Attention(ctypes.Structure):
    """struct emrs_attention"""

    _fields_ = [("dtype", ctypes.c_uint32), ("causal", ctypes.c_uint32), ("heads", ctypes.c_uint32),
                ("kv_heads", ctypes.c_uint32), ("dim", ctypes.c_uint32), ("offset_bytes", ctypes.c_uint32),
                ("rows", ctypes.c_uint64), ("key_rows", ctypes.c_uint64), ("documents", ctypes.c_uint64),
                ("offsets", ctypes.c_void_p), ("key_offsets", ctypes.c_void_p),
                ("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("q_strides", ctypes.c_uint64 * 2), ("k_strides", ctypes.c_uint64 * 2), ("v_strides", ctypes.c_uint64 * 2),
                ("scale", ctypes.c_float), ("reserved", ctypes.c_uint32), ("out", ctypes.c_void_p), ("out_rest", ctypes.c_void_p),
                ("lse", ctypes.c_void_p), ("grad_out", ctypes.c_void_p), ("grad_out_strides", ctypes.c_uint64 * 2), ("grad_q", ctypes.c_void_p),
                ("grad_k", ctypes.c_void_p), ("grad_v", ctypes.c_void_p), ("workspace", ctypes.c_void_p),
                ("workspace_bytes", ctypes.c_uint64)]


EMRS_FP32, EMRS_BF16, EMRS_FP16 = 0, 1, 2
EMRS_NORM_GATE_NONE, EMRS_NORM_GATE_CHANNEL, EMRS_NORM_GATE_TOKEN = 0, 1, 2
EMRS_NORM_MAX_HIDDEN = 16384
EMRS_EXPERTS_MAX = 256
EMRS_ATTENTION_MAX_DIM = 128
EMRS_LOSS_MAX_SHARDS = 64
EMRS_MUON_MAX_MATRICES = 32
EMRS_MUON_MAX_STEPS = 16

_lib: Optional[ctypes.CDLL] = None


def load(path: str = LIB_PATH) -> ctypes.CDLL:
    """Load libemrs; raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise RuntimeError(
            f"libemrs is not built ({path} missing); run __graft_entry__.build() or "
            "python -m elasticmegatron_amd.build")
    lib = ctypes.CDLL(path)
    P, U64, U32, I = ctypes.c_void_p, ctypes.c_uint64, ctypes.c_uint32, ctypes.c_int
    lib.emrs_last_error.restype = ctypes.c_char_p
    lib.emrs_last_error.argtypes = []
    lib.emrs_abi_version.restype = I
    lib.emrs_device_count.restype = I
    lib.emrs_plan_create.restype = I
    lib.emrs_plan_create.argtypes = [P, U64, P, U32, P, U32, U32, ctypes.POINTER(P)]
    lib.emrs_plan_stats_get.restype = I
    lib.emrs_plan_stats_get.argtypes = [P, ctypes.POINTER(PlanStats)]
    lib.emrs_plan_execute.restype = I
    lib.emrs_plan_execute.argtypes = [P, P, P, P]
    lib.emrs_plan_prepare.restype = I
    lib.emrs_plan_prepare.argtypes = [P, P]
    lib.emrs_plan_destroy.restype = I
    lib.emrs_plan_destroy.argtypes = [P]
    lib.emrs_get_tuning.restype = I
    lib.emrs_get_tuning.argtypes = [ctypes.POINTER(Tuning)]
    lib.emrs_set_tuning.restype = I
    lib.emrs_set_tuning.argtypes = [ctypes.POINTER(Tuning)]
    lib.emrs_synth_fill.restype = I
    lib.emrs_synth_fill.argtypes = [P, U64, P, P, U32, U64, P]
    lib.emrs_synth_verify.restype = I
    lib.emrs_synth_verify.argtypes = [P, U64, P, P, U32, U64, P, ctypes.POINTER(U64), ctypes.POINTER(U64)]
    lib.emrs_plan_compare.restype = I
    lib.emrs_plan_compare.argtypes = [P, P, P, P, P, U32, P, P]
    lib.emrs_plan_compare_static.restype = I
    lib.emrs_plan_compare_static.argtypes = [P, P, P, P, P, U32, P, P]
    lib.emrs_xor_checksum.restype = I
    lib.emrs_xor_checksum.argtypes = [P, U64, P, P]
    lib.emrs_ipc_export.restype = I
    lib.emrs_ipc_export.argtypes = [P, U64, P]
    lib.emrs_ipc_open.restype = I
    lib.emrs_ipc_open.argtypes = [P, ctypes.POINTER(P)]
    lib.emrs_ipc_close.restype = I
    lib.emrs_ipc_close.argtypes = [P]
    lib.emrs_ipc_open_count.restype = I
    lib.emrs_ipc_open_count.argtypes = []
    lib.emrs_loss_workspace.restype = I
    lib.emrs_loss_workspace.argtypes = [ctypes.POINTER(Loss), I, ctypes.POINTER(U64)]
    lib.emrs_muon_workspace.restype = I
    lib.emrs_muon_workspace.argtypes = [ctypes.POINTER(Muon), ctypes.POINTER(U64)]
    lib.emrs_norm_workspace.restype = I
    lib.emrs_norm_workspace.argtypes = [ctypes.POINTER(Norm), ctypes.POINTER(U64)]
    lib.emrs_attention_workspace.restype = I
    lib.emrs_attention_workspace.argtypes = [ctypes.POINTER(Attention), I, ctypes.POINTER(U64)]
    lib.emrs_experts_workspace.restype = I
    lib.emrs_experts_workspace.argtypes = [ctypes.POINTER(Experts), I, ctypes.POINTER(U64)]
    for fn, record in ((lib.emrs_loss_forward, Loss), (lib.emrs_loss_backward, Loss), (lib.emrs_muon_step, Muon),
                       (lib.emrs_adamw_step, AdamW), (lib.emrs_norm_forward, Norm), (lib.emrs_norm_backward, Norm),
                       (lib.emrs_experts_forward, Experts), (lib.emrs_experts_backward, Experts),
                       (lib.emrs_attention_forward, Attention), (lib.emrs_attention_backward, Attention)):
        fn.restype = I
        fn.argtypes = [ctypes.POINTER(record), P]
    if lib.emrs_abi_version() != 8:
        raise RuntimeError("libemrs ABI version mismatch")
    _lib = lib
    return lib


def _check(rc: int, where: str) -> None:
    if rc != EMRS_OK:
        raise EmrsError(rc, where, load().emrs_last_error().decode(errors="replace"))


def _u64_buffer(vals: Sequence[int]) -> np.ndarray:
    a = np.array(vals if len(vals) else [0], dtype=np.uint64)
    if a.ndim != 1:
        raise ValueError("expected a flat sequence of integers")
    return a


def _ptr_array(ptrs: Sequence[int]):
    """A C array of device pointers over one buffer (no per-element ctypes objects: a per-tensor plan
    passes thousands).  The array keeps the buffer alive.  Of a list of 900 integers array.array makes
    it in 39 us where numpy takes 64; what it does not take, numpy converts or refuses."""
    if type(ptrs) is list and ptrs:
        try:
            a = array.array("Q", ptrs)
            return (ctypes.c_void_p * len(ptrs)).from_buffer(a)
        except (TypeError, OverflowError):
            pass
    a = _u64_buffer(ptrs)
    return (ctypes.c_void_p * a.size).from_buffer(a)


def _u64_array(vals: Sequence[int]):
    a = _u64_buffer(vals)
    return (ctypes.c_uint64 * a.size).from_buffer(a)


def device_count() -> int:
    return int(load().emrs_device_count())


def get_tuning() -> Tuning:
    t = Tuning()
    _check(load().emrs_get_tuning(ctypes.byref(t)), "emrs_get_tuning")
    return t


def set_tuning(blocks_per_cu: int = 0, nontemporal: bool = True, xcd_remap: int = 1, run: int = 4,
               persistent: bool = False, lanes: int = 0, units: int = 1, buffer_ops: bool = False,
               chunk_index: bool = True, warm_tables: bool = True) -> None:
    """Launch shape of every later execution.  The default runs one workgroup of ``lanes`` lanes
    (0: 64) with ``units`` 16-byte units each (0: a whole chunk of 256 units per workgroup) per piece
    of a chunk, each finding its segment in the plan's chunk table (``chunk_index``; False: by a
    bounded binary search); ``persistent=True`` selects a persistent grid, which ``blocks_per_cu``
    and ``run`` shape.  ``xcd_remap`` 1 (or True) has each of the 8 XCDs work through runs of
    consecutive chunks, 2 through one eighth of the pieces (the persistent grid: an eighth of the chunks
    for both); 0 (or False) keeps the hardware's order.  ``warm_tables``: with the chunk table, the first
    workgroups of each copy launch read it and the segment descriptors, so that a launch after unrelated
    work starts from cached tables."""
    t = Tuning(blocks_per_cu, 1 if nontemporal else 0, int(xcd_remap), run, 1 if persistent else 0, lanes,
               units, 1 if buffer_ops else 0, 1 if chunk_index else 0, 1 if warm_tables else 0)
    _check(load().emrs_set_tuning(ctypes.byref(t)), "emrs_set_tuning")


class Plan:
    """An uploaded-on-demand copy plan (emrs_plan)."""

    def __init__(self, segments: np.ndarray, src_buf_bytes: Sequence[int], dst_buf_bytes: Sequence[int],
                 check_disjoint: bool = False):
        lib = load()
        segs = np.ascontiguousarray(segments, dtype=SEGMENT_DTYPE)
        self._handle = ctypes.c_void_p()
        self.n_src = len(src_buf_bytes)
        self.n_dst = len(dst_buf_bytes)
        sb, db = _u64_array(src_buf_bytes), _u64_array(dst_buf_bytes)
        rc = lib.emrs_plan_create(segs.ctypes.data if len(segs) else None, len(segs), sb, self.n_src,
                                  db, self.n_dst, EMRS_PLAN_CHECK_DISJOINT if check_disjoint else 0,
                                  ctypes.byref(self._handle))
        _check(rc, "emrs_plan_create")

    def stats(self) -> PlanStats:
        st = PlanStats()
        _check(load().emrs_plan_stats_get(self._handle, ctypes.byref(st)), "emrs_plan_stats_get")
        return st

    def execute(self, src_ptrs: Sequence[int], dst_ptrs: Sequence[int], stream: int = 0) -> None:
        if len(src_ptrs) != self.n_src or len(dst_ptrs) != self.n_dst:
            raise ValueError("wrong number of base pointers")
        rc = load().emrs_plan_execute(self._handle, _ptr_array(src_ptrs), _ptr_array(dst_ptrs),
                                      ctypes.c_void_p(int(stream)))
        _check(rc, "emrs_plan_execute")

    def prepare(self, stream: int = 0) -> None:
        """Upload the plan's tables to the current device now (emrs_plan_prepare), so that its first
        execution there runs as fast as later ones."""
        _check(load().emrs_plan_prepare(self._handle, ctypes.c_void_p(int(stream))), "emrs_plan_prepare")

    def compare(self, src_ptrs: Sequence[int], dst_ptrs: Sequence[int], groups: Optional[np.ndarray] = None,
                aux_groups: Optional[np.ndarray] = None, n_groups: int = 1, stream: int = 0,
                no_alloc: bool = False) -> np.ndarray:
        """emrs_plan_compare: per group, how the destination differs from what the plan writes.

        ``groups`` / ``aux_groups`` hold one group id per input segment.
        Returns ``n_groups`` records of :data:`COMPARE_DTYPE`.  Waits for ``stream``.
        ``no_alloc``: run emrs_plan_compare_static, which allocates no device memory (its
        working set must fit in EMRS_STATIC_SCRATCH_BYTES).
        """
        if len(src_ptrs) != self.n_src or len(dst_ptrs) != self.n_dst:
            raise ValueError("wrong number of base pointers")
        n_in = self.stats().n_segments
        arrs = []
        for g in (groups, aux_groups):
            if g is None:
                arrs.append(None)
                continue
            g = np.ascontiguousarray(g, dtype=np.uint32)
            if g.shape != (n_in,):
                raise ValueError(f"need one group id per segment ({n_in})")
            arrs.append(g)
        out = np.zeros(max(1, n_groups), dtype=COMPARE_DTYPE)
        fn = load().emrs_plan_compare_static if no_alloc else load().emrs_plan_compare
        rc = fn(self._handle, _ptr_array(src_ptrs), _ptr_array(dst_ptrs),
                arrs[0].ctypes.data if arrs[0] is not None and n_in else None,
                arrs[1].ctypes.data if arrs[1] is not None and n_in else None,
                int(n_groups), out.ctypes.data, ctypes.c_void_p(int(stream)))
        _check(rc, "emrs_plan_compare_static" if no_alloc else "emrs_plan_compare")
        return out

    def close(self) -> None:
        if getattr(self, "_handle", None):
            load().emrs_plan_destroy(self._handle)
            self._handle = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def synth_fill(pieces: np.ndarray, ptrs: Sequence[int], buf_bytes: Sequence[int], seed: int, stream: int = 0) -> None:
    pcs = np.ascontiguousarray(pieces, dtype=PIECE_DTYPE)
    rc = load().emrs_synth_fill(pcs.ctypes.data if len(pcs) else None, len(pcs), _ptr_array(ptrs),
                                _u64_array(buf_bytes), len(ptrs), int(seed), ctypes.c_void_p(int(stream)))
    _check(rc, "emrs_synth_fill")


def xor_checksum(ptr: int, nbytes: int, out_ptr: int, stream: int = 0) -> None:
    """Enqueue the XOR of every 32-bit word of device memory [ptr, ptr + nbytes) into the device
    word at ``out_ptr``."""
    rc = load().emrs_xor_checksum(ctypes.c_void_p(int(ptr)), int(nbytes), ctypes.c_void_p(int(out_ptr)),
                                  ctypes.c_void_p(int(stream)))
    _check(rc, "emrs_xor_checksum")


def synth_verify(pieces: np.ndarray, ptrs: Sequence[int], buf_bytes: Sequence[int], seed: int,
                 stream: int = 0):
    """(mismatching elements, first bad (piece index, element index) or None)."""
    pcs = np.ascontiguousarray(pieces, dtype=PIECE_DTYPE)
    bad, first = ctypes.c_uint64(0), ctypes.c_uint64(0)
    rc = load().emrs_synth_verify(pcs.ctypes.data if len(pcs) else None, len(pcs), _ptr_array(ptrs),
                                  _u64_array(buf_bytes), len(ptrs), int(seed), ctypes.c_void_p(int(stream)),
                                  ctypes.byref(bad), ctypes.byref(first))
    _check(rc, "emrs_synth_verify")
    f = first.value
    return int(bad.value), (None if f == 2 ** 64 - 1 else (f >> 40, f & ((1 << 40) - 1)))


# struct emrs_ipc_buffer: an exported buffer, as plain bytes that travel between processes.
IPC_BUFFER_DTYPE = np.dtype([("handle", "u1", (64,)), ("offset", "<u8"), ("bytes", "<u8"),
                             ("allocation_bytes", "<u8"), ("device", "<i4"), ("reserved", "<u4")])
assert IPC_BUFFER_DTYPE.itemsize == 96
EMRS_IPC_MAX_ALLOCATION_BYTES = 2 << 30  # exclusive


def ipc_export(ptr: int, nbytes: int) -> np.ndarray:
    """emrs_ipc_export: the record describing device buffer [ptr, ptr + nbytes) to another process."""
    rec = np.zeros(1, dtype=IPC_BUFFER_DTYPE)
    _check(load().emrs_ipc_export(ctypes.c_void_p(int(ptr)), int(nbytes), rec.ctypes.data), "emrs_ipc_export")
    return rec[0]


def ipc_open(record) -> int:
    """emrs_ipc_open: map an exported buffer on the current device; returns its address."""
    rec = np.ascontiguousarray(np.asarray(record, dtype=IPC_BUFFER_DTYPE).reshape(1))
    out = ctypes.c_void_p()
    _check(load().emrs_ipc_open(rec.ctypes.data, ctypes.byref(out)), "emrs_ipc_open")
    return int(out.value)


def ipc_close(ptr: int) -> None:
    """emrs_ipc_close: drop one reference that :func:`ipc_open` returned."""
    _check(load().emrs_ipc_close(ctypes.c_void_p(int(ptr))), "emrs_ipc_close")


def ipc_open_count() -> int:
    """Allocations this process holds open through :func:`ipc_open`."""
    return int(load().emrs_ipc_open_count())


# ----- operators of a training step -----


def loss_workspace(a: Loss, backward: bool) -> int:
    """emrs_loss_workspace: bytes of workspace that the call wants."""
    n = ctypes.c_uint64()
    _check(load().emrs_loss_workspace(ctypes.byref(a), 1 if backward else 0, ctypes.byref(n)), "emrs_loss_workspace")
    return int(n.value)


def loss_forward(a: Loss, stream: int = 0) -> None:
    _check(load().emrs_loss_forward(ctypes.byref(a), ctypes.c_void_p(int(stream))), "emrs_loss_forward")


def loss_backward(a: Loss, stream: int = 0) -> None:
    _check(load().emrs_loss_backward(ctypes.byref(a), ctypes.c_void_p(int(stream))), "emrs_loss_backward")


def muon_workspace(a: Muon) -> int:
    """emrs_muon_workspace: bytes of workspace that the call wants."""
    n = ctypes.c_uint64()
    _check(load().emrs_muon_workspace(ctypes.byref(a), ctypes.byref(n)), "emrs_muon_workspace")
    return int(n.value)


def muon_step(a: Muon, stream: int = 0) -> None:
    _check(load().emrs_muon_step(ctypes.byref(a), ctypes.c_void_p(int(stream))), "emrs_muon_step")


def adamw_step(a: AdamW, stream: int = 0) -> None:
    _check(load().emrs_adamw_step(ctypes.byref(a), ctypes.c_void_p(int(stream))), "emrs_adamw_step")


def norm_workspace(a: Norm) -> int:
    """emrs_norm_workspace: bytes of workspace that backward wants."""
    n = ctypes.c_uint64()
    _check(load().emrs_norm_workspace(ctypes.byref(a), ctypes.byref(n)), "emrs_norm_workspace")
    return int(n.value)


def norm_forward(a: Norm, stream: int = 0) -> None:
    rc = (_lib or load()).emrs_norm_forward(ctypes.byref(a), stream)
    if rc:
        _check(rc, "emrs_norm_forward")


def norm_backward(a: Norm, stream: int = 0) -> None:
    rc = (_lib or load()).emrs_norm_backward(ctypes.byref(a), stream)
    if rc:
        _check(rc, "emrs_norm_backward")


def experts_workspace(a: Experts, backward: bool) -> int:
    """emrs_experts_workspace: bytes of workspace that the call wants, 0 for none."""
    n = ctypes.c_uint64()
    _check(load().emrs_experts_workspace(ctypes.byref(a), 1 if backward else 0, ctypes.byref(n)), "emrs_experts_workspace")
    return int(n.value)


def experts_forward(a: Experts, stream: int = 0) -> None:
    rc = (_lib or load()).emrs_experts_forward(ctypes.byref(a), stream)
    if rc:
        _check(rc, "emrs_experts_forward")


def experts_backward(a: Experts, stream: int = 0) -> None:
    rc = (_lib or load()).emrs_experts_backward(ctypes.byref(a), stream)
    if rc:
        _check(rc, "emrs_experts_backward")


def attention_workspace(a: Attention, backward: bool) -> int:
    """emrs_attention_workspace: bytes of workspace that the call wants, 0 for none."""
    n = ctypes.c_uint64()
    _check(load().emrs_attention_workspace(ctypes.byref(a), 1 if backward else 0, ctypes.byref(n)), "emrs_attention_workspace")
    return int(n.value)


def attention_forward(a: Attention, stream: int = 0) -> None:
    rc = (_lib or load()).emrs_attention_forward(ctypes.byref(a), stream)
    if rc:
        _check(rc, "emrs_attention_forward")


def attention_backward(a: Attention, stream: int = 0) -> None:
    rc = (_lib or load()).emrs_attention_backward(ctypes.byref(a), stream)
    if rc:
        _check(rc, "emrs_attention_backward")
