"""What the layers' operators refuse, before any work reaches a device (no GPU needed)."""

import ctypes
import math

import pytest
import torch
from torch.autograd import forward_ad

from elasticmegatron_amd import _native, training


def _record(kind, fields, kw):
    a = kind()
    keep = []
    for k, v in {**fields, **kw}.items():
        if k.endswith("strides"):
            getattr(a, k)[:] = v
        elif isinstance(v, list):
            table = (ctypes.c_uint64 * len(v))(*v)
            keep.append(table)
            setattr(a, k, ctypes.addressof(table))
        else:
            setattr(a, k, v)
    a._keep = keep
    return a


def _norm(**kw):
    """A valid call's record (its addresses are never read), with ``kw`` over it."""
    return _record(_native.Norm, dict(
        dtype=_native.EMRS_BF16, residual_dtype=_native.EMRS_FP32, gate_kind=_native.EMRS_NORM_GATE_CHANNEL, tokens=10, hidden=64,
        residual=0x10000, residual_stride=64, branch=0x20000, branch_stride=64, gate=0x30000, gate_stride=64, branch_weight=0x40000, weight=0x50000,
        residual_scale=1.0, eps=1e-5, stream=0x60000, stream_stride=64, normed=0x70000, stream_rms=0x80000, branch_rms=0x90000, grad_stream=0xa0000,
        grad_normed=0xb0000, grad_residual=0xc0000, grad_branch=0xd0000, grad_gate=0xe0000, grad_weight=0xf0000, grad_branch_weight=0x100000,
        workspace=0x200000, workspace_bytes=1 << 40), kw)


BOTH = [
    (dict(dtype=0), -1), (dict(dtype=3), -1), (dict(residual_dtype=2), -1), (dict(gate_kind=3), -1),
    (dict(hidden=0), -10), (dict(hidden=16385), -10), (dict(tokens=1 << 31), -10),
    (dict(branch=0), -1), (dict(gate=0), -1), (dict(branch_stride=63), -1), (dict(gate_kind=2, gate_stride=63), -1),
    (dict(reserved=1), -1), (dict(branch=0x20001), -3), (dict(gate=0x30001), -3), (dict(weight=0x50001), -3), (dict(stream=0x60002), -3), (dict(stream_rms=0x80002), -3),
]


@pytest.mark.parametrize("kw,code", BOTH + [
    (dict(residual=0), -1), (dict(residual_stride=63), -1), (dict(weight=0), -1), (dict(stream=0, normed=0), -1), (dict(residual=0x10002), -3),
])
def test_norm_forward_refuses(kw, code):
    with pytest.raises(_native.EmrsError) as e:
        _native.norm_forward(_norm(**kw))
    assert e.value.code == code


@pytest.mark.parametrize("kw,code", BOTH + [
    (dict(grad_stream=0, grad_normed=0), -1), (dict(weight=0), -1), (dict(stream=0), -1), (dict(stream_rms=0), -1), (dict(stream_stride=63), -1),
    (dict(branch_rms=0), -1), (dict(grad_normed=0), -1), (dict(branch_weight=0), -1), (dict(gate_kind=0), -1),
    (dict(grad_stream=0xa0002), -3), (dict(grad_residual=0xc0002), -3), (dict(grad_weight=0xf0001), -3),
    (dict(workspace=0), -1), (dict(workspace_bytes=100), -1), (dict(workspace=0x200010), -3), (dict(tokens=0), -1),
])
def test_norm_backward_refuses(kw, code):
    with pytest.raises(_native.EmrsError) as e:
        _native.norm_backward(_norm(**kw))
    assert e.value.code == code


def _experts(**kw):
    return _record(_native.Experts, dict(
        dtype=_native.EMRS_BF16, n_experts=2, rows=10, n_in=64, n_out=32, counts=0x10000, counts_bytes=4, x=0x20000, x_stride=64,
        weights=[0x30000, 0x40000], weight_stride=64, y=0x50000, grad_y=0x60000, grad_y_stride=32, grad_x=0x70000, grad_weights=[0x80000, 0x90000],
        workspace=0x200000, workspace_bytes=1 << 40), kw)


SIZES = [
    (dict(dtype=0), -1), (dict(n_experts=0), -1), (dict(n_experts=257), -1), (dict(rows=(1 << 30) + 1), -10), (dict(rows=1 << 30), -10), (dict(n_in=0), -10),
    (dict(n_out=0), -10), (dict(n_in=(1 << 20) + 1), -10), (dict(counts=0), -1), (dict(counts_bytes=2), -1), (dict(counts=0x10002), -3),
    (dict(weights=None), -1), (dict(weights=[0, 0x40000]), -1), (dict(weights=[0x30001, 0x40000]), -3), (dict(weight_stride=63), -1),
    (dict(weight_stride=(1 << 21) + 1), -1), (dict(x=0), -1), (dict(x=0x20001), -3), (dict(x_stride=63), -1),
    (dict(n_in=63, x_stride=63, weight_stride=63, workspace=0), -1), (dict(n_in=63, x_stride=63, weight_stride=63, workspace=0x200010), -3),
    (dict(x_stride=65, workspace_bytes=100), -1), (dict(reserved=1), -1),
]


@pytest.mark.parametrize("kw,code", SIZES + [(dict(y=0), -1), (dict(y=0x50001), -3)])
def test_experts_forward_refuses(kw, code):
    with pytest.raises(_native.EmrsError) as e:
        _native.experts_forward(_experts(**kw))
    assert e.value.code == code


@pytest.mark.parametrize("kw,code", SIZES + [
    (dict(grad_y=0), -1), (dict(grad_y=0x60001), -3), (dict(grad_y_stride=31), -1), (dict(grad_x=None, grad_weights=None), -1),
    (dict(grad_weights=[0, 0x90000]), -1), (dict(grad_weights=[0x80001, 0x90000]), -3), (dict(grad_x=0x70001), -3),
])
def test_experts_backward_refuses(kw, code):
    with pytest.raises(_native.EmrsError) as e:
        _native.experts_backward(_experts(**kw))
    assert e.value.code == code


def test_experts_workspace():
    """None where rows lie on 16 bytes and sums are short; copies of what does not; room for the parts of cut tiles."""
    assert _native.experts_workspace(_experts(), False) == _native.experts_workspace(_experts(), True) == 0
    assert _native.experts_workspace(_experts(n_in=63, x_stride=63, weight_stride=63), False) == 10 * 64 * 2 + 2 * 32 * 64 * 2
    assert _native.experts_workspace(_experts(rows=4096, n_in=8192, x_stride=8192, weight_stride=8192), False) == 64 << 20


def _attention(**kw):
    return _record(_native.Attention, dict(
        dtype=_native.EMRS_BF16, causal=1, heads=4, kv_heads=2, dim=64, offset_bytes=4, rows=10, key_rows=12, documents=2, offsets=0x10000,
        key_offsets=0x20000, q=0x30000, k=0x40000, v=0x50000, q_strides=(256, 64), k_strides=(128, 64), v_strides=(128, 64), scale=0.125, out=0x60000,
        out_rest=0x68000, lse=0x70000, grad_out=0x80000, grad_out_strides=(256, 64), grad_q=0x90000, grad_k=0xa0000, grad_v=0xb0000,
        workspace=0x200000, workspace_bytes=1 << 40), kw)


SHAPES = [
    (dict(dtype=0), -1), (dict(heads=0), -1), (dict(kv_heads=0), -1), (dict(kv_heads=3), -1), (dict(heads=4098), -10), (dict(dim=0), -10), (dict(dim=129), -10),
    (dict(documents=0), -10), (dict(documents=(1 << 20) + 1), -10), (dict(rows=(1 << 28) + 1), -10), (dict(key_rows=(1 << 28) + 1), -10),
    (dict(scale=0.0), -1), (dict(scale=-1.0), -1), (dict(scale=math.inf), -1), (dict(scale=math.nan), -1),
    (dict(offsets=0), -1), (dict(key_offsets=0), -1), (dict(offset_bytes=2), -1), (dict(offsets=0x10002), -3),
    (dict(offsets=0, key_offsets=0, rows=11), -1), (dict(q=0), -1), (dict(k=0), -1), (dict(v=0), -1), (dict(q=0x30001), -3), (dict(out=0), -1),
    (dict(out=0x60004), -3), (dict(out_rest=0x68004), -3), (dict(lse=0x70002), -3), (dict(q_strides=(1 << 41, 64)), -10),
    (dict(dim=60, workspace=0), -1), (dict(dim=60, workspace_bytes=64), -1), (dict(dim=60, workspace=0x200010), -3),
    (dict(reserved=1), -1), (dict(documents=256, workspace=0), -1), (dict(documents=256, workspace_bytes=128), -1),
]


@pytest.mark.parametrize("kw,code", SHAPES)
def test_attention_forward_refuses(kw, code):
    with pytest.raises(_native.EmrsError) as e:
        _native.attention_forward(_attention(**kw))
    assert e.value.code == code


@pytest.mark.parametrize("kw,code", SHAPES + [
    (dict(grad_out=0), -1), (dict(grad_out=0x80001), -3), (dict(lse=0), -1), (dict(grad_q=None, grad_k=None, grad_v=None), -1), (dict(grad_v=None), -1),
    (dict(grad_q=0x90004), -3), (dict(grad_k=0xa0002), -3), (dict(workspace=0), -1),
])
def test_attention_backward_refuses(kw, code):
    with pytest.raises(_native.EmrsError) as e:
        _native.attention_backward(_attention(**kw))
    assert e.value.code == code


def test_attention_keeps_no_probabilities():
    """8192 queries of 32 heads to as many keys: 4.3 GB of probabilities in 16 bits."""
    a = _attention(heads=32, kv_heads=8, dim=128, rows=8192, key_rows=8192, q_strides=(4096, 128), k_strides=(1024, 128), v_strides=(1024, 128),
                   grad_out_strides=(4096, 128))
    assert _native.attention_workspace(a, False) == 0
    # Two parts of grad_k and of grad_v in 32 bits, and two numbers for each query and head.
    assert _native.attention_workspace(a, True) <= 2 * 2 * (8192 * 8 * 128 * 4) + 2 * (8192 * 32 * 4) + 4096


def test_null_records_and_no_device():
    lib = _native.load()
    n = ctypes.c_uint64()
    for name, two in (("norm", False), ("experts", True), ("attention", True)):
        ask = getattr(lib, f"emrs_{name}_workspace")
        assert (ask(None, 0, ctypes.byref(n)) if two else ask(None, ctypes.byref(n))) == -1
        assert getattr(lib, f"emrs_{name}_forward")(None, None) == getattr(lib, f"emrs_{name}_backward")(None, None) == -1
    assert lib.emrs_norm_workspace(ctypes.byref(_norm()), None) == -1
    if _native.device_count() == 0:
        for call, a in ((_native.norm_forward, _norm()), (_native.norm_backward, _norm()), (_native.experts_forward, _experts()),
                        (_native.experts_backward, _experts()), (_native.attention_forward, _attention()), (_native.attention_backward, _attention())):
            with pytest.raises(_native.EmrsError) as e:
                call(a)
            assert e.value.code == -6
    # Nothing to do needs no device either.
    _native.norm_forward(_norm(tokens=0))
    _native.experts_forward(_experts(rows=0))
    _native.attention_forward(_attention(rows=0))


B = lambda *s: torch.ones(*s, dtype=torch.bfloat16)  # noqa: E731
COUNTS = torch.tensor([2, 2], dtype=torch.int32)
CALLS = {
    "rms_norm, x": lambda d: training.rms_norm(d(B(4, 8)), B(8)),
    "rms_norm, weight": lambda d: training.rms_norm(B(4, 8), d(B(8))),
    "residual_norm, branch": lambda d: training.residual_norm(B(4, 8), d(B(4, 8)), B(8)),
    "residual_norm, gate": lambda d: training.residual_norm(B(4, 8), B(4, 8), gate=d(B(8))),
    "expert_linear, x": lambda d: training.expert_linear(d(B(4, 8)), [B(8, 8)] * 2, COUNTS),
    "expert_linear, weight": lambda d: training.expert_linear(B(4, 8), [B(8, 8), d(B(8, 8))], COUNTS),
    "attention, q": lambda d: training.attention(d(B(4, 2, 8)), B(4, 2, 8), B(4, 2, 8)),
    "attention, v": lambda d: training.attention(B(4, 2, 8), B(4, 2, 8), d(B(4, 2, 8))),
}


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("with_grad", [True, False])
def test_tangents_and_tensors_on_no_gpu(call, with_grad):
    with torch.set_grad_enabled(with_grad), forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            CALLS[call](lambda t: forward_ad.make_dual(t, torch.ones_like(t)))
        with pytest.raises(ValueError, match="a GPU is wanted"):
            CALLS[call](lambda t: t.requires_grad_())


def test_arguments_that_are_no_tensors():
    for call in (lambda: training.rms_norm([1.0], B(8)), lambda: training.rms_norm(B(4, 8), None), lambda: training.residual_norm(1.0, 2.0, 3.0),
                 lambda: training.expert_linear([1.0], [[2.0]], [1]), lambda: training.attention(1.0, 2.0, 3.0)):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(ValueError):
        training.expert_linear(B(4, 8), [], COUNTS)
