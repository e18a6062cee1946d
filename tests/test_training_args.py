"""What the operators of a training step refuse, before any work reaches a device (no GPU needed)."""

import ctypes

import pytest
import torch

from elasticmegatron_amd import _native, training


def _table(*values):
    return (ctypes.c_uint64 * len(values))(*values)


def _loss(**kw):
    """A valid call's record (its addresses are never read), with ``kw`` over it."""
    keep = dict(weights=_table(0x10000, 0x20000), weight_strides=_table(64, 64), shard_rows=_table(100, 50))
    keep.update({k: v for k, v in kw.items() if k in keep})
    fields = dict(dtype=_native.EMRS_BF16, n_shards=2, tokens=10, hidden_size=64, hidden=0x30000, hidden_stride=64,
                  vocab_start=0, vocab_size=150, target=0x40000, ignore_index=-100, lse=0x50000, target_logit=0x60000,
                  loss=0x70000, grad_loss=0x80000, grad_hidden=0x90000, workspace=0x100000, workspace_bytes=1 << 40)
    fields.update({k: v for k, v in kw.items() if k not in keep})
    a = _native.Loss()
    for k, v in fields.items():
        setattr(a, k, v)
    for k, v in keep.items():
        setattr(a, k, None if v is None else ctypes.addressof(v))
    a._keep = keep
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=0), -1), (dict(dtype=7), -1),
    (dict(n_shards=0), -1), (dict(n_shards=65), -1),
    (dict(weights=None), -1), (dict(shard_rows=None), -1), (dict(weight_strides=None), -1),
    (dict(weights=_table(0, 0x20000)), -1),
    (dict(weights=_table(0x10001, 0x20000)), -3),
    (dict(hidden_size=0), -10), (dict(hidden_size=1 << 21), -10),
    (dict(tokens=(1 << 21) + 1), -10),
    (dict(hidden_stride=63), -1), (dict(hidden_stride=1 << 22), -1),
    (dict(weight_strides=_table(64, 63)), -1),
    (dict(shard_rows=_table(1 << 31, 1)), -10),
    (dict(hidden=0), -1), (dict(target=0), -1), (dict(hidden=0x30001), -3), (dict(target=0x40004), -3),
    (dict(lse=0), -1), (dict(target_logit=0), -1),
    (dict(workspace_bytes=100), -1), (dict(workspace=0), -1), (dict(workspace=0x100010), -3),
])
def test_loss_refuses(kw, code):
    with pytest.raises(_native.EmrsError) as e:
        _native.loss_forward(_loss(**kw))
    assert e.value.code == code


@pytest.mark.parametrize("kw,code", [(dict(grad_loss=0), -1), (dict(lse=0), -1), (dict(tokens=0), -1),
                                     (dict(shard_rows=_table(0, 0)), -1), (dict(workspace_bytes=100), -1)])
def test_loss_backward_refuses(kw, code):
    with pytest.raises(_native.EmrsError) as e:
        _native.loss_backward(_loss(**kw))
    assert e.value.code == code


def test_loss_workspace_keeps_no_logits():
    """Less than the logits of 4096 tokens and 128256 rows in 16 bits (1.05 GB), forward by far."""
    a = _loss(n_shards=1, tokens=4096, hidden_size=4096, hidden_stride=4096, weight_strides=_table(4096),
              shard_rows=_table(128256), vocab_size=128256)
    assert _native.loss_workspace(a, False) < 64 << 20
    assert _native.loss_workspace(a, True) < 512 << 20


def _muon(**kw):
    names = ("grad", "momentum", "main", "image", "out")
    tables = dict(grad=_table(0x10000, 0x20000), momentum=_table(0x30000, 0x40000), main=_table(0x50000, 0x60000),
                  image=_table(0x70000, 0x80000), out=None)
    tables.update({k: v for k, v in kw.items() if k in names})
    coefficients = (ctypes.c_float * 15)(*([3.4445, -4.775, 2.0315] * 5))
    fields = dict(count=2, grad_dtype=0, rows=10, cols=20, steps=5, nesterov=1, mu=0.9, eps=1e-7, decay=0.0, rate=0.1,
                  workspace=0x1000000, workspace_bytes=1 << 40, coefficients=ctypes.addressof(coefficients))
    fields.update({k + "_stride": 20 for k in names})
    fields.update({k: v for k, v in kw.items() if k not in names})
    a = _native.Muon()
    for k, v in fields.items():
        setattr(a, k, v)
    for k, v in tables.items():
        setattr(a, k, None if v is None else ctypes.addressof(v))
    a._keep = (tables, coefficients)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(count=0), -1), (dict(count=33), -1), (dict(grad_dtype=3), -1),
    (dict(rows=0), -10), (dict(cols=0), -10), (dict(rows=(1 << 20) + 1), -10), (dict(rows=40000, cols=40000), -10),
    (dict(steps=0), -1), (dict(steps=17), -1), (dict(coefficients=0), -1),
    (dict(grad=None), -1), (dict(main=None, image=None), -1), (dict(main=None, out=None), -1),
    (dict(out=_table(0x90000, 0xa0000)), -1),             # out and main together
    (dict(main=None, out=_table(0x90000, 0xa0000)), -1),  # an image without main
    (dict(grad_stride=19), -1), (dict(main_stride=19), -1), (dict(image_stride=0), -1),
    (dict(grad=_table(0x10000, 0)), -1), (dict(grad=_table(0x10002, 0x20000)), -3), (dict(momentum=_table(0x30001, 0x40000)), -3),
    (dict(workspace_bytes=1000), -1), (dict(workspace=0x1000080), -3),
])
def test_muon_refuses(kw, code):
    with pytest.raises(_native.EmrsError) as e:
        _native.muon_step(_muon(**kw))
    assert e.value.code == code


def _adamw(**kw):
    fields = dict(n=100, main=0x10000, exp_avg=0x20000, exp_avg_sq=0x30000, grad=0x40000, grad_dtype=0, step=1, image=0x50000,
                  lr=0.1, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0)
    fields.update(kw)
    a = _native.AdamW()
    for k, v in fields.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(grad_dtype=3), -1), (dict(step=0), -1), (dict(beta1=1.0), -1), (dict(beta2=-0.1), -1), (dict(beta1=float("nan")), -1),
    (dict(n=1 << 39), -10), (dict(main=0), -1), (dict(grad=0), -1), (dict(main=0x10002), -3), (dict(grad=0x40002), -3),
    (dict(image=0x50001), -3),
])
def test_adamw_refuses(kw, code):
    with pytest.raises(_native.EmrsError) as e:
        _native.adamw_step(_adamw(**kw))
    assert e.value.code == code
    _native.adamw_step(_adamw(n=0))  # nothing to do


def test_null_records_and_no_device():
    lib = _native.load()
    n = ctypes.c_uint64()
    assert lib.emrs_loss_workspace(None, 0, ctypes.byref(n)) == -1
    assert lib.emrs_loss_workspace(ctypes.byref(_loss()), 0, None) == -1
    assert lib.emrs_loss_forward(None, None) == lib.emrs_loss_backward(None, None) == -1
    assert lib.emrs_muon_workspace(None, ctypes.byref(n)) == lib.emrs_muon_step(None, None) == -1
    assert lib.emrs_adamw_step(None, None) == -1
    if _native.device_count() == 0:
        for call, a in ((_native.loss_forward, _loss()), (_native.loss_backward, _loss()), (_native.muon_step, _muon()),
                        (_native.adamw_step, _adamw())):
            with pytest.raises(_native.EmrsError) as e:
                call(a)
            assert e.value.code == -6


def test_tensors_have_to_be_on_a_gpu():
    h, w, t = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(10, 8, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    m = torch.zeros(4, 4)
    for call in (lambda: training.linear_cross_entropy(h, w, t), lambda: training.vocab_statistics(h, w, t),
                 lambda: training.vocab_gradients(h, w, t, torch.zeros(4), torch.zeros(4)),
                 lambda: training.orthogonalise(m), lambda: training.muon_step(m, m.clone(), m.clone(), lr=0.1),
                 lambda: training.adamw_step(m, m.clone(), m.clone(), m.clone(), lr=0.1, step=1)):
        with pytest.raises(ValueError, match="a GPU is wanted"):
            call()


def test_arguments_that_are_no_tensors():
    with pytest.raises(TypeError):
        training.linear_cross_entropy([1.0], [2.0], [3])
    with pytest.raises(TypeError):
        training.adamw_step(1.0, 2.0, 3.0, 4.0, lr=0.1, step=1)
    with pytest.raises(TypeError):
        training.orthogonalise([1.0, 2.0])
