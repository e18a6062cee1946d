"""What the operators of a training step refuse of tensors on the GPU."""

import pytest
import torch

from elasticmegatron_amd import training

pytestmark = pytest.mark.gpu


def _z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype, device="cuda")


BF16, FP16, I64 = torch.bfloat16, torch.float16, torch.int64


def test_loss_refuses(gpu_device):
    h, w, t = _z(4, 8, dtype=BF16), _z(10, 8, dtype=BF16), _z(4, dtype=I64)
    f = training.linear_cross_entropy
    for error, call in [
        (TypeError, lambda: f(h.float(), w.float(), t)),
        (TypeError, lambda: f(h, w.half(), t)),
        (TypeError, lambda: f(h, w, t.int())),
        (ValueError, lambda: f(h, w, t[:3])),
        (ValueError, lambda: f(h, w[:, :7], t)),
        (ValueError, lambda: f(h, w[0], t)),
        (ValueError, lambda: f(h, [], t)),
        (ValueError, lambda: f(h, [w] * 65, t)),
        (ValueError, lambda: f(h, w, t, reduction="median")),
        (ValueError, lambda: f(h, w, t, vocab_size=-1)),
        (ValueError, lambda: f(h, w.cpu(), t)),
        (ValueError, lambda: training.vocab_statistics(h, w, t, vocab_start=-1)),
        (ValueError, lambda: training.vocab_gradients(h, w, t, _z(3), _z(4))),
        (ValueError, lambda: training.vocab_gradients(h, w, t, _z(4), _z(4).cpu())),
    ]:
        with pytest.raises(error):
            call()
    assert f(h, w, t).isfinite()  # and what it takes still runs


def test_no_second_derivative(gpu_device):
    h, w, t = torch.ones(4, 8, dtype=BF16, device="cuda", requires_grad=True), _z(10, 8, dtype=BF16), _z(4, dtype=I64)
    g, = torch.autograd.grad(training.linear_cross_entropy(h, w, t), h, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), h)


def test_muon_refuses(gpu_device):
    m, b, g = _z(6, 8), _z(6, 8), _z(6, 8)
    f = training.muon_step
    for error, call in [
        (TypeError, lambda: f(m.half(), b, g, lr=0.1)),
        (TypeError, lambda: f(m, b.to(BF16), g, lr=0.1)),
        (TypeError, lambda: f(m, b, g.double(), lr=0.1)),
        (TypeError, lambda: f(m, b, g, model=_z(6, 8, dtype=FP16), lr=0.1)),
        (ValueError, lambda: f(m, b, g[:5], lr=0.1)),
        (ValueError, lambda: f([m, m], [b, b], [g], lr=0.1)),
        (ValueError, lambda: f([m], [b], [], lr=0.1)),
        (ValueError, lambda: f([m, _z(6, 9)], [b, b], [g, g], lr=0.1)),
        (TypeError, lambda: training.orthogonalise([g, g.to(BF16)])),
        (ValueError, lambda: f(_z(8, 6).t(), b, g, lr=0.1)),           # written in place: rows are wanted
        (ValueError, lambda: f(m, _z(1, 8).expand(6, 8), g, lr=0.1)),
        (ValueError, lambda: f(m, b, g, lr=0.1, steps=0)),
        (ValueError, lambda: f(m, b, g, lr=0.1, coefficients=[(1, 2, 3)] * 4)),
        (ValueError, lambda: f(_z(48), b, g, lr=0.1)),
        (ValueError, lambda: f(m.cpu(), b, g, lr=0.1)),
    ]:
        with pytest.raises(error):
            call()
    f(m, b, g, lr=0.1)


def test_adamw_refuses(gpu_device):
    w, m, v, g = (_z(12) for _ in range(4))
    f = training.adamw_step
    for error, call in [
        (TypeError, lambda: f(w.half(), m, v, g, lr=0.1, step=1)),
        (TypeError, lambda: f(w, m, v, g.double(), lr=0.1, step=1)),
        (TypeError, lambda: f(w, m, v, g, model=_z(12), lr=0.1, step=1)),
        (ValueError, lambda: f(w, m[:11], v, g, lr=0.1, step=1)),
        (ValueError, lambda: f(_z(24)[::2], m, v, g, lr=0.1, step=1)),
        (ValueError, lambda: f(w, m, v, g, lr=0.1, step=0)),
        (ValueError, lambda: f(w, m, v, g.cpu(), lr=0.1, step=1)),
    ]:
        with pytest.raises(error):
            call()
    f(w, m, v, _z(24)[::2], lr=0.1, step=1)  # a strided gradient is only read
