"""Newton-Schulz with more steps than usual, and with a triple of its own for each: the polynomials' product
on directions that the matrix does not have is the product of the a, which leaves the 16-bit range."""

import math

import pytest
import torch

from elasticmegatron_amd import training

pytestmark = pytest.mark.gpu

A, B, C = training.MUON_COEFFICIENTS
# Steep at first, p(1) = 1 in the end: the a of the first five are 8.2, 4.1, 3.9, 3.3 and 2.3.
STEEP = [(8.2, -23.4, 17.2), (4.1, -2.95, 0.55), (3.9, -2.9, 0.55), (3.3, -2.48, 0.51), (2.3, -1.67, 0.42)] + [(1.875, -1.25, 0.375)] * 11
# A step's products are off by at most a fifth of what five of them are (their roundings to 16 bits), and
# carry what earlier steps were off by on without growth: singular values gather where |d/ds s p(s)| is about 1.
STEP, BF16 = 2e-3 / 5, 2.0 ** -9


def _newton_schulz(u, coefficients, eps=1e-7):
    x = u.double()
    x = x / (torch.linalg.matrix_norm(x) + eps)
    for a, b, c in coefficients:
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x


def _room(coefficients, rank=None):
    """How far the result may be off in norm.  Directions that a matrix of low rank does not have begin with
    the rounding of X's two parts, 2^-22 of its norm, and grow by every a."""
    noise = 0.0 if rank is None else 2.0 ** -22 * math.prod(a for a, _, _ in coefficients) / math.sqrt(rank)
    return STEP * max(5, len(coefficients)) + BF16 + noise


def _off(got, want):
    return float((got.double() - want).norm() / want.norm())


def _full(rows, cols, seed=0):
    return torch.randn(rows, cols, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def _low(rows, cols, rank):
    """``rank`` equal singular values."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, _ = torch.linalg.qr(torch.randn(rows, rank, generator=gen, device="cuda", dtype=torch.float64))
    p, _ = torch.linalg.qr(torch.randn(cols, rank, generator=gen, device="cuda", dtype=torch.float64))
    return (q @ p.t()).float()


def _schedule(kind, steps):
    return [(A, B, C)] * steps if kind == "same" else STEEP[:steps]


@pytest.mark.parametrize("kind,steps", [("same", 6), ("same", 7), ("same", 8), ("same", 10), ("same", 16),
                                        ("steep", 5), ("steep", 6), ("steep", 7), ("steep", 8), ("steep", 16)])
@pytest.mark.parametrize("rows,cols", [(200, 600), (1300, 260), (192, 640)])
def test_full_rank(gpu_device, rows, cols, kind, steps):
    u, own = _full(rows, cols), _schedule(kind, steps)
    got = training.orthogonalise(u, steps=steps, coefficients=own)
    assert got.isfinite().all()
    assert _off(got, _newton_schulz(u, own)) <= _room(own)


@pytest.mark.parametrize("kind,steps", [("same", 7), ("same", 8), ("same", 10), ("steep", 6), ("steep", 7), ("steep", 8)])
@pytest.mark.parametrize("rows,cols", [(192, 640), (1300, 260)])
def test_low_rank(gpu_device, rows, cols, kind, steps):
    u, own = _low(rows, cols, 16), _schedule(kind, steps)
    got = training.orthogonalise(u, steps=steps, coefficients=own)
    assert got.isfinite().all()
    assert _off(got, _newton_schulz(u, own)) <= _room(own, 16)


def test_update_of_a_matrix_with_rows_of_zeros(gpu_device):
    """Sixteen steps: the weights stay finite, and rows without gradient only decay."""
    grad = _full(256, 1024)
    grad[200:] = 0
    main, momentum = _full(256, 1024, 1), torch.zeros_like(grad)
    before, image = main.clone(), torch.empty(256, 1024, dtype=torch.bfloat16, device="cuda")
    training.muon_step(main, momentum, grad, model=image, lr=0.01, weight_decay=0.5, steps=16)
    assert main.isfinite().all() and image.isfinite().all()
    assert (main[200:] - before[200:] * (1 - 0.005)).abs().le(2.0 ** -22 * before[200:].abs()).all()


def test_one_workspace_serves_any_coefficients(gpu_device):
    """The native call's workspace, asked for without coefficients, is enough for steps of either kind."""
    import ctypes

    from elasticmegatron_amd import _native

    u, out = _full(200, 600), torch.empty(200, 600, dtype=torch.bfloat16, device="cuda")
    a = _native.Muon()
    a.count, a.grad_dtype, a.rows, a.cols, a.steps = 1, _native.EMRS_FP32, 200, 600, 8
    grad, to = (ctypes.c_uint64 * 1)(u.data_ptr()), (ctypes.c_uint64 * 1)(out.data_ptr())
    a.grad, a.grad_stride, a.out, a.out_stride, a.eps = ctypes.addressof(grad), 600, ctypes.addressof(to), 600, 1e-7
    scratch = torch.empty(_native.muon_workspace(a), dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = scratch.data_ptr(), scratch.numel()
    for own in ([(A, B, C)] * 8, [(2.0, -1.5, 0.5)] * 8):
        own_c = (ctypes.c_float * 24)(*(x for r in own for x in r))
        a.coefficients = ctypes.addressof(own_c)
        _native.muon_step(a, torch.cuda.current_stream().cuda_stream)
        assert _off(out, _newton_schulz(u, own)) <= _room(own)
