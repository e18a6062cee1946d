"""Matrices whose sides or bytes are near the ends of 32-bit offsets."""

import pytest
import torch

from elasticmegatron_amd import training
from tests.test_gpu_training_loss import _inputs
from tests.test_gpu_training_muon import BF16, PRODUCTS, _newton_schulz, _off
from tests.test_gpu_training_uneven import _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1, 5, 300])
def test_weights_past_2_to_31_bytes(gpu_device, tokens):
    h, w, target, g = _inputs(tokens, 2048, [600000], torch.bfloat16, ignored=0.0)
    target[-1] = 599999
    _check(h, w[0], target, g)  # with d's smallest step, which rows of so small a probability reach


@pytest.mark.parametrize("rows,cols", [(600000, 1024), (130, 1 << 20), (1 << 20, 130), (4096, 4096), (3000, 8200)])
def test_long_matrices(gpu_device, rows, cols):
    u = torch.randn(rows, cols, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda")
    want = _newton_schulz(u) if rows <= cols else _newton_schulz(u.t().contiguous()).t()
    assert _off(training.orthogonalise(u), want) <= PRODUCTS + BF16
    main, momentum = torch.zeros_like(u), torch.zeros_like(u)
    training.muon_step(main, momentum, u, lr=1.0, rms_scale=0.5, nesterov=False)
    assert torch.equal(momentum, u)
    want *= -0.5 * max(rows, cols) ** 0.5
    assert _off(main, want) <= PRODUCTS
