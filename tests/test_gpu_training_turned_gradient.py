"""AdamW takes a gradient as a flat run of its weights' elements, and refuses one whose sides are turned."""

import pytest
import torch

from elasticmegatron_amd import training

pytestmark = pytest.mark.gpu


def _state(*shape):
    return [torch.ones(*shape, device="cuda") for _ in range(3)]


@pytest.mark.parametrize("main,grad", [((4, 6), (6, 4)), ((2, 3, 4), (2, 4, 3)), ((4, 1, 6), (6, 4))])
def test_refused(gpu_device, main, grad):
    state = _state(*main)
    with pytest.raises(ValueError, match="another order"):
        training.adamw_step(*state, torch.ones(*grad, device="cuda"), lr=0.1, step=1)
    assert all((t == 1).all() for t in state)


@pytest.mark.parametrize("main,grad", [((4, 6), (24,)), ((24,), (4, 6)), ((4, 6), (2, 2, 6)), ((1, 24), (24, 1)), ((4, 6), (4, 1, 6))])
def test_taken(gpu_device, main, grad):
    g = torch.arange(24.0, device="cuda")
    state, want = _state(*main), _state(24)
    training.adamw_step(*state, g.view(grad), lr=0.1, step=1)
    training.adamw_step(*want, g, lr=0.1, step=1)
    assert all(torch.equal(a.view(-1), b) for a, b in zip(state, want))


def test_a_transposed_view_of_the_right_shape(gpu_device):
    g = torch.arange(24.0, device="cuda").view(6, 4).t()
    state, want = _state(4, 6), _state(4, 6)
    training.adamw_step(*state, g, lr=0.1, step=1)
    training.adamw_step(*want, g.contiguous(), lr=0.1, step=1)
    assert all(torch.equal(a, b) for a, b in zip(state, want))
