"""What the updates write counts as changed in place: a graph that saved it refuses to go on."""

import pytest
import torch

from elasticmegatron_amd import training

pytestmark = pytest.mark.gpu


def _inputs():
    gen = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    hidden, weight = r(6, 64).to(torch.bfloat16), (r(100, 64) / 8).to(torch.bfloat16)
    return hidden.requires_grad_(), weight, torch.randint(0, 100, (6,), generator=gen, device="cuda"), r(100, 64)


def _adamw(main, grad, model=None):
    training.adamw_step(main, torch.zeros_like(main), torch.zeros_like(main), grad, model=model, lr=0.1, step=1)


def _muon(main, grad, model=None):
    training.muon_step(main, torch.zeros_like(main), grad, model=model, lr=0.1)


@pytest.mark.parametrize("update", [_adamw, _muon])
def test_a_graph_refuses_a_changed_image(gpu_device, update):
    hidden, weight, target, main = _inputs()
    loss = training.linear_cross_entropy(hidden, weight, target)
    update(main, torch.ones_like(main), weight)
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
    loss = training.linear_cross_entropy(hidden, weight, target)  # the new weights' graph runs
    update(main, torch.ones_like(main))                           # which this does not change
    loss.backward()


@pytest.mark.parametrize("update", [_adamw, _muon])
def test_a_graph_of_torch_operators_refuses_changed_weights(gpu_device, update):
    _, _, _, main = _inputs()
    x = torch.ones(6, 64, device="cuda", requires_grad=True)
    out = (x @ main.t()).sum()
    update(main, torch.ones_like(main))
    with pytest.raises(RuntimeError, match="inplace operation"):
        out.backward()


def test_every_tensor_that_is_written_counts(gpu_device):
    hidden, _, _, main = _inputs()
    m, v, image, grad = torch.zeros_like(main), torch.zeros_like(main), main.to(torch.bfloat16), torch.ones_like(main)
    tensors = (main, m, v, image, grad)
    before = [t._version for t in tensors]
    training.adamw_step(main, m, v, grad, model=image, lr=0.1, step=1)
    assert [t._version > b for t, b in zip(tensors, before)] == [True] * 4 + [False]
    before = [t._version for t in tensors]
    training.muon_step([main], [m], [grad], model=[image], lr=0.1)
    assert [t._version > b for t, b in zip(tensors, before)] == [True, True, False, True, False]


def test_views_of_an_arena_count_for_it(gpu_device):
    arena = torch.ones(1000, device="cuda")
    x = torch.ones(1000, device="cuda", requires_grad=True)
    out = (x * arena).sum()
    _adamw(arena[100:200], torch.ones(100, device="cuda"))
    with pytest.raises(RuntimeError, match="inplace operation"):
        out.backward()


def test_tensors_of_inference_mode(gpu_device):
    with torch.inference_mode():
        main = torch.ones(8, 8, device="cuda")
        _adamw(main, torch.ones(8, 8, device="cuda"))
        _muon(main, torch.ones(8, 8, device="cuda"))
    assert (main != 1).all()
