"""Matrices of one update that share memory are refused before any of them is written."""

import pytest
import torch

from elasticmegatron_amd import training

pytestmark = pytest.mark.gpu


def _r(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def test_refusals(gpu_device):
    main, buf, grad = _r(2, 6, 8), _r(2, 6, 8), _r(2, 6, 8)
    arena = _r(200)
    near = [arena[:48].view(6, 8), arena[40:88].view(6, 8)]  # a row in common
    image = torch.zeros(2, 6, 8, dtype=torch.bfloat16, device="cuda")
    kept = [t.clone() for t in (main, buf, grad, arena, image)]
    step = lambda *a, **k: training.muon_step(*a, lr=0.1, **k)  # noqa: E731
    for call in (
        lambda: step([main[0], main[0]], list(buf), list(grad)),     # tied weights listed twice
        lambda: step(list(main), [buf[0], buf[0]], list(grad)),
        lambda: step(near, list(buf), list(grad)),
        lambda: step(list(main), near, list(grad)),
        lambda: step(main, buf, grad, model=image[:1].expand(2, 6, 8)),
        lambda: step(main[:1].expand(2, 6, 8), buf, grad),
        lambda: step(main, main, grad),
        lambda: step(main, buf, buf),
        lambda: step(main, buf, grad, model=main.view(torch.bfloat16)[:, :, :8]),
        lambda: step([*main] * 20, [*buf] * 20, [*grad] * 20),        # more than one native call
    ):
        with pytest.raises(ValueError, match="share memory"):
            call()
    assert all(torch.equal(a, b) for a, b in zip(kept, (main, buf, grad, arena, image)))


@pytest.mark.parametrize("rows,cols", [(24, 40), (130, 260)])
def test_what_is_taken(gpu_device, rows, cols):
    """Matrices between each other's rows, one gradient for all, and a gradient in its own image's place."""
    main, buf, grad = _r(3, rows, cols), _r(3, rows, cols, seed=1), _r(3, rows, cols, seed=2)
    between = [torch.zeros(rows, 3, cols, device="cuda").transpose(0, 1).copy_(t) for t in (main, buf)]
    columns = torch.zeros(rows, 2 * cols, device="cuda")
    same = grad[:1].expand(3, rows, cols)
    want_main, want_buf = main.clone(), buf.clone()
    for _ in range(2):
        training.muon_step(want_main, want_buf, same.contiguous(), lr=0.1)
        training.muon_step(*between, same, lr=0.1)
    assert torch.equal(between[0], want_main) and torch.equal(between[1], want_buf)
    # a matrix and its momentum side by side in one arena
    w, b = columns[:, :cols].copy_(main[0]), columns[:, cols:].copy_(buf[0])
    want_main, want_buf = main[0].clone(), buf[0].clone()
    training.muon_step(want_main, want_buf, grad[0], lr=0.1)
    training.muon_step(w, b, grad[0], lr=0.1)
    assert torch.equal(w, want_main) and torch.equal(b, want_buf)
    # its gradient where its image goes
    image = grad[0].to(torch.bfloat16)
    want_main, want_buf, want_image = main[0].clone(), buf[0].clone(), torch.zeros_like(image)
    training.muon_step(want_main, want_buf, image.clone(), model=want_image, lr=0.1)
    training.muon_step(main[0], buf[0], image, model=image, lr=0.1)
    assert torch.equal(main[0], want_main) and torch.equal(image, want_image)
