"""AdamW over more elements than one row of a launch's grid has lanes."""

import pytest
import torch

from elasticmegatron_amd import training

pytestmark = pytest.mark.gpu


def test_more_than_2_to_32_elements_off_16_bytes(gpu_device):
    n = 2 ** 32 + 515
    whole = [torch.full((n + 2,), x, device="cuda") for x in (1.0, 0.5, 0.25)]
    main, m, v = (t[1:n + 1] for t in whole)
    grad = torch.full((n,), 2.0, dtype=torch.bfloat16, device="cuda")
    places = [0, 1, 2 ** 31 - 1, 2 ** 31, 2 ** 32 - 1, 2 ** 32, n - 1]
    for i, at in enumerate(places):
        main[at] = 2.0 + i
    training.adamw_step(main, m, v, grad, lr=0.5, weight_decay=0.25, step=3)
    small = [torch.full((len(places) + 1,), x, device="cuda") for x in (1.0, 0.5, 0.25)]
    small[0][1:] = torch.arange(len(places), device="cuda") + 2.0
    training.adamw_step(*small, torch.full((len(places) + 1,), 2.0, device="cuda"), lr=0.5, weight_decay=0.25, step=3)
    for i, at in enumerate(places):
        assert main[at] == small[0][1 + i]
        main[at] = small[0][0]
    for got, want in zip((main, m, v), small):
        assert got.min() == got.max() == want[0]
    assert all(t[0] == x and t[-1] == x for t, x in zip(whole, (1.0, 0.5, 0.25)))
