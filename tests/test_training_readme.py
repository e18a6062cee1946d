"""The README's training step is a call that the package takes, and does what its names say."""

import ast
import inspect
import os
import re

import pytest
import torch

from elasticmegatron_amd import training

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _snippet():
    with open(os.path.join(ROOT, "README.md")) as f:
        section = f.read().split("### A training step", 1)[1]
    return re.search(r"```python\n(.*?)```", section, re.S).group(1)


def test_every_call_fits_its_function():
    calls = [n for n in ast.walk(ast.parse(_snippet()))
             if isinstance(n, ast.Call) and isinstance(n.func, ast.Attribute) and getattr(n.func.value, "id", None) == "training"]
    assert {c.func.attr for c in calls} == {"linear_cross_entropy", "muon_step", "adamw_step"}
    for c in calls:
        inspect.signature(getattr(training, c.func.attr)).bind(*c.args, **{k.arg: k.value for k in c.keywords})


@pytest.mark.gpu
def test_the_snippet_trains(gpu_device):
    r = lambda *shape: torch.randn(*shape, device="cuda")  # noqa: E731
    hidden = r(6, 64).to(torch.bfloat16).requires_grad_()
    shards = [(r(16000, 64) / 8).to(torch.bfloat16).requires_grad_() for _ in range(2)]
    names = dict(hidden=hidden, shards=shards, target=torch.randint(0, 32000, (6,), device="cuda"),
                 mains=[r(64, 96), r(64, 96)], momenta=[r(64, 96), r(64, 96)], grads=[r(64, 96), r(64, 96)],
                 images=[torch.zeros(64, 96, dtype=torch.bfloat16, device="cuda") for _ in range(2)],
                 main=r(50), exp_avg=r(50), exp_avg_sq=r(50).square(), grad=r(50), image=torch.zeros(50, dtype=torch.bfloat16, device="cuda"))
    before = {k: [t.clone() for t in v] if isinstance(v, list) else v.clone() for k, v in names.items()}
    exec(_snippet(), names)  # noqa: S102: the package's own document
    assert hidden.grad.any() and all(w.grad.any() for w in shards)
    for i in range(2):
        assert torch.equal(names["grads"][i], before["grads"][i])
        want = 0.95 * before["momenta"][i] + before["grads"][i]
        assert (names["momenta"][i] - want).abs().max() < 1e-5
        assert not torch.equal(names["mains"][i], before["mains"][i])
        assert torch.equal(names["images"][i], names["mains"][i].to(torch.bfloat16))
    assert torch.equal(names["grad"], before["grad"])
    assert not torch.equal(names["main"], before["main"]) and torch.equal(names["image"], names["main"].to(torch.bfloat16))
