"""The README's calls of the layers' operators are calls that the package takes, and give what they say."""

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
    return re.findall(r"```python\n(.*?)```", section, re.S)[1]


def test_every_call_fits_its_function():
    calls = [n for n in ast.walk(ast.parse(_snippet()))
             if isinstance(n, ast.Call) and isinstance(n.func, ast.Attribute) and getattr(n.func.value, "id", None) == "training"]
    assert {c.func.attr for c in calls} == {"rms_norm", "residual_norm", "attention", "expert_linear"}
    for c in calls:
        inspect.signature(getattr(training, c.func.attr)).bind(*c.args, **{k.arg: k.value for k in c.keywords})


@pytest.mark.gpu
def test_the_snippet_runs(gpu_device):
    b = lambda *shape: torch.randn(*shape, device="cuda").to(torch.bfloat16)  # noqa: E731
    names = dict(training=training, stream=b(6, 64), norm_weight=b(64), q=b(6, 4, 16), k=b(6, 2, 16), v=b(6, 2, 16), block_out=b(6, 64),
                 offsets=torch.tensor([0, 2, 6], device="cuda"), x_by_expert=b(6, 64), expert_weights=[b(32, 64) for _ in range(3)],
                 counts=torch.tensor([4, 0, 2], device="cuda"))
    before = names["stream"].double()
    exec(_snippet(), names)  # noqa: S102: the package's own document
    assert names["out"].shape == (6, 4, 16) and names["y"].shape == (6, 32)
    want = before + names["block_out"].double()
    assert (names["stream"].double() - want).abs().le(2.0 ** -8 * want.abs() + 2.0 ** -23 * before.abs().max()).all()
    assert torch.equal(names["out"][0], names["v"][0].repeat_interleave(2, 0))  # a document's first row sees itself alone
    want = names["x_by_expert"][5].double() @ names["expert_weights"][2].double().t()
    room = 2.0 ** -8 * want.abs() + 2.0 ** -17 * (names["x_by_expert"][5].double().abs() @ names["expert_weights"][2].double().abs().t())
    assert (names["y"][5].double() - want).abs().le(room).all()
