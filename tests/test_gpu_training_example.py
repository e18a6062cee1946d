"""The example that trains through a switch runs, learns, and does not notice the switch."""

import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_training_goes_on_through_a_switch(gpu_device):
    spec = importlib.util.spec_from_file_location("train_through_switch", os.path.join(ROOT, "examples", "train_through_switch.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    switched, plain = example.run(8, 4), example.run(8, None)
    assert switched[:5] == pytest.approx(plain[:5], rel=1e-5)  # the switch moves bits, and shards only join in another order
    # A last bit of the loss's sums moves an update by a rounding of its bf16 image at most: 2^-8 of a weight.
    assert switched[5:] == pytest.approx(plain[5:], rel=2 ** -7)
    assert plain[0] == pytest.approx(6.908, abs=0.1)  # log 1000: an untrained model
    assert plain[-1] < plain[0] - 0.5 and switched[-1] < switched[0] - 0.5
