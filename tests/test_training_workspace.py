"""The loss's workspace is bounded whatever the vocabulary and the tokens are (no GPU needed)."""

import ctypes

import pytest

from elasticmegatron_amd import _native


def _bytes(tokens, rows, hidden, dtype, shards=1, backward=True):
    table = lambda x: (ctypes.c_uint64 * shards)(*[x] * shards)  # noqa: E731
    tables = table(0x10000), table(hidden), table(rows // shards)
    a = _native.Loss(dtype, shards, tokens, hidden, 0x30000, hidden, *map(ctypes.addressof, tables), 0, rows, 0x40000, -100)
    grads = table(0x50000)
    a.grad_hidden, a.grad_weights = 0x90000, ctypes.addressof(grads)
    return _native.loss_workspace(a, backward)


@pytest.mark.parametrize("dtype", [_native.EMRS_BF16, _native.EMRS_FP16])
@pytest.mark.parametrize("tokens", [1, 8, 64, 256, 257, 300, 512, 769, 1024, 2048, 4096])
@pytest.mark.parametrize("rows,hidden,shards", [(32000, 4096, 1), (128256, 4096, 1), (128512, 4096, 4), (128256, 8192, 1), (1 << 20, 4096, 8)])
def test_gradients(tokens, rows, hidden, shards, dtype):
    """128 MB of d in either orientation and 256 of transposed weights, beside what goes with tokens x hidden:
    transposed hidden states, and the partial sums of their gradient, of which large products have few."""
    assert _bytes(tokens, rows, hidden, dtype, shards) <= (512 << 20) + 8 * max(tokens, 256) * hidden * 2


@pytest.mark.parametrize("tokens", [1, 2, 64, 300, 4096])
@pytest.mark.parametrize("rows,hidden", [(128256, 4097), (128256, 8190), (32000, 1001)])
def test_rows_off_16_bytes(tokens, rows, hidden):
    """A padded copy of as much of the weight as the bound allows, and the padded hidden states."""
    padded = -(-hidden // 64) * 64
    states = max(tokens, 256) * padded * 2
    pairs = rows // 16 * tokens * 8 // 2 if tokens > 1 else rows
    assert _bytes(tokens, rows, hidden, _native.EMRS_BF16, backward=False) <= (256 << 20) + 2 * states + pairs
    assert _bytes(tokens, rows, hidden, _native.EMRS_BF16) <= (768 << 20) + 9 * states
