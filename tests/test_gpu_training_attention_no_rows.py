"""Attention of no queries or no keys, in either type."""

import pytest
import torch

from elasticmegatron_amd import training

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 20])
@pytest.mark.parametrize("wanted", ["qkv", "q"])
@pytest.mark.parametrize("rows,key_rows", [(0, 0), (0, 5), (5, 0), (0, 300), (300, 0)])
def test_a_side_without_rows(gpu_device, rows, key_rows, wanted, dim, dtype):
    """Zeros of every gradient's shape: one document, several of which none has any, and a batch."""
    make = lambda n, heads: torch.ones(n, heads, dim, dtype=dtype, device="cuda")  # noqa: E731
    q, k, v = make(rows, 4), make(key_rows, 2), make(key_rows, 2)
    at, key_at = (torch.tensor([0, n // 2, n], device="cuda") for n in (rows, key_rows))
    calls = [((q, k, v), dict(offsets=at, key_offsets=key_at))]
    if rows or key_rows:  # rows that are no document's
        calls.append(((q, k, v), dict(offsets=at * 0, key_offsets=key_at * 0)))
    calls.append(((q[None], k[None], v[None]), {}))
    for operands, kw in calls:
        leaves = [t.clone().requires_grad_(name in wanted) for t, name in zip(operands, "qkv")]
        out = training.attention(*leaves, **kw)
        assert out.shape == operands[0].shape and not out.any()
        leaves = [t for t in leaves if t.requires_grad]
        for t, grad in zip(leaves, torch.autograd.grad(out, leaves, torch.ones_like(out))):
            assert grad.shape == t.shape and grad.dtype == dtype and not grad.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,key_rows", [(0, 0), (0, 5), (5, 0), (300, 0)])
@pytest.mark.parametrize("wanted", ["k", "v", "kv"])
def test_keys_and_values_alone(gpu_device, wanted, rows, key_rows, dtype):
    """Gradients of no rows are wanted, and none of the queries' rows."""
    make = lambda n, heads: torch.ones(1, n, heads, 64, dtype=dtype, device="cuda")  # noqa: E731
    leaves = [t.requires_grad_(name in wanted) for t, name in zip((make(rows, 4), make(key_rows, 2), make(key_rows, 2)), "qkv")]
    out = training.attention(*leaves)
    leaves = [t for t in leaves if t.requires_grad]
    for t, grad in zip(leaves, torch.autograd.grad(out, leaves, torch.ones_like(out))):
        assert grad.shape == t.shape and grad.dtype == dtype and not grad.any()
