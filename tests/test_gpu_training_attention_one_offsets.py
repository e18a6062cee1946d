"""One tensor of offsets for queries and for keys, of which there are more rows: documents' keys are the rows at the offsets,
and the rows behind them are no document's."""

import math

import pytest
import torch

from tests.test_gpu_training_attention import BF16, FP16, _close, _formula, _inputs, _offsets, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths,heads,kv_heads,dim,dtype,causal,index,spare", [
    ([3, 5], 8, 2, 64, BF16, True, torch.int64, 0),
    ([3, 5], 8, 2, 64, BF16, False, torch.int32, 0),
    ([1] * 8, 32, 8, 128, BF16, True, torch.int32, 0),        # single tokens
    ([1] * 8, 12, 6, 100, FP16, True, torch.int64, 4),
    ([2, 0, 31, 7], 6, 2, 128, FP16, False, torch.int32, 5),
    ([64], 4, 1, 128, BF16, True, torch.int32, 0),            # the longest whose heads are rows of one tile
    ([40, 1, 0, 20], 15, 3, 32, BF16, True, torch.int64, 3),
    ([1, 2, 0, 1] * 15 + [3, 1], 4, 2, 64, BF16, True, torch.int32, 0),            # 62 documents: the most that are walked
    ([1, 2, 0, 1] * 15 + [3, 1], 4, 2, 64, FP16, False, torch.int64, 6),
    ([1, 2, 0, 1] * 15 + [3, 1, 2], 4, 2, 64, BF16, True, torch.int64, 0),         # 63: listed
    ([1, 2, 0, 1] * 15 + [3, 1, 2], 8, 2, 64, BF16, False, torch.int32, 2),
    ([300], 4, 2, 64, BF16, True, torch.int32, 0),            # too long for that
    ([130, 20], 4, 1, 128, FP16, True, torch.int64, 11),
])
def test_more_rows_of_keys(gpu_device, lengths, heads, kv_heads, dim, dtype, causal, index, spare):
    rows, group = sum(lengths) + spare, heads // kv_heads
    for times in {group, 1, group + 1}:  # so many rows of keys for each of queries
        q, k, v, g, at, _ = _inputs(lengths, heads, kv_heads, dim, dtype, [*lengths, (times - 1) * rows], spare)
        offsets = _offsets(at, index)
        got = _run(q, k, v, g, offsets=offsets, key_offsets=offsets, causal=causal)
        apart = _run(q, k, v, g, offsets=offsets, key_offsets=offsets.clone(), causal=causal)
        assert k.shape[0] == times * rows and all(torch.equal(a, b) for a, b in zip(got, apart))
        want, err = _formula(q, k, v, g, at, at, causal, 1 / math.sqrt(dim))
        for t, w, e, what in zip(got, want, err, ("out", "grad_q", "grad_k", "grad_v")):
            _close(t, w, e, (what, times))
        assert not got[2][at[-1]:].any() and not got[3][at[-1]:].any()
