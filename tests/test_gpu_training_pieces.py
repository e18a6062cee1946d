"""Vocabularies whose copies of weights, transposed or padded, are made a piece at a time."""

import pytest
import torch

from elasticmegatron_amd import training
from tests.test_gpu_training_loss import _check_gradients, _formula, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,hidden,rows,vocab,dtype", [
    (300, 2048, [70000], 69990, torch.bfloat16),
    (770, 4096, [20000, 20000], 39000, torch.float16),
    (260, 4096, [9000, 30000, 500], None, torch.bfloat16),  # shards of several sizes, one of several pieces
    (1, 4097, [40000], None, torch.bfloat16),               # rows off 16 bytes
    (3, 4097, [40000], 39999, torch.float16),
    (300, 2500, [60000], None, torch.bfloat16),
])
def test_several_pieces(gpu_device, tokens, hidden, rows, vocab, dtype):
    vocab = sum(rows) if vocab is None else vocab
    h, w, target, g = _inputs(tokens, hidden, rows, dtype, vocab=vocab, ignored=0.0 if tokens < 4 else 0.2)
    lse, logit = training.vocab_statistics(h, w, target, vocab_size=vocab)
    gh, gw = training.vocab_gradients(h, w, target, lse, g, vocab_size=vocab)
    _check_gradients(h, w, target, g, vocab, torch.where(target >= 0, lse - logit, 0.0), gh, gw)
    want, *_, off = _formula(h, w, target, g, vocab)
    loss = training.linear_cross_entropy(h, w, target, vocab_size=vocab, reduction="none")
    assert (loss.double() - want).abs().le(off).all()
