"""A training step on resident state: the loss, the Muon update and the AdamW update.

The state that :class:`~elasticmegatron_amd.megatron_manager.training_state.TrainingState` holds is what
these read and write: the output layer's bf16 vocabulary shards, and main / exp_avg / exp_avg_sq.

  linear_cross_entropy      loss of every token from hidden states and vocabulary shards, with its gradient
  vocab_statistics          one process's part of that loss, where its shards are on several
  merge_vocab_statistics    the whole loss's statistics from every process's part
  vocab_gradients           one process's part of its gradient
  orthogonalise             Newton-Schulz products on matrices
  muon_step                 momentum, Newton-Schulz, decayed weights and their bf16 image
  adamw_step                the same for what is no matrix, with Adam's two moments

Kernels run on the current stream of the tensors' device, as torch's own operators do; outputs and
workspaces come from torch's caching allocator.  There is no fallback: without a GPU and the built
library every call raises.  The loss has reverse-mode derivatives, once; nothing has forward-mode ones, and tensors
that carry a tangent are refused.  What an update writes counts as changed in place.
"""

from .adamw import adamw_step
from .loss import linear_cross_entropy, merge_vocab_statistics, vocab_gradients, vocab_statistics
from .muon import MUON_COEFFICIENTS, muon_step, orthogonalise

__all__ = ["linear_cross_entropy", "vocab_statistics", "merge_vocab_statistics", "vocab_gradients", "orthogonalise",
           "muon_step", "adamw_step", "MUON_COEFFICIENTS"]
