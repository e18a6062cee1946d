"""A training step on resident state: operators of the layers, the loss, the Muon update and the AdamW update.

The state that :class:`~elasticmegatron_amd.megatron_manager.training_state.TrainingState` holds is what
these read and write: the bf16 images of the layers and of the output layer's vocabulary shards, and
main / exp_avg / exp_avg_sq.

  rms_norm                  the norm before a block
  residual_norm             a block's output into the residual stream, and the norm behind it
  attention                 attention within packed documents
  expert_linear             products of tokens with their experts' matrices
  linear_cross_entropy      loss of every token from hidden states and vocabulary shards, with its gradient
  vocab_statistics          one process's part of that loss, where its shards are on several
  merge_vocab_statistics    the whole loss's statistics from every process's part
  vocab_gradients           one process's part of its gradient
  orthogonalise             Newton-Schulz products on matrices
  muon_step                 momentum, Newton-Schulz, decayed weights and their bf16 image
  adamw_step                the same for what is no matrix, with Adam's two moments

Kernels run on the current stream of the tensors' device, as torch's own operators do; outputs and
workspaces come from torch's caching allocator.  There is no fallback: without a GPU and the built
library every call raises.  The loss and the layers' operators have reverse-mode derivatives, once; nothing
has forward-mode ones, and tensors that carry a tangent are refused.  What an update writes counts as changed
in place.
"""

from .adamw import adamw_step
from .experts import expert_linear
from .loss import linear_cross_entropy, merge_vocab_statistics, vocab_gradients, vocab_statistics
from .muon import MUON_COEFFICIENTS, muon_step, orthogonalise
from .norm import residual_norm, rms_norm
from .packed_attention import attention

__all__ = ["rms_norm", "residual_norm", "attention", "expert_linear", "linear_cross_entropy", "vocab_statistics",
           "merge_vocab_statistics", "vocab_gradients", "orthogonalise", "muon_step", "adamw_step", "MUON_COEFFICIENTS"]
