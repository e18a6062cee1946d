"""Forward-mode derivatives: no operator of a training step has one, and none drops a tangent (no GPU needed)."""

import pytest
import torch
from torch.autograd import forward_ad

from elasticmegatron_amd import training

H, W = torch.ones(4, 8, dtype=torch.bfloat16), torch.ones(10, 8, dtype=torch.bfloat16)
T, F, M = torch.zeros(4, dtype=torch.int64), torch.ones(4), torch.ones(6, 8)


def _dual(t):
    return forward_ad.make_dual(t.clone(), torch.ones_like(t))


CALLS = {
    "hidden": lambda d: training.linear_cross_entropy(d(H), W, T),
    "shard": lambda d: training.linear_cross_entropy(H, [W, d(W)], T, reduction="none"),
    "statistics": lambda d: training.vocab_statistics(H, d(W), T),
    "gradients": lambda d: training.vocab_gradients(d(H), W, T, F, F),
    "gradients, lse": lambda d: training.vocab_gradients(H, W, T, d(F), F),
    "gradients, grad_loss": lambda d: training.vocab_gradients(H, W, T, F, d(F)),
    "orthogonalise": lambda d: training.orthogonalise(d(M)),
    "orthogonalise, several": lambda d: training.orthogonalise([M, d(M)]),
    "muon, grad": lambda d: training.muon_step(M, M.clone(), d(M), lr=0.1),
    "muon, main": lambda d: training.muon_step([d(M)], [M], [M], lr=0.1),
    "adamw, grad": lambda d: training.adamw_step(M, M.clone(), M.clone(), d(M), lr=0.1, step=1),
    "adamw, main": lambda d: training.adamw_step(d(M), M, M.clone(), M.clone(), lr=0.1, step=1),
}


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("with_grad", [True, False])
def test_tangents_are_refused(call, with_grad):
    with torch.set_grad_enabled(with_grad), forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            CALLS[call](_dual)
        with pytest.raises(ValueError, match="a GPU is wanted"):  # a level alone is no tangent
            CALLS[call](lambda t: t)


@pytest.mark.gpu
def test_no_tangent_is_dropped_on_the_gpu(gpu_device):
    h, w, t = H.cuda(), W.cuda(), T.cuda()
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            training.linear_cross_entropy(_dual(h), w, t)
        assert training.linear_cross_entropy(h, w, t).isfinite()
    with pytest.raises(Exception):
        torch.func.jvp(lambda x: training.linear_cross_entropy(x, w, t), (h,), (torch.ones_like(h),))
