"""residual_norm without the next block's norm: what backward does not read is not kept, and may change."""

import pytest
import torch

from elasticmegatron_amd import training

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
N, H = 37, 136


def _inputs(parts, residual=BF16):
    gen = torch.Generator(device="cuda").manual_seed(1)
    make = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    kw = {"branch_weight": make(H).to(BF16)} if "norm" in parts else {}
    if "gate" in parts:
        kw["gate"] = make(H).to(BF16)
    if "token" in parts:
        kw["gate"] = make(N, H).to(BF16)
    return make(N, H).to(residual), make(N, H).to(BF16), kw, make(N, H).to(residual)


def _leaves(r, b, kw):
    r, b = r.detach().clone().requires_grad_(), b.detach().clone().requires_grad_()
    kw = {k: t.detach().clone().requires_grad_() for k, t in kw.items()}
    return r, b, kw, [r, b, *kw.values()]


CASES = [((), BF16, 1.0), ((), BF16, 0.5), ((), torch.float32, 1.0), (("gate",), BF16, 1.0), (("token",), torch.float32, 0.75), (("norm",), BF16, 1.0),
         (("norm", "gate"), torch.float32, 0.5), (("norm", "token"), BF16, 1.0)]


@pytest.mark.parametrize("parts,residual,scale", CASES)
def test_what_is_kept(gpu_device, parts, residual, scale):
    """The branch and what it is multiplied by, where there is such a thing, and 1 / rms where the branch has a norm."""
    r, b, kw, g = _inputs(parts, residual)
    r, b, kw, leaves = _leaves(r, b, kw)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        stream = training.residual_norm(r, b, residual_scale=scale, **kw)
    read = [b.data_ptr(), *(t.data_ptr() for t in kw.values())] if parts else []
    assert {t.data_ptr() for t in kept if t.dtype == BF16} == set(read)
    others = [t for t in kept if t.data_ptr() not in read]
    assert all(t.dtype == torch.float32 and t.numel() <= 2 * N for t in others) and len(others) == ("norm" in parts)
    assert stream.data_ptr() not in {t.data_ptr() for t in kept}


@pytest.mark.parametrize("parts,residual,scale", CASES)
def test_the_output_may_change_in_place(gpu_device, parts, residual, scale):
    """As that of a sum may, and the residual, which backward does not read either."""
    r, b, kw, g = _inputs(parts, residual)
    r, b, kw, leaves = _leaves(r, b, kw)
    want = torch.autograd.grad(training.residual_norm(r, b, residual_scale=scale, **kw), leaves, g)
    stream = training.residual_norm(r, b, residual_scale=scale, **kw)
    stream.mul_(2)
    with torch.no_grad():
        r.add_(1)
    got = torch.autograd.grad(stream, leaves, g / 2)  # exact, in powers of two
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    if not parts:
        assert torch.equal(want[0], (g * scale).to(residual)) and torch.equal(want[1], g.to(BF16))


@pytest.mark.parametrize("parts,residual,scale", CASES)
def test_hooks_and_several_backwards(gpu_device, parts, residual, scale):
    r, b, kw, g = _inputs(parts, residual)
    r, b, kw, leaves = _leaves(r, b, kw)
    stream = training.residual_norm(r, b, residual_scale=scale, **kw)
    want = torch.autograd.grad(stream, leaves, g, retain_graph=True)
    assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(stream, leaves, g), want))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        stream = training.residual_norm(r, b, residual_scale=scale, **kw)
    taken = [torch.full((4096,), 7.0, device="cuda") for _ in range(64)]  # other addresses for what comes back
    assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(stream, leaves, g), want)) and len(taken) == 64
    if parts:
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:1]):
            stream = training.residual_norm(r, b, residual_scale=scale, **kw)
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            torch.autograd.grad(stream, leaves, g)


def test_no_tokens(gpu_device):
    for kw in ({}, dict(branch_weight=torch.ones(H, dtype=BF16, device="cuda", requires_grad=True))):
        r, b = (torch.ones(0, H, dtype=BF16, device="cuda", requires_grad=True) for _ in range(2))
        stream = training.residual_norm(r, b, **kw)
        got = torch.autograd.grad(stream, [r, b, *kw.values()], torch.ones_like(stream))
        assert [t.shape for t in got] == [t.shape for t in (r, b, *kw.values())] and not any(t.any() for t in got)
