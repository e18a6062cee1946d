"""The loss's backward pass runs on what autograd saved: hooks see and replace it, it goes with the graph, and
nothing is read at an address that forward once saw."""

import gc
import weakref

import pytest
import torch

from elasticmegatron_amd import training

pytestmark = pytest.mark.gpu


def _inputs(tokens=40, hidden=128, rows=(200, 100), seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(tokens, hidden, generator=gen, device="cuda").to(torch.bfloat16)
    w = [(torch.randn(r, hidden, generator=gen, device="cuda") / 8).to(torch.bfloat16) for r in rows]
    target = torch.randint(0, sum(rows), (tokens,), generator=gen, device="cuda")
    target[3] = -100
    return h, w, target, torch.rand(tokens, generator=gen, device="cuda")


def _layouts(h, w, target):
    """The same values, as they lie and as they have to be copied first."""
    yield h, w, target
    yield h.t().contiguous().t(), [x.t().contiguous().t() for x in w], torch.stack([target, target], 1)[:, 0]


def test_hooks_see_what_backward_reads(gpu_device):
    """A hook that returns copies on another place, and one that returns other values (whose probabilities stay below one)."""
    h, w, target, g = _inputs()
    lse, _ = training.vocab_statistics(h, w, target)
    want_h, want_w = training.vocab_gradients(h, w, target, lse, g)
    half_h, half_w = training.vocab_gradients(h, [x * 0.5 for x in w], target, lse, g)
    for hid, shards, t in _layouts(h, w, target):
        hid, shards = hid.detach().requires_grad_(), [x.detach().requires_grad_() for x in shards]
        packed = []

        def pack(x):
            packed.append(x)
            return x.cpu()

        for unpack, expect_h, expect_w in (
                (lambda x: x.cuda(), want_h, want_w),
                (lambda x: x.cuda() * 0.5 if x.dim() == 2 and x.shape[0] in (200, 100) else x.cuda(), half_h, half_w)):
            with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
                loss = training.linear_cross_entropy(hid, shards, t, reduction="none")
            got = torch.autograd.grad(loss, [hid, *shards], g)
            assert torch.equal(got[0], expect_h) and all(torch.equal(a, b) for a, b in zip(got[1:], expect_w))
        assert {tuple(x.shape) for x in packed} >= {(40, 128), (200, 128), (100, 128)}


def test_checkpointing_runs_forward_again(gpu_device):
    from torch.utils.checkpoint import checkpoint

    h, w, target, g = _inputs()
    x = h.detach().requires_grad_()
    want, = torch.autograd.grad(training.linear_cross_entropy(x, w, target, reduction="none"), x, g)
    loss = checkpoint(lambda y: training.linear_cross_entropy(y * 1.0, w, target, reduction="none"), x, use_reentrant=False)
    got, = torch.autograd.grad(loss, x, g)
    assert torch.equal(got, want)


def test_what_is_saved_goes_with_the_graph(gpu_device):
    """A loss that is kept after backward keeps neither its hidden states nor copies of the weights."""
    for transposed in (False, True):
        h, w, target, _ = _inputs(rows=(4000,))
        leaf = h.detach().requires_grad_()
        hid = leaf * 1.0
        weight = (w[0].t().contiguous().t() if transposed else w[0]).detach().requires_grad_()
        gone = weakref.ref(hid)
        gc.collect()
        before = torch.cuda.memory_allocated()
        loss = training.linear_cross_entropy(hid, weight, target)
        loss.backward()
        weight.grad = leaf.grad = None
        del hid
        gc.collect()
        assert gone() is None
        # the loss itself stays, and less than a row of weights of anything else; the hidden states went
        assert torch.cuda.memory_allocated() - before < 4000 * 2
        with pytest.raises(RuntimeError):
            loss.backward()


def test_a_weight_whose_storage_moves(gpu_device):
    """Sharded parameters free their storage after forward and gather it again for backward, elsewhere."""
    h, w, target, g = _inputs(rows=(5000,))
    h.requires_grad_()
    weight = w[0].clone().requires_grad_()
    want = torch.autograd.grad(training.linear_cross_entropy(h, weight, target, reduction="none"), [h, weight], g)
    loss = training.linear_cross_entropy(h, weight, target, reduction="none")
    storage, size, place = weight.untyped_storage(), weight.untyped_storage().size(), weight.data_ptr()
    values = weight.detach().cpu()
    storage.resize_(0)
    taken = [torch.full((size // 2,), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(32)]  # the old place among them
    storage.resize_(size)
    with torch.autograd._unsafe_preserve_version_counter(weight), torch.no_grad():
        weight.copy_(values)
    assert weight.data_ptr() != place and len(taken) == 32
    got = torch.autograd.grad(loss, [h, weight], g)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("changed", ["hidden", "weight", "target"])
def test_changes_in_place_are_refused_or_not_seen(gpu_device, changed):
    """Inputs that are read as they lie are refused once changed; of those that had to be copied, the copy counts."""
    for copied, (hid, shards, t) in enumerate(_layouts(*_inputs()[:3])):
        g = _inputs()[3]
        leaf = hid.detach().requires_grad_()
        want, = torch.autograd.grad(training.linear_cross_entropy(leaf, shards, t, reduction="none"), leaf, g)
        loss = training.linear_cross_entropy(leaf, shards, t, reduction="none")
        with torch.no_grad():
            {"hidden": leaf, "weight": shards[1], "target": t}[changed].zero_()
        if copied:
            got, = torch.autograd.grad(loss, leaf, g)
            assert torch.equal(got, want)
        else:
            with pytest.raises(RuntimeError, match="inplace operation"):
                torch.autograd.grad(loss, leaf, g)


def test_two_backwards_of_one_graph(gpu_device):
    h, w, target, g = _inputs()
    h = h.view(2, 20, 128).requires_grad_()
    loss = training.linear_cross_entropy(h, w, target.view(2, 20), reduction="none")
    first, = torch.autograd.grad(loss, h, g.view(2, 20), retain_graph=True)
    again, = torch.autograd.grad(loss, h, g.view(2, 20))
    assert torch.equal(first, again)


@pytest.mark.parametrize("changed", ["hidden", "target"])
def test_views_of_inputs_are_refused_too(gpu_device, changed):
    """Hidden states of more dimensions are read through a view, whose base counts."""
    h, w, target, _ = _inputs()
    h, target = h.view(2, 20, 128).requires_grad_(), target.view(2, 20)
    loss = training.linear_cross_entropy(h, w, target)
    with torch.no_grad():
        {"hidden": h, "target": target}[changed].zero_()
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
