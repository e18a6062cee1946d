"""The layers' backward passes run on what autograd saved: hooks see and replace it, it goes with the graph, and nothing
is read at an address that forward once saw."""

import gc
import weakref

import pytest
import torch

from elasticmegatron_amd import training

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _normal(seed, *shapes):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(*s, generator=gen, device="cuda").to(BF16) for s in shapes]


def _norm():
    x = _normal(1, (30, 136), (30, 136), (136,), (136,), (136,))
    return x, lambda r, b, w, bw, g: training.residual_norm(r, b, w, branch_weight=bw, gate=g)[1], _normal(2, (30, 136))[0]


def _norm_alone():
    return _normal(3, (30, 136), (136,)), training.rms_norm, _normal(4, (30, 136))[0]


def _experts():
    x = _normal(5, (50, 72), (40, 72), (40, 72), (40, 72))
    counts = torch.tensor([20, 0, 25], device="cuda")
    return x, lambda x, *w: training.expert_linear(x, w, counts), _normal(6, (50, 40))[0]


def _attention():
    offsets = torch.tensor([0, 33, 70], dtype=torch.int32, device="cuda")
    return _normal(7, (70, 4, 64), (70, 2, 64), (70, 2, 64)), lambda q, k, v: training.attention(q, k, v, offsets=offsets), _normal(8, (70, 4, 64))[0]


def _batches():
    return _normal(9, (2, 35, 4, 64), (2, 35, 2, 64), (2, 35, 2, 64)), training.attention, _normal(10, (2, 35, 4, 64))[0]


CASES = {"norm": _norm, "norm alone": _norm_alone, "experts": _experts, "attention": _attention, "attention, batches": _batches}


def _leaves(x, turned):
    """The same values as they lie, or as they have to be copied first."""
    return [(t.transpose(-1, -2).contiguous().transpose(-1, -2) if turned and t.dim() > 1 else t).detach().requires_grad_() for t in x]


@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_hooks_see_what_backward_reads(gpu_device, case, turned):
    x, call, g = CASES[case]()
    leaves = _leaves(x, False)
    want = torch.autograd.grad(call(*leaves), leaves, g)
    leaves, places = _leaves(x, turned), []

    def pack(t):
        places.append(t.data_ptr())
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.cuda()):
        out = call(*leaves)
    taken = [torch.full((4096,), 7.0, device="cuda") for _ in range(64)]  # other addresses for what comes back
    got = torch.autograd.grad(out, leaves, g)
    assert len(places) >= len(x) and len(taken) == 64
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("case", CASES)
def test_hooks_may_replace_values(gpu_device, case):
    """What comes back from the hooks counts: zeros for everything give zeros, or what zeros give."""
    x, call, g = CASES[case]()
    leaves = _leaves(x, False)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t * 0 if t.is_floating_point() else t):
        out = call(*leaves)
    for a, t in zip(torch.autograd.grad(out, leaves, g), x):
        assert a.shape == t.shape and a.isfinite().all()
        if case == "experts" or "norm" in case:
            assert not a.any()


@pytest.mark.parametrize("case", CASES)
def test_hooks_that_return_something_else_are_refused(gpu_device, case):
    x, call, g = CASES[case]()
    for change in (lambda t: t[:1], lambda t: t.float() if t.dtype == BF16 else t.double(), lambda t: t.cpu()):
        leaves = _leaves(x, False)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            out = call(*leaves)
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            torch.autograd.grad(out, leaves, g)


@pytest.mark.parametrize("case", CASES)
def test_checkpointing_and_two_backwards(gpu_device, case):
    from torch.utils.checkpoint import checkpoint

    x, call, g = CASES[case]()
    leaves = _leaves(x, False)
    out = call(*leaves)
    want = torch.autograd.grad(out, leaves, g, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, g), want))
    got = torch.autograd.grad(checkpoint(call, *leaves, use_reentrant=False), leaves, g)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("case", CASES)
def test_what_is_saved_goes_with_the_graph(gpu_device, case):
    x, call, g = CASES[case]()
    leaf, *rest = _leaves(x, False)
    first = leaf * 1.0
    gone = weakref.ref(first)
    out = call(first, *rest)
    out.backward(g)
    del first
    gc.collect()
    assert gone() is None
    with pytest.raises(RuntimeError):
        out.backward(g)


@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_changes_in_place(gpu_device, case, turned):
    """Inputs that are read as they lie are refused once changed, through views too; of those that had to be copied, the copy counts.
    (The stream that a norm's gradient reads is its output, and of its inputs the residual is not read again.)"""
    x, call, g = CASES[case]()
    for i in range(len(x)):
        leaves = _leaves(x, turned)
        want = torch.autograd.grad(call(*leaves), leaves, g)
        out = call(*leaves)
        with torch.no_grad():
            leaves[i].add_(1)
        may = case == "norm" and i == 0 or turned and leaves[i].dim() > 1 and not leaves[i].is_contiguous()
        if may and not (case == "norm alone"):
            assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, g), want))
        else:
            with pytest.raises(RuntimeError, match="inplace operation"):
                torch.autograd.grad(out, leaves, g)


def test_a_stream_that_is_changed_in_place(gpu_device):
    x, _, g = _norm()
    leaves = _leaves(x, False)
    stream, normed = training.residual_norm(*leaves[:3], branch_weight=leaves[3], gate=leaves[4])
    stream.mul_(2)
    with pytest.raises(RuntimeError, match="inplace operation"):
        torch.autograd.grad(normed, leaves, g)


def test_weights_whose_storage_moves(gpu_device):
    """Sharded parameters free their storage after forward and gather it again for backward, elsewhere."""
    for case in ("experts", "norm alone"):
        x, call, g = CASES[case]()
        leaves = _leaves([x[0], *(t.repeat(1, 1).clone() for t in x[1:])] if case == "experts" else [x[0], x[1].clone()], False)
        want = torch.autograd.grad(call(*leaves), leaves, g)
        out = call(*leaves)
        weight = leaves[1]
        storage, size, place, values = weight.untyped_storage(), weight.untyped_storage().size(), weight.data_ptr(), weight.detach().cpu()
        storage.resize_(0)
        taken = [torch.full((size // 2,), float("nan"), dtype=BF16, device="cuda") for _ in range(64)]  # the old place among them
        storage.resize_(size)
        with torch.autograd._unsafe_preserve_version_counter(weight), torch.no_grad():
            weight.copy_(values)
        assert weight.data_ptr() != place and len(taken) == 64
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, g), want))


@pytest.mark.parametrize("case", CASES)
def test_two_captured_graphs(gpu_device, case):
    """Two graphs of one operator, replayed in turn with eager work between: their scratch does not meet."""
    x, call, g = CASES[case]()
    others = [t * 0.5 for t in x]

    def step(values):
        leaves = _leaves(values, False)
        out = call(*leaves)
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]

    want = [step(x), step(others)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x), step(others)
    torch.cuda.current_stream().wait_stream(side)
    graphs, got = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph, values in zip(graphs, (x, others)):
        with torch.cuda.graph(graph):
            got.append(step(values))
    for _ in range(3):
        for graph in graphs:
            graph.replay()
            step(x)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
            for t in a:
                t.fill_(3)
