"""Products of tokens with their experts' matrices, against the formula in 64 bits and against differences."""

import math

import pytest
import torch

from elasticmegatron_amd import training

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
UNIT = {BF16: 2.0 ** -8, FP16: 2.0 ** -11}  # half a step, relative
STEP = {BF16: 2.0 ** -134, FP16: 2.0 ** -25}  # half the smallest number


def _inputs(counts, n_in, n_out, dtype, spare=0, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows = sum(max(0, c) for c in counts) + spare
    x = torch.randn(rows, n_in, generator=gen, device="cuda").to(dtype)
    w = [(torch.randn(n_out, n_in, generator=gen, device="cuda") / math.sqrt(n_in)).to(dtype) for _ in counts]
    g = torch.randn(rows, n_out, generator=gen, device="cuda").to(dtype)
    return x, w, torch.tensor(counts, dtype=torch.int32, device="cuda"), g


def _formula(x, w, counts, g):
    """(value, sum of the absolute products) of every output, in 64 bits."""
    y = [torch.zeros(len(x), w[0].shape[0], dtype=torch.double, device="cuda") for _ in range(2)]
    gx = [torch.zeros(x.shape, dtype=torch.double, device="cuda") for _ in range(2)]
    gw, lo = [], 0
    for e, c in enumerate(counts):
        hi = min(len(x), lo + max(0, c))
        parts = []
        for i, f in enumerate((lambda t: t.double(), lambda t: t.double().abs())):
            a, b, d = f(x[lo:hi]), f(w[e]), f(g[lo:hi])
            y[i][lo:hi], gx[i][lo:hi] = a @ b.t(), d @ b
            parts.append(d.t() @ a)
        gw.append(parts)
        lo = hi
    return y, gx, gw


def _close(got, want, terms, what):
    """One rounding to the type, and sums in 32 bits: at most `terms` roundings of the absolute sum."""
    value, size = want
    off = (got.double() - value).abs()
    e = terms * 2.0 ** -24 * size
    room = e + UNIT[got.dtype] * (value.abs() + e) + STEP[got.dtype]
    assert off.le(room).all(), (what, float((off - room).max()))


def _run(x, w, counts, g):
    x, w = x.detach().requires_grad_(), [t.detach().requires_grad_() for t in w]
    y = training.expert_linear(x, w, counts)
    gx, *gw = torch.autograd.grad(y, [x, *w], g)
    return y.detach(), gx, gw


def _check(x, w, counts, g, y, gx, gw):
    want_y, want_gx, want_gw = _formula(x, w, counts.tolist(), g)
    assert y.dtype == gx.dtype == x.dtype and y.shape == (len(x), w[0].shape[0])
    _close(y, want_y, x.shape[1], "y")
    _close(gx, want_gx, w[0].shape[0], "grad_x")
    for e, (a, b) in enumerate(zip(gw, want_gw)):
        assert a.shape == w[e].shape and a.dtype == w[e].dtype
        _close(a, b, max(1, len(x)), f"grad_w {e}")


CASES = [
    ([1], 8, 8, BF16, 0),
    ([1], 1, 1, FP16, 0),
    ([0, 1, 0], 64, 64, BF16, 0),
    ([0, 0], 32, 40, BF16, 5),                     # nobody got a token
    ([3, 0, 5, 1], 100, 36, FP16, 2),              # sides that are no multiples of 8
    ([7, 9], 1000, 333, BF16, 0),
    ([2, 0, 0, 2], 4096, 512, BF16, 0),
    ([31, 33, 1, 64, 63], 136, 264, FP16, 1),      # around the tiles' sizes
    ([65, 127, 128, 129, 0, 255, 257], 72, 520, BF16, 0),
    ([400, 0, 1000, 3], 512, 256, BF16, 17),
    ([1500, 600], 256, 1376, FP16, 0),
    ([1, 2, 3, 4] * 16, 64, 96, BF16, 0),          # 64 experts: two steps of the prefix sum
    ([5] * 63, 40, 48, BF16, 1),
    ([0, 3, 1] * 85, 24, 32, FP16, 3),             # 255
    ([0] * 200 + [40] + [0] * 55, 72, 64, BF16, 0),  # 256
    ([3000, 1], 520, 1000, BF16, 0),
    ([5000], 200, 264, FP16, 0),
    ([2100, 1900, 96], 2048, 768, BF16, 0),
    ([12, 20], 8200, 72, BF16, 0),
    ([0, 1, 0, 0, 0, 1], 4096, 1000, BF16, 0),     # one token's experts: weights read by rows
    ([2], 520, 37, FP16, 0),
    ([0, 1], 1001, 130, BF16, 1),                  # and a row of none
    ([0] * 70 + [1], 264, 64, BF16, 1),
]


@pytest.mark.parametrize("counts,n_in,n_out,spare", [([2100, 1999], 8200, 4360, 7), ([3000, 1, 1090], 4352, 8192, 0)])
def test_long_sums_are_cut(gpu_device, counts, n_in, n_out, spare):
    """The tiles of the last round are cut along a long k: of y where n_in is long, of grad_x where n_out is."""
    x, w, c, g = _inputs(counts, n_in, n_out, BF16, spare)
    got = _run(x, w, c, g)
    _check(x, w, c, g, *got)
    again = _run(x, w, c, g)
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


@pytest.mark.parametrize("counts,n_in,n_out,dtype,spare", CASES)
def test_outputs_and_gradients(gpu_device, counts, n_in, n_out, dtype, spare):
    x, w, c, g = _inputs(counts, n_in, n_out, dtype, spare)
    y, gx, gw = _run(x, w, c, g)
    _check(x, w, c, g, y, gx, gw)
    if spare:
        assert not y[-spare:].any() and not gx[-spare:].any()
    with torch.no_grad():
        assert torch.equal(training.expert_linear(x, w, c.long()), y)
    again = _run(x, w, c, g)
    assert torch.equal(again[1], gx) and all(torch.equal(a, b) for a, b in zip(again[2], gw))  # the same bits every time


@pytest.mark.parametrize("n_in,n_out", [(512, 264), (100, 72)])
def test_stacked_weights_and_strides(gpu_device, n_in, n_out):
    x, w, c, g = _inputs([40, 0, 99, 5], n_in, n_out, BF16, 3)
    y, gx, gw = _run(x, w, c, g)
    stack = torch.stack(w).requires_grad_()
    leaf = x.clone().requires_grad_()
    out = training.expert_linear(leaf, stack, c)
    a, b = torch.autograd.grad(out, [leaf, stack], g)
    assert torch.equal(out, y) and torch.equal(a, gx) and torch.equal(b, torch.stack(gw))
    views = [lambda t: torch.cat([t, t], 1)[:, t.shape[1]:], lambda t: torch.cat([t, t[:, :3]], 1)[:, :t.shape[1]],
             lambda t: torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape), lambda t: t.t().contiguous().t()]
    for make in views:
        other = _run(make(x), [make(t) for t in w], c, make(g))
        assert torch.equal(other[0], y) and torch.equal(other[1], gx) and all(torch.equal(p, q) for p, q in zip(other[2], gw))
    mixed = _run(x, [views[i % 4](t) for i, t in enumerate(w)], c, g)  # every matrix with a stride of its own
    assert torch.equal(mixed[0], y) and torch.equal(mixed[1], gx)


def test_counts_that_do_not_fit(gpu_device):
    """Counts below 0 count as 0; where they sum to more than there are rows, rows end first."""
    x, w, _, g = _inputs([50, 50, 50], 72, 64, BF16)
    big = 2 ** 62
    for counts, means in [([-5, 60, 200], [0, 60, 90]), ([big, big, big], [150, 0, 0]), ([100, big, -big], [100, 50, 0])]:
        for dtype in (torch.int64, torch.int32) if max(map(abs, counts)) < 2 ** 31 else (torch.int64,):
            got = _run(x, w, torch.tensor(counts, dtype=dtype, device="cuda"), g)
            want = _run(x, w, torch.tensor(means, device="cuda"), g)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and all(torch.equal(a, b) for a, b in zip(got[2], want[2]))


def test_no_rows(gpu_device):
    x, w, c, g = _inputs([0, 0], 24, 40, BF16)
    y, gx, gw = _run(x, w, c, g)
    assert y.shape == (0, 40) and gx.shape == (0, 24) and not any(t.any() for t in gw)


def test_experts_do_not_touch_each_other(gpu_device):
    """NaN in an expert's rows, and in the matrix of one without rows, stay where they are."""
    x, w, c, g = _inputs([70, 0, 130], 264, 136, BF16, 10)
    y, gx, gw = _run(x, w, c, g)
    bad = [x.clone(), [t.clone() for t in w], g.clone()]
    bad[0][:70], bad[1][1][:], bad[2][200:], bad[0][200:] = math.nan, math.nan, math.nan, math.inf
    y2, gx2, gw2 = _run(bad[0], bad[1], c, bad[2])
    assert torch.equal(y[70:], y2[70:]) and torch.equal(gx, gx2) and torch.equal(gw[2], gw2[2]) and not gw2[1].any()
    assert y2[:70].isnan().all()


def test_only_what_is_wanted(gpu_device):
    x, w, c, g = _inputs([20, 41], 64, 72, FP16)
    _, gx, gw = _run(x, w, c, g)
    leaf = x.clone().requires_grad_()
    a, = torch.autograd.grad(training.expert_linear(leaf, w, c), leaf, g)
    one = w[1].clone().requires_grad_()
    b, = torch.autograd.grad(training.expert_linear(x, [w[0], one], c), one, g)
    assert torch.equal(a, gx) and torch.equal(b, gw[1])


def test_against_differences(gpu_device):
    """The product is linear in both: one difference of the formula is its derivative."""
    x, w, c, g = _inputs([9, 0, 22], 40, 56, FP16)
    _, gx, gw = _run(x, w, c, g)
    gen = torch.Generator(device="cuda").manual_seed(3)
    value = lambda a, b: float((_formula(a, b, c.tolist(), g)[0][0] * g.double()).sum())  # noqa: E731
    here = value(x, w)
    v = torch.randn(x.shape, generator=gen, device="cuda").double()
    slope, along = value(x.double() + v, w) - here, (gx.double() * v)
    # One rounding an entry: 16 standard deviations of their sum.
    assert abs(slope - float(along.sum())) <= 16 * UNIT[FP16] * float(along.square().sum().sqrt()) + 1e-9
    v = torch.randn(w[2].shape, generator=gen, device="cuda").double()
    slope, along = value(x, [*w[:2], w[2].double() + v]) - here, (gw[2].double() * v)
    assert abs(slope - float(along.sum())) <= 16 * UNIT[FP16] * float(along.square().sum().sqrt()) + 1e-9


def test_refuses(gpu_device):
    z = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    x, w, c = z(6, 16), [z(8, 16), z(8, 16)], torch.tensor([2, 4], device="cuda")
    f = training.expert_linear
    for error, call in [
        (TypeError, lambda: f(x.float(), [t.float() for t in w], c)),
        (TypeError, lambda: f(x, [w[0], w[1].half()], c)),
        (TypeError, lambda: f(x, w, c.float())),
        (TypeError, lambda: f(x, [w[0], None], c)),
        (TypeError, lambda: f([1.0], w, c)),
        (ValueError, lambda: f(x, w, c[:1])),
        (ValueError, lambda: f(x, w, c.cpu())),
        (ValueError, lambda: f(x.cpu(), w, c)),
        (ValueError, lambda: f(x, [w[0], w[1][:7]], c)),
        (ValueError, lambda: f(x, [t[:, :15] for t in w], c)),
        (ValueError, lambda: f(x[None], w, c)),
        (ValueError, lambda: f(x, [], c)),
        (ValueError, lambda: f(x, [w[0]] * 257, z(257, dtype=torch.int32))),
        (ValueError, lambda: f(x, [torch.stack(w)] * 2, c)),
        (ValueError, lambda: f(x, z(2, 0, 16), c)),
        (ValueError, lambda: f(z(6, 0), [z(8, 0)] * 2, c)),
    ]:
        with pytest.raises(error):
            call()
    assert f(x, w, c).shape == (6, 8)


def test_second_derivative_and_changes_in_place(gpu_device):
    x, w, c, g = _inputs([4, 4], 16, 16, BF16)
    x.requires_grad_()
    a, = torch.autograd.grad(training.expert_linear(x, w, c), x, g, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(a.sum(), x)
    y = training.expert_linear(x, w, c)
    w[0].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, g)


@pytest.mark.parametrize("n_in,n_out", [(136, 264), (100, 36)])
def test_captured_and_on_another_stream(gpu_device, n_in, n_out):
    """A graph reads the counts that are there when it is replayed."""
    x, w, c, g = _inputs([30, 0, 97], n_in, n_out, BF16, 4)
    want = _run(x, w, c, g)
    flat = lambda r: [r[0], r[1], *r[2]]  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            got = _run(x, w, c, g)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(flat(got), flat(want)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _run(x, w, c, g)
    for counts in ([30, 0, 97], [0, 131, 0], [64, 1, 60]):
        c.copy_(torch.tensor(counts, dtype=torch.int32))
        for t in flat(got):
            t.fill_(7)
        graph.replay()
        want = _run(x, w, c, g)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(flat(got), flat(want)))
