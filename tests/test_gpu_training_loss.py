"""The loss over the vocabulary and its gradient, against the formula in 64 bits and against differences."""

import math

import pytest
import torch

from elasticmegatron_amd import training

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # one rounding to 8 or 11 significant bits, relative


def _inputs(tokens, hidden, rows, dtype, seed=0, ignored=0.2, vocab=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    vocab = sum(rows) if vocab is None else vocab
    h = torch.randn(tokens, hidden, generator=gen, device="cuda")
    w = [(torch.randn(r, hidden, generator=gen, device="cuda") * 2 / math.sqrt(hidden)).to(dtype) for r in rows]
    target = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    target[torch.rand(tokens, generator=gen, device="cuda") < ignored] = -100
    g = (torch.rand(tokens, generator=gen, device="cuda") - 0.3) / tokens
    return h.to(dtype), w, target, g


def _formula(h, shards, target, g, vocab):
    """loss, gradients and what bounds their errors, in 64 bits."""
    h, w = h.double(), torch.cat(list(shards)).double()
    counts = target >= 0
    x = h @ w.t()
    x[:, vocab:] = -math.inf
    lse = torch.logsumexp(x, 1)
    at = target.clamp(min=0)[:, None]
    loss = torch.where(counts, lse - x.gather(1, at)[:, 0], 0.0)
    d = torch.exp(x - lse[:, None])
    d.scatter_add_(1, at, torch.full_like(lse, -1.0)[:, None])
    d *= torch.where(counts, g.double(), 0.0)[:, None]
    # Sums of `hidden` products in 32 bits: eight standard deviations of their roundings, twice (x and lse),
    # and a few units of the exponential and the logarithm.
    size = (h.abs() @ w.abs().t()).amax(1)
    off = 16 * math.sqrt(h.shape[1]) * 2.0 ** -24 * size + 4e-6
    return loss, d, d @ w, d.t() @ h, off


def _check_gradients(h, shards, target, g, vocab, loss, gh, gw):
    want, d, dh, dw, off = _formula(h, shards, target, g, vocab)
    assert (loss.double() - want).abs().le(off).all()
    u = UNIT[h.dtype]
    w = torch.cat(list(shards)).double()
    # d has one rounding and the error of its exponent, which is relative to the probability and not to the
    # probability less one; the result has one rounding.  fp16 also has a smallest step, of d (after its
    # scaling) and of the result.
    p = d.clone()
    p.scatter_add_(1, target.clamp(min=0)[:, None], torch.where(target >= 0, g.double(), 0.0)[:, None])
    e = d.abs() * u + p.abs() * off[:, None]
    step_d, step = (float(g.abs().max()) * 2.0 ** -39, 2.0 ** -25) if h.dtype == torch.float16 else (0.0, 0.0)
    room = lambda a, b, s: a + u * 1.01 * s.abs() + step_d * b + step + 1e-12  # noqa: E731
    assert (gh.double() - dh).abs().le(room(e @ w.abs(), w.abs().sum(0)[None], dh)).all()
    got = torch.cat(list(gw)).double()
    hs = torch.where((target >= 0)[:, None], h.double().abs(), 0.0)
    assert (got - dw).abs().le(room(e.t() @ hs, hs.sum(0)[None], dw)).all()
    assert not got[vocab:].any()


@pytest.mark.parametrize("tokens,hidden,rows,vocab,dtype", [
    (1, 64, [128], None, torch.bfloat16),
    (1, 4096, [512], None, torch.bfloat16),
    (3, 8, [1], None, torch.bfloat16),
    (2, 1, [5], None, torch.float16),            # a hidden size that is no multiple of 8
    (17, 100, [300], None, torch.bfloat16),
    (16, 1000, [700], None, torch.float16),
    (33, 72, [999], 990, torch.bfloat16),
    (64, 128, [256, 256], 300, torch.bfloat16),  # a shard with padding rows
    (65, 136, [100, 100, 100, 100], 201, torch.bfloat16),  # whole shards of padding
    (255, 512, [2000, 1, 37], None, torch.bfloat16),
    (257, 520, [4099], 4000, torch.float16),
    (300, 1001, [1030], 1029, torch.bfloat16),
    (500, 512, [8000] * 4, None, torch.bfloat16),
    (2048, 1024, [32000], 31990, torch.bfloat16),
    (5000, 256, [3000, 3000], 5999, torch.bfloat16),
])
def test_loss_and_gradients(gpu_device, tokens, hidden, rows, vocab, dtype):
    vocab = sum(rows) if vocab is None else vocab
    h, w, target, g = _inputs(tokens, hidden, rows, dtype, vocab=vocab)
    h.requires_grad_()
    for x in w:
        x.requires_grad_()
    loss = training.linear_cross_entropy(h, w, target, vocab_size=vocab, reduction="none")
    assert loss.dtype == torch.float32 and loss.shape == target.shape
    gh, *gw = torch.autograd.grad(loss, [h, *w], g)
    _check_gradients(h.detach(), [x.detach() for x in w], target, g, vocab, loss.detach(), gh, gw)
    with torch.no_grad():
        assert torch.equal(training.linear_cross_entropy(h, w, target, vocab_size=vocab, reduction="none"), loss)


@pytest.mark.parametrize("tokens,hidden,rows,vocab,dtype", [
    (256, 40, [270000], 269990, torch.bfloat16),       # more rows than one piece of d holds
    (1000, 24, [35000, 35000], 69000, torch.float16),
    (130, 1003, [4100, 4000], 8090, torch.bfloat16),   # rows that do not lie on 16 bytes, shards of two sizes
    (1024, 200, [1500, 1500], None, torch.float16),
])
def test_few_tokens_and_many_rows(gpu_device, tokens, hidden, rows, vocab, dtype):
    """grad_hidden's product takes the weights as they lie."""
    vocab = sum(rows) if vocab is None else vocab
    h, w, target, g = _inputs(tokens, hidden, rows, dtype, vocab=vocab)
    for x in w:  # what does not count may hold anything
        if sum(rows) > vocab and x is w[-1]:
            x[vocab - sum(rows):] = math.nan
    lse, logit = training.vocab_statistics(h, w, target, vocab_size=vocab)
    gh, gw = training.vocab_gradients(h, w, target, lse, g, vocab_size=vocab)
    clean = [x.nan_to_num(0.0) for x in w]
    loss = torch.where(target >= 0, lse - logit, 0.0)
    _check_gradients(h, clean, target, g, vocab, loss, gh, gw)


@pytest.mark.parametrize("tokens", [1, 2, 5, 15, 16, 31, 40, 63, 64, 100, 130])
@pytest.mark.parametrize("hidden,rows,dtype", [(256, [1000], torch.bfloat16), (1000, [333, 512], torch.float16),
                                               (48, [70], torch.bfloat16)])
def test_scores_of_few_tokens(gpu_device, tokens, hidden, rows, dtype):
    h, w, target, g = _inputs(tokens, hidden, rows, dtype, seed=tokens, ignored=0.1)
    loss = training.linear_cross_entropy(h, w, target, reduction="none")
    want, *_, off = _formula(h, w, target, g, sum(rows))
    assert (loss.double() - want).abs().le(off).all()


def test_same_bits_on_every_run(gpu_device):
    h, w, target, g = _inputs(700, 320, [5000], torch.bfloat16)
    runs = []
    for _ in range(3):
        lse, logit = training.vocab_statistics(h, w, target)
        gh, gw = training.vocab_gradients(h, w, target, lse, g)
        runs.append([lse, logit, gh, *gw])
    for again in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], again))


def test_reductions_and_shapes(gpu_device):
    h, w, target, _ = _inputs(24, 64, [100], torch.bfloat16)
    h, target = h.view(2, 12, 64), target.view(2, 12)
    each = training.linear_cross_entropy(h, w[0], target, reduction="none")
    assert each.shape == (2, 12)
    assert torch.equal(training.linear_cross_entropy(h, w[0], target, reduction="sum"), each.sum())
    mean = training.linear_cross_entropy(h, w[0], target)
    assert torch.equal(mean, each.sum() / (target != -100).sum())
    h.requires_grad_()
    training.linear_cross_entropy(h, w[0], target).backward()
    got = h.grad.clone()
    h.grad = None
    (training.linear_cross_entropy(h, w[0], target, reduction="sum") / (target != -100).sum()).backward()
    assert torch.equal(got, h.grad)


@pytest.mark.parametrize("shape", [(24,), (2, 12)])
def test_losses_scaled_in_place(gpu_device, shape):
    h, w, target, _ = _inputs(24, 64, [100], torch.bfloat16)
    h, target = h.view(*shape, 64).requires_grad_(), target.view(shape)
    loss = training.linear_cross_entropy(h, w[0], target, reduction="none")
    want, = torch.autograd.grad((loss * 0.5).sum(), h)
    loss = training.linear_cross_entropy(h, w[0], target, reduction="none")
    loss *= 0.5
    got, = torch.autograd.grad(loss.sum(), h)
    assert torch.equal(got, want)


def test_no_tokens_no_rows_and_nothing_that_counts(gpu_device):
    h, w, target, g = _inputs(8, 64, [100], torch.bfloat16)
    empty = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    weight = w[0].clone().requires_grad_()
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    loss = training.linear_cross_entropy(empty, weight, none, reduction="none")
    assert loss.shape == (0,)
    gh, gw = torch.autograd.grad(loss.sum(), [empty, weight])
    assert gh.shape == (0, 64) and not gw.any()
    assert math.isnan(float(training.linear_cross_entropy(empty, weight, none)))
    # Every token ignored.
    all_ignored = torch.full((8,), -100, device="cuda")
    hid = h.clone().requires_grad_()
    loss = training.linear_cross_entropy(hid, weight, all_ignored, reduction="none")
    assert not loss.any()
    gh, gw = torch.autograd.grad(loss, [hid, weight], torch.ones_like(loss))
    assert not gh.any() and not gw.any()
    # No rows at all, and none that counts.
    for rows, size in ((w[0][:0], None), (w[0], 0)):
        lse, logit = training.vocab_statistics(h, rows, target, vocab_size=size)
        assert (lse == -math.inf).all() and (logit == -math.inf).all()
    gh, gw = training.vocab_gradients(h, w[0][:0], target, torch.zeros(8, device="cuda"), g)
    assert not gh.any() and gw[0].shape == (0, 64)
    # A target outside the vocabulary has no probability.
    outside = target.clone()
    outside[3] = 100
    outside[4] = -7
    loss = training.linear_cross_entropy(h, w[0], outside, reduction="none")
    assert torch.equal(loss.isinf(), (outside == 100) | (outside == -7))


@pytest.mark.parametrize("tokens", [4, 200])
def test_what_does_not_count_may_hold_anything(gpu_device, tokens):
    """NaN and infinities in ignored tokens' states and in padding rows reach nothing; in a token that
    counts they reach that token's loss alone."""
    h, w, target, g = _inputs(tokens, 72, [300], torch.bfloat16, ignored=0.0)
    target %= 250
    target[1] = -100
    clean = training.linear_cross_entropy(h, w, target, vocab_size=250, reduction="none")
    lse, _ = training.vocab_statistics(h, w, target, vocab_size=250)
    gh, gw = training.vocab_gradients(h, w, target, lse, g, vocab_size=250)
    bad_h, bad_w = h.clone(), w[0].clone()
    bad_h[1] = math.nan
    bad_h[1, 5] = math.inf
    bad_w[250:] = math.nan
    bad_w[260] = math.inf
    assert torch.equal(training.linear_cross_entropy(bad_h, bad_w, target, vocab_size=250, reduction="none"), clean)
    lse, _ = training.vocab_statistics(bad_h, bad_w, target, vocab_size=250)
    got_h, got_w = training.vocab_gradients(bad_h, bad_w, target, lse, g, vocab_size=250)
    assert torch.equal(got_h, gh) and torch.equal(got_w[0], gw[0])
    bad_h[2, 0] = math.nan
    loss = training.linear_cross_entropy(bad_h, bad_w, target, vocab_size=250, reduction="none")
    assert torch.equal(loss.isnan(), torch.arange(tokens, device="cuda") == 2)
    assert torch.equal(loss[3:], clean[3:])


def test_large_logits(gpu_device):
    """Logits of several hundred, and equal ones: the maximum is taken out before the exponential."""
    h = torch.full((5, 64), 8.0, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(100, 64, dtype=torch.bfloat16, device="cuda")
    w[7] = 1.0
    w[9] = -1.0
    target = torch.tensor([7, 9, 0, 7, 9], device="cuda")
    loss = training.linear_cross_entropy(h, w, target, reduction="none")
    want = torch.tensor([0.0, 1024.0, 512.0, 0.0, 1024.0], device="cuda")
    assert torch.equal(loss, want)
    same = training.linear_cross_entropy(torch.zeros_like(h), w, target, reduction="none")
    assert (same.double() - math.log(100)).abs().max() < 4e-6


def test_processes_parts_make_the_whole(gpu_device):
    """Statistics and gradients from parts of the vocabulary, as processes of tensor parallelism hold them."""
    h, w, target, g = _inputs(150, 256, [500, 500, 500], torch.bfloat16, vocab=1400)
    target[0], target[1], target[2] = 0, 499, 1399
    parts = [training.vocab_statistics(h, x, target, vocab_start=500 * i, vocab_size=1400) for i, x in enumerate(w)]
    lse, logit = training.merge_vocab_statistics(*(torch.stack(p) for p in zip(*parts)))
    counts = target != -100
    grads = [training.vocab_gradients(h, x, target, lse, g, vocab_start=500 * i, vocab_size=1400) for i, x in enumerate(w)]
    gh = sum(p[0].double() for p in grads)
    want, d, dh, dw, off = _formula(h, w, target, g, 1400)
    assert ((lse - logit).double() - want)[counts].abs().le(off[counts]).all()
    room = 3 * 2.0 ** -9 * (d.abs() @ torch.cat(w).double().abs())
    assert (gh - dh).abs().le(room + 1e-7).all()
    whole = torch.cat([p[1][0] for p in grads]).double()
    assert (whole - dw).norm() <= 2.0 ** -8 * dw.norm()


def test_strides_and_alignment(gpu_device):
    """Rows at any stride and any alignment give the values of their contiguous copies."""
    h, w, target, g = _inputs(40, 128, [200], torch.bfloat16)

    def both(hid, wt):
        lse, logit = training.vocab_statistics(hid, wt, target)
        gh, gw = training.vocab_gradients(hid, wt, target, lse, g)
        return [lse, logit, gh, *gw]

    want = both(h, w[0])
    arena = torch.zeros(200 * 160 + 40 * 200 + 7, dtype=torch.bfloat16, device="cuda")
    for offset, stride in ((0, 136), (1, 128), (3, 131), (8, 160)):
        wt = arena[offset:offset + 200 * stride].as_strided((200, 128), (stride, 1), offset)
        wt.copy_(w[0])
        for got, expect in zip(both(h, wt), want):
            assert torch.equal(got, expect), (offset, stride)
    for hid in (torch.zeros(40, 256, dtype=torch.bfloat16, device="cuda")[:, 64:192].copy_(h),
                torch.zeros(40, 131, dtype=torch.bfloat16, device="cuda")[:, 1:129].copy_(h),
                torch.zeros(128, 40, dtype=torch.bfloat16, device="cuda").t().copy_(h)):
        for got, expect in zip(both(hid, w[0]), want):
            assert torch.equal(got, expect)
    # Every token the same state: a broadcast input, whose gradient autograd sums.
    one = h[:1].clone().requires_grad_()
    loss = training.linear_cross_entropy(one.expand(40, 128), w[0], target, reduction="none")
    got, = torch.autograd.grad(loss, one, g)
    copies = h[:1].expand(40, 128).contiguous().requires_grad_()
    loss = training.linear_cross_entropy(copies, w[0], target, reduction="none")
    each, = torch.autograd.grad(loss, copies, g)
    assert torch.equal(got, each.sum(0, keepdim=True))


def test_only_the_wanted_gradients(gpu_device):
    h, w, target, g = _inputs(40, 128, [200, 100], torch.bfloat16)
    lse, _ = training.vocab_statistics(h, w, target)
    gh, gw = training.vocab_gradients(h, w, target, lse, g)
    hid = h.clone().requires_grad_()
    got, = torch.autograd.grad(training.linear_cross_entropy(hid, w, target, reduction="none"), hid, g)
    assert torch.equal(got, gh)
    second = w[1].clone().requires_grad_()
    got, = torch.autograd.grad(training.linear_cross_entropy(h, [w[0], second], target, reduction="none"), second, g)
    assert torch.equal(got, gw[1])


def test_small_gradient_weights_in_fp16(gpu_device):
    """A gradient weight of 2^-24 is below fp16's normal range; the products see it scaled."""
    h, w, target, _ = _inputs(64, 128, [500], torch.float16, ignored=0.0)
    lse, _ = training.vocab_statistics(h, w, target)
    big = training.vocab_gradients(h, w, target, lse, torch.full((64,), 2.0 ** -4, device="cuda"))
    small = training.vocab_gradients(h, w, target, lse, torch.full((64,), 2.0 ** -14, device="cuda"))
    for a, b in ((big[0], small[0]), (big[1][0], small[1][0])):
        assert (b.double() * 2 ** 10 - a.double()).abs().max() <= 2.0 ** -15  # the result's own smallest step


@pytest.mark.parametrize("up,weight", [(-60, -40), (60, 45)])  # powers of two of hidden and of grad_loss
@pytest.mark.parametrize("tokens,hidden,rows", [(40, 72, [130]), (600, 256, [3000, 3000])])
def test_scales_far_from_one(gpu_device, tokens, hidden, rows, up, weight):
    """hidden 2^up, weights 2^-up and grad_loss 2^weight of the plain ones: the same logits, and the same
    gradients times a power of two each: to the last bit where that is in the range of normal numbers."""
    h, w, target, g = _inputs(tokens, hidden, rows, torch.bfloat16)
    lse, logit = training.vocab_statistics(h, w, target)
    gh, gw = training.vocab_gradients(h, w, target, lse, g)
    far_h, far_w, far_g = h * 2.0 ** up, [x * 2.0 ** -up for x in w], g * 2.0 ** weight
    far_lse, far_logit = training.vocab_statistics(far_h, far_w, target)
    assert torch.equal(lse, far_lse) and torch.equal(logit, far_logit)
    far_gh, far_gw = training.vocab_gradients(far_h, far_w, target, far_lse, far_g)
    for got, want, by in ((far_gh, gh, weight - up), *((a, b, weight + up) for a, b in zip(far_gw, gw))):
        want = want.double() * 2.0 ** by
        room = torch.where(want.abs() < 2.0 ** -126, 2.0 ** -126, 0.0)
        assert (room == 0).any() and (got.double() - want).abs().le(room).all()


def test_gradient_against_differences(gpu_device):
    """Loss differences over steps that bf16 holds exactly."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    t, hidden, vocab = 24, 64, 300
    h = (0.5 + 0.25 * torch.rand(t, hidden, generator=gen, device="cuda")).to(torch.bfloat16)  # steps of 2^-8
    w = (0.5 + 0.25 * torch.rand(vocab, hidden, generator=gen, device="cuda")).to(torch.bfloat16)
    target = torch.randint(0, vocab, (t,), generator=gen, device="cuda")
    lse, _ = training.vocab_statistics(h, w, target)
    ones = torch.ones(t, device="cuda")
    gh, gw = training.vocab_gradients(h, w, target, lse, ones)
    total = lambda a, b: float(training.linear_cross_entropy(a, b, target, reduction="none").double().sum())  # noqa: E731
    for x, grad, loss in ((h, gh, lambda v: total(v, w)), (w, gw[0], lambda v: total(h, v))):
        step = (torch.randint(0, 2, x.shape, generator=gen, device="cuda") * 2 - 1).to(torch.bfloat16) * 2.0 ** -8
        assert torch.equal((x + step) - step, x)
        difference = (loss(x + step) - loss(x - step)) / 2
        by_gradient = float((grad.double() * step.double()).sum())
        # Roundings of the losses; the third derivative's share is (change of a logit)^3; the gradient's own
        # rounding (two of 2^-9 on every product that its sum has).
        change = float((x.double().shape[0] ** 0) * 64 * 2.0 ** -8 * 0.75)
        room = 2e-6 * t + t * change ** 3 / 6 + 2 * 2.0 ** -9 * float(grad.double().abs().sum()) * 2.0 ** -8 * 4
        assert abs(difference - by_gradient) <= room
        assert room < 0.2 * float(grad.double().abs().sum()) * 2.0 ** -8  # a wrong sign or factor would show


def test_on_another_stream(gpu_device):
    h, w, target, g = _inputs(300, 256, [4000], torch.bfloat16)
    lse, _ = training.vocab_statistics(h, w, target)
    want = training.vocab_gradients(h, w, target, lse, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again, _ = training.vocab_statistics(h, w, target)
        got = training.vocab_gradients(h, w, target, again, g)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, lse) and torch.equal(got[0], want[0]) and torch.equal(got[1][0], want[1][0])


def test_replays_of_a_graph(gpu_device):
    h, w, target, g = _inputs(130, 256, [1000], torch.bfloat16)
    lse, _ = training.vocab_statistics(h, w, target)
    training.vocab_gradients(h, w, target, lse, g)  # warm
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got_lse, got_logit = training.vocab_statistics(h, w, target)
        got_h, got_w = training.vocab_gradients(h, w, target, got_lse, g)
    for seed in range(1, 4):
        h2, _, t2, g2 = _inputs(130, 256, [1000], torch.bfloat16, seed=seed)
        h.copy_(h2), target.copy_(t2), g.copy_(g2)
        graph.replay()
        torch.cuda.synchronize()
        lse, logit = training.vocab_statistics(h, w, target)
        gh, gw = training.vocab_gradients(h, w, target, lse, g)
        assert torch.equal(got_lse, lse) and torch.equal(got_logit, logit)
        assert torch.equal(got_h, gh) and torch.equal(got_w[0], gw[0])
