"""Tokens whose loss counts for very different amounts: each one's gradient is as exact as if it were alone."""

import math

import pytest
import torch

from elasticmegatron_amd import training

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # one rounding to 8 or 11 significant bits, relative


def _inputs(tokens, hidden, rows, dtype, spread, largest):
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    r = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    h, w = r(tokens, hidden).to(dtype), (r(rows, hidden) * 2 / math.sqrt(hidden)).to(dtype)
    target = torch.randint(0, rows, (tokens,), generator=gen, device="cuda")
    target[torch.rand(tokens, generator=gen, device="cuda") < 0.1] = -100
    g = largest * 10.0 ** (-spread * torch.rand(tokens, generator=gen, device="cuda"))
    g[0], target[0] = largest, 1
    g[1] = 0.0
    g[torch.rand(tokens, generator=gen, device="cuda") < 0.5] *= -1
    if tokens > 2:
        g[2], target[2] = 1e30, -100  # ignored: its weight is no scale of anything
    return h, w, target, g


def _check(h, w, target, g):
    lse, logit = training.vocab_statistics(h, w, target)
    gh, (gw,) = training.vocab_gradients(h, w, target, lse, g)
    hd, wd, counts = h.double(), w.double(), target >= 0
    gd = torch.where(counts, g.double(), 0.0)
    x = hd @ wd.t()
    p = torch.exp(x - torch.logsumexp(x, 1)[:, None])
    d = p * gd[:, None]
    rows = counts.nonzero()[:, 0]
    d[rows, target[rows]] -= gd[rows]
    u = UNIT[h.dtype]
    # One rounding of d; its exponent's error, relative to the probability: sums of `hidden` products in 32 bits
    # (sixteen standard deviations of x's and lse's roundings) and a few units of exponential and logarithm.
    size = (hd.abs() @ wd.abs().t()).amax(1)
    off = 16 * math.sqrt(h.shape[1]) * 2.0 ** -24 * size + 4e-6
    e = d.abs() * u + (p * gd.abs()[:, None]) * off[:, None]
    # d's smallest step: with a token's own scale its weight lies in [2^13, 2^14), fp16's step is 2^-24.
    step = gd.abs() * 2.0 ** -38
    tiny = 2.0 ** -25 if h.dtype == torch.float16 else 0.0  # half the result's own smallest step
    want = d @ wd
    room = e @ wd.abs() + step[:, None] * wd.abs().sum(0) + 1.01 * u * want.abs() + tiny
    assert (gh.double() - want).abs().le(room).all()
    # grad_weights sums over the tokens: hidden states carry the weights' ratio there, in fp16 under a scale that
    # brings the largest to [2^13, 2^14), and lose what is below its step (powers of two: twice the ratio at most).
    hc = torch.where(counts[:, None], hd.abs(), 0.0)
    share = d.abs() / gd.abs().clamp(min=1e-300)[:, None]
    lost = float(gd.abs().max()) * float(hc.max()) * 2.0 ** -37 * share.sum(0)
    want = d.t() @ hd
    room = e.t() @ hc + step @ hc + lost[:, None] + 1.01 * u * want.abs() + tiny
    assert (gw.double() - want).abs().le(room).all()


@pytest.mark.parametrize("tokens,hidden,rows,dtype", [
    (3, 64, 100, torch.bfloat16),
    (64, 256, 3000, torch.bfloat16),      # d in two bf16 parts
    (257, 128, 2000, torch.bfloat16),
    (512, 256, 32000, torch.bfloat16),
    (700, 1000, 5000, torch.bfloat16),
    (700, 1001, 500, torch.bfloat16),     # rows off 16 bytes
    (2048, 128, 70000, torch.bfloat16),   # several pieces of d
    (130, 200, 1500, torch.float16),      # the weights as they lie
    (900, 72, 1500, torch.float16),
])
@pytest.mark.parametrize("spread", [0, 4, 10, 20])
def test_weights_of_tokens_over_many_decades(gpu_device, tokens, hidden, rows, dtype, spread):
    if dtype == torch.float16 and spread > 4:
        spread = 7  # results of 16 bits with five of exponent hold no more
    _check(*_inputs(tokens, hidden, rows, dtype, spread, 1e3 if dtype == torch.float16 else 0.3))


def test_one_token_does_not_depend_on_the_others_weights(gpu_device):
    """Its row of the hidden states' gradient keeps its bits, whatever the others count for."""
    for tokens, dtype in ((300, torch.bfloat16), (40, torch.bfloat16), (40, torch.float16), (900, torch.float16)):
        h, w, target, _ = _inputs(tokens, 128, 2000, dtype, 0, 1.0)
        target[:3] = 5
        lse, _ = training.vocab_statistics(h, w, target)
        rows = []
        for others in (1.0, 1e6, 1e12):
            g = torch.full((tokens,), others, device="cuda")
            g[7] = 0.625
            rows.append(training.vocab_gradients(h, w, target, lse, g)[0][7])
        assert target[7] < 0 or rows[0].any()
        assert torch.equal(rows[0], rows[1]) and torch.equal(rows[0], rows[2])


def test_weights_that_are_not_finite_spoil_their_own_rows(gpu_device):
    h, w, target, g = _inputs(300, 128, 2000, torch.bfloat16, 10, 0.5)
    target[5:8] = 9
    lse, _ = training.vocab_statistics(h, w, target)
    clean, _ = training.vocab_gradients(h, w, target, lse, g)
    g[5], g[6], g[7] = math.nan, math.inf, -math.inf
    gh, _ = training.vocab_gradients(h, w, target, lse, g)
    bad = torch.zeros(300, dtype=torch.bool, device="cuda")
    bad[5:8] = True
    assert not gh[bad].isfinite().any() and torch.equal(gh[~bad], clean[~bad])


@pytest.mark.parametrize("tokens", [40, 300])
def test_weights_at_the_end_of_their_range(gpu_device, tokens):
    """grad_loss of 2^120, against weights of 2^-60: the plain gradient times 2^60, to the last bit."""
    h, w, target, g = _inputs(tokens, 128, 2000, torch.bfloat16, 1, 1.0)
    g[2] = 1.0
    lse, _ = training.vocab_statistics(h, w, target)
    gh, _ = training.vocab_gradients(h, w, target, lse, g)
    far, _ = training.vocab_gradients(h * 2.0 ** 60, w * 2.0 ** -60, target, lse, g * 2.0 ** 120)
    assert torch.equal(far.double(), gh.double() * 2.0 ** 60)
