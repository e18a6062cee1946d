"""The norms around a block with what joins it to the residual stream, against the formula in 64 bits and against differences."""

import math

import pytest
import torch

from elasticmegatron_amd import training

pytestmark = pytest.mark.gpu

EPS = 1e-5
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
UNIT = {BF16: 2.0 ** -8, FP16: 2.0 ** -11, FP32: 2.0 ** -24}  # at least half a step, relative
STEP = {BF16: 2.0 ** -134, FP16: 2.0 ** -25, FP32: 2.0 ** -150}  # half the smallest number


def _inputs(tokens, h, dtype, stream=None, branch_norm=False, gate=None, seed=0, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    x = dict(residual=(normal(tokens, h) * 3).to(stream or dtype), branch=normal(tokens, h).to(dtype), weight=(1 + 0.3 * normal(h)).to(dtype))
    if branch_norm:
        x["branch_weight"] = (1 + 0.3 * normal(h)).to(dtype)
    if gate:
        x["gate"] = normal(*((h,) if gate == "channel" else (tokens, h))).to(dtype)
    return x, [normal(tokens, h).to(stream or dtype), normal(tokens, h).to(dtype)]


def _formula(x, grads, scale):
    """Outputs, gradients and what bounds their errors but for the last rounding, in 64 bits.

    Sums in 32 bits go through at most 46 additions one after the other in a row (32 of a lane's, 6 in a wave, 8
    waves) and tokens / 512 + 100 over tokens; with the products and roots around them, 100 roundings bound a row's."""
    f = 100 * 2.0 ** -24
    r, b, w = (x[k].double() for k in ("residual", "branch", "weight"))
    bw, g = (x[k].double() if k in x else None for k in ("branch_weight", "gate"))
    rb = ((b * b).mean(-1, keepdim=True) + EPS).rsqrt()
    hat_b = b * rb
    n = b if bw is None else hat_b * bw
    s = scale * r + (n if g is None else g * n)
    e_s = f * ((scale * r).abs() + (n if g is None else g * n).abs())
    rs = ((s * s).mean(-1, keepdim=True) + EPS).rsqrt()
    hat = s * rs
    # The square root of a mean of squares is off by no more than the values are, in root mean square.
    e_rs = rs * ((e_s.square().mean(-1, keepdim=True)).sqrt() * rs + f)
    out, err = [s, hat * w], [e_s, w.abs() * (e_s * rs + s.abs() * e_rs + f * hat.abs())]
    if grads is None:
        return out, err
    ds, do = (t.double() for t in grads)
    u = UNIT[x["residual"].dtype]
    e_hat = u * hat.abs() + e_s * rs + s.abs() * e_rs  # of the stream as it was rounded
    d = do * w
    c, e_c = (d * hat).mean(-1, keepdim=True), (d.abs() * (e_hat + f * hat.abs())).mean(-1, keepdim=True)
    total = ds + rs * (d - hat * c)
    e = f * (ds.abs() + rs * (d.abs() + (hat * c).abs())) + rs * (e_hat * c.abs() + hat.abs() * e_c) + e_rs * (d - hat * c).abs()
    over = (ds.shape[0] / 512 + 200) * 2.0 ** -24
    grad, grad_err = dict(residual=scale * total, weight=(do * hat).sum(0)), dict(residual=abs(scale) * e, weight=(do.abs() * (e_hat + over * hat.abs())).sum(0))
    dn, e_n = (total, e) if g is None else (total * g, e * g.abs() + f * (total * g).abs())
    if g is not None:
        dg, e_g = total * n, e * n.abs() + (f + over) * (total * n).abs()
        grad["gate"], grad_err["gate"] = (dg.sum(0), e_g.sum(0)) if g.dim() == 1 and b.dim() == 2 else (dg, e_g)
    if bw is not None:
        grad["branch_weight"], grad_err["branch_weight"] = (dn * hat_b).sum(0), (e_n * hat_b.abs() + (f + over) * (dn * hat_b).abs()).sum(0)
        q, e_q = dn * bw, e_n * bw.abs()
        c = (q * hat_b).mean(-1, keepdim=True)
        e_c = (e_q * hat_b.abs() + f * (q * hat_b).abs()).mean(-1, keepdim=True)
        dn = rb * (q - hat_b * c)
        e_n = rb * (e_q + hat_b.abs() * e_c + 2 * f * (q.abs() + (hat_b * c).abs()))
    grad["branch"], grad_err["branch"] = dn, e_n
    return out, err, grad, grad_err


def _close(got, want, err, what):
    u, step = UNIT[got.dtype], STEP[got.dtype]
    off = (got.double() - want).abs()
    room = err + u * (want.abs() + err) + step
    assert off.le(room).all(), (what, float((off - room).max()), float((off / room).max()))


def _run(x, grads, scale):
    x = {k: v.detach().requires_grad_() for k, v in x.items()}
    outputs = training.residual_norm(x["residual"], x["branch"], x["weight"], branch_weight=x.get("branch_weight"), gate=x.get("gate"),
                                     residual_scale=scale, eps=EPS)
    got = dict(zip(x, torch.autograd.grad(outputs, list(x.values()), grads)))
    return [o.detach() for o in outputs], got


CASES = [
    (1, 1, BF16, None, False, None, 1.0),
    (1, 8, BF16, None, True, "channel", 0.5),
    (3, 7, FP16, None, True, "token", 1.0),
    (5, 64, BF16, FP32, False, None, 2.0),
    (2, 500, FP16, FP32, True, None, 1.0),
    (17, 512, BF16, None, False, None, 1.0),
    (64, 513, BF16, None, True, "channel", 0.9),
    (100, 1000, FP16, None, False, "token", 1.0),
    (33, 1024, BF16, None, False, "channel", 1.0),
    (9, 2047, BF16, FP32, True, "token", -1.5),
    (50, 2048, BF16, None, True, None, 0.7),
    (40, 2056, FP16, FP32, True, "channel", 1.0),
    (700, 4096, BF16, None, False, None, 1.0),
    (20, 4097, BF16, None, False, None, 1.0),
    (300, 5120, BF16, FP32, True, "channel", 1.0),
    (30, 8192, FP16, None, True, "token", 0.5),
    (4, 12000, BF16, None, True, "channel", 1.0),
    (3, 16383, BF16, FP32, False, None, 1.0),
    (6, 16384, FP16, None, True, "channel", 1.0),
    (5000, 136, BF16, None, True, "channel", 1.0),
    (2600, 1000, BF16, FP32, False, None, 1.0),
]


@pytest.mark.parametrize("tokens,h,dtype,stream,branch_norm,gate,scale", CASES)
def test_outputs_and_gradients(gpu_device, tokens, h, dtype, stream, branch_norm, gate, scale):
    x, grads = _inputs(tokens, h, dtype, stream, branch_norm, gate)
    want, err, grad, grad_err = _formula(x, grads, scale)
    got, got_grad = _run(x, grads, scale)
    assert got[0].dtype == (stream or dtype) and got[1].dtype == dtype
    for g, w, e, what in zip(got, want, err, ("stream", "normed")):
        _close(g, w, e, what)
    for k, v in x.items():
        assert got_grad[k].dtype == v.dtype and got_grad[k].shape == v.shape
        _close(got_grad[k], grad[k], grad_err[k], k)
    with torch.no_grad():
        again = training.residual_norm(x["residual"], x["branch"], x["weight"], branch_weight=x.get("branch_weight"), gate=x.get("gate"),
                                       residual_scale=scale, eps=EPS)
    assert all(torch.equal(a, b) for a, b in zip(again, got))
    _, same = _run(x, grads, scale)
    assert all(torch.equal(same[k], got_grad[k]) for k in x)  # the same bits every time


@pytest.mark.parametrize("tokens,h,dtype,wide", [(7, 512, BF16, False), (130, 1000, FP16, True), (1, 4096, BF16, True), (12, 77, BF16, False)])
def test_norm_alone(gpu_device, tokens, h, dtype, wide):
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = (torch.randn(tokens, h, generator=gen, device="cuda") * 5).to(FP32 if wide else dtype).requires_grad_()
    w = torch.randn(h, generator=gen, device="cuda").to(dtype).requires_grad_()
    g = torch.randn(tokens, h, generator=gen, device="cuda").to(dtype)
    y = training.rms_norm(x, w, eps=EPS)
    gx, gw = torch.autograd.grad(y, [x, w], g)
    zero = torch.zeros_like(x)
    parts = dict(residual=x.detach(), branch=zero.detach().to(dtype), weight=w.detach())
    want, err, grad, grad_err = _formula(parts, [zero.detach(), g], 1.0)
    _close(y.detach(), want[1], err[1], "y")
    _close(gx, grad["residual"], grad_err["residual"], "x")
    _close(gw, grad["weight"], grad_err["weight"], "weight")


def test_norm_behind_the_block_alone(gpu_device):
    """No weight: the stream is all that comes back."""
    x, grads = _inputs(37, 264, BF16, FP32, True, "channel")
    leaves = {k: v.requires_grad_() for k, v in x.items() if k != "weight"}
    stream = training.residual_norm(leaves["residual"], leaves["branch"], branch_weight=leaves["branch_weight"], gate=leaves["gate"],
                                    residual_scale=0.8, eps=EPS)
    got = dict(zip(leaves, torch.autograd.grad(stream, list(leaves.values()), grads[0])))
    want, err, grad, grad_err = _formula({k: v.detach() for k, v in x.items()}, [grads[0], torch.zeros_like(grads[1])], 0.8)
    _close(stream.detach(), want[0], err[0], "stream")
    for k in leaves:
        _close(got[k], grad[k], grad_err[k], k)


@pytest.mark.parametrize("used", ["stream", "normed"])
def test_one_output_of_two_is_used(gpu_device, used):
    x, grads = _inputs(21, 520, BF16, None, True, "token")
    leaves = {k: v.detach().requires_grad_() for k, v in x.items()}
    stream, normed = training.residual_norm(leaves["residual"], leaves["branch"], leaves["weight"], branch_weight=leaves["branch_weight"],
                                            gate=leaves["gate"], eps=EPS)
    keys = [k for k in leaves if used == "normed" or k != "weight"]
    got = torch.autograd.grad(stream if used == "stream" else normed, [leaves[k] for k in keys], grads[0 if used == "stream" else 1])
    rest = [grads[0], torch.zeros_like(grads[1])] if used == "stream" else [torch.zeros_like(grads[0]), grads[1]]
    _, _, grad, grad_err = _formula(x, rest, 1.0)
    for k, g in zip(keys, got):
        _close(g, grad[k], grad_err[k], k)


def test_only_what_is_wanted(gpu_device):
    x, grads = _inputs(50, 136, BF16, None, True, "channel")
    _, every = _run(x, grads, 1.0)
    for only in x:
        leaves = {k: v.detach().requires_grad_(k == only) for k, v in x.items()}
        outputs = training.residual_norm(leaves["residual"], leaves["branch"], leaves["weight"], branch_weight=leaves["branch_weight"],
                                         gate=leaves["gate"], eps=EPS)
        g, = torch.autograd.grad(outputs, [leaves[only]], grads)
        assert torch.equal(g, every[only])


def test_strides_and_shapes(gpu_device):
    """Views of wider rows, rows off 16 bytes, turned gradients and inputs, and leading dimensions."""
    x, grads = _inputs(24, 256, BF16, None, True, "token")
    want, want_grad = _run(x, grads, 1.0)
    for make in (lambda t: torch.cat([t, t], -1)[..., t.shape[-1]:],
                 lambda t: torch.cat([t, t[..., :3]], -1)[..., :t.shape[-1]],
                 lambda t: torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape),
                 lambda t: t.t().contiguous().t() if t.dim() == 2 else t):
        views = {k: make(v) for k, v in x.items()}
        assert all(torch.equal(views[k], x[k]) for k in x)
        got, got_grad = _run(views, [make(g) for g in grads], 1.0)
        # Another order of sums: within two roundings of each other.
        for a, b in [*zip(got, want), *((got_grad[k], want_grad[k]) for k in x)]:
            assert (a.double() - b.double()).abs().le(2 * UNIT[BF16] * b.double().abs() + 2.0 ** -14).all()
    cube = {k: v.view(4, 6, 256) if v.dim() == 2 else v for k, v in x.items()}
    got, got_grad = _run(cube, [g.view(4, 6, 256) for g in grads], 1.0)
    assert got[0].shape == got_grad["gate"].shape == (4, 6, 256)
    assert all(torch.equal(a.view(24, 256), b) for a, b in zip(got, want))
    one, _ = _run({k: v[3] if v.dim() == 2 else v for k, v in x.items()}, [g[3] for g in grads], 1.0)
    assert all(torch.equal(a, b[3]) for a, b in zip(one, want))


def test_no_tokens(gpu_device):
    x, grads = _inputs(0, 64, BF16, None, True, "channel")
    got, grad = _run(x, grads, 1.0)
    assert got[0].shape == (0, 64) and not grad["weight"].any() and not grad["gate"].any() and grad["branch"].shape == (0, 64)


def test_rows_do_not_touch_each_other(gpu_device):
    """A token of infinities and NaN leaves the others' bits as they are."""
    x, grads = _inputs(40, 1000, BF16, None, True, "token")
    got, grad = _run(x, grads, 1.0)
    bad = {k: v.clone() for k, v in x.items()}
    bad["branch"][7], bad["residual"][20, 5] = math.nan, math.inf
    got_bad, grad_bad = _run(bad, grads, 1.0)
    keep = torch.ones(40, dtype=torch.bool, device="cuda")
    keep[[7, 20]] = False
    for a, b in [*zip(got, got_bad), *((grad[k], grad_bad[k]) for k in ("residual", "branch", "gate"))]:
        assert torch.equal(a[keep], b[keep])
    assert got_bad[1][7].isnan().all()


@pytest.mark.parametrize("size", [0.0, 1e-20, 1e-3, 200.0])
def test_sizes_of_rows(gpu_device, size):
    """eps decides where a row is small; rows of zeros give zeros, and finite gradients."""
    x, grads = _inputs(5, 300, BF16, FP32, True)
    x["residual"] *= size
    x["branch"] *= size
    want, err, grad, grad_err = _formula(x, grads, 1.0)
    got, got_grad = _run(x, grads, 1.0)
    _close(got[1], want[1], err[1], "normed")
    for k in x:
        assert got_grad[k].isfinite().all()
        _close(got_grad[k], grad[k], grad_err[k], k)


def test_against_differences(gpu_device):
    """The gradients of the kernels against differences of the formula's outputs, along random directions."""
    x, grads = _inputs(6, 96, FP16, FP32, True, "channel")
    _, grad = _run(x, grads, 0.7)

    def value(t):
        out = _formula(t, None, 0.7)[0]
        return sum(float((o * g.double()).sum()) for o, g in zip(out, grads))

    gen = torch.Generator(device="cuda").manual_seed(9)
    for k in x:
        v = torch.randn(x[k].shape, generator=gen, device="cuda").double()
        at = lambda h: value({**{n: t.double() for n, t in x.items()}, k: x[k].double() + h * v})  # noqa: E731
        slope = (at(1e-5) - at(-1e-5)) / 2e-5
        along = float((grad[k].double() * v).sum())
        # Each entry of the gradient has one rounding to its type (and hat's): 16 standard deviations of their sum.
        room = 16 * UNIT[FP16] * float((grad[k].double() * v).square().sum().sqrt()) + 1e-6 * abs(slope) + 1e-6
        assert abs(slope - along) <= room, (k, slope, along, room)


def test_refuses(gpu_device):
    z = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    r, b, w = z(4, 8), z(4, 8), z(8)
    f = training.residual_norm
    for error, call in [
        (TypeError, lambda: f(r, None, w)),
        (TypeError, lambda: f(None, b, w)),
        (TypeError, lambda: training.rms_norm(r, None)),
        (TypeError, lambda: f(r, b.float(), w)),
        (TypeError, lambda: f(r, b, w.half())),
        (TypeError, lambda: f(r.half(), b, w)),
        (TypeError, lambda: f(r, b, w, gate=z(8, dtype=FP32))),
        (TypeError, lambda: f(r.double(), b, w)),
        (ValueError, lambda: f(r, b[:3], w)),
        (ValueError, lambda: f(r, b, w[:7])),
        (ValueError, lambda: f(r, b, w, branch_weight=z(4, 8))),
        (ValueError, lambda: f(r, b, w, gate=z(4, 1))),
        (ValueError, lambda: f(r, b, w.cpu())),
        (ValueError, lambda: f(r.cpu(), b, w)),
        (ValueError, lambda: training.rms_norm(z(2, 16385), z(16385))),
        (ValueError, lambda: training.rms_norm(z(2, 0), z(0))),
        (ValueError, lambda: training.rms_norm(z(()), w)),
    ]:
        with pytest.raises(error):
            call()
    assert f(r, b, w)[1].isfinite().all()


def test_second_derivative_and_changes_in_place(gpu_device):
    x, grads = _inputs(4, 64, BF16)
    leaves = {k: v.requires_grad_() for k, v in x.items()}
    outputs = training.residual_norm(leaves["residual"], leaves["branch"], leaves["weight"])
    g, = torch.autograd.grad(outputs, [leaves["branch"]], grads, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), leaves["branch"])
    outputs = training.residual_norm(leaves["residual"], leaves["branch"], leaves["weight"])
    with torch.no_grad():
        leaves["weight"].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(outputs, [leaves["branch"]], grads)


def test_captured_and_on_another_stream(gpu_device):
    """Forward and backward in a graph, replayed with other work between, and on a stream of their own."""
    x, grads = _inputs(70, 520, BF16, None, True, "channel")
    want, want_grad = _run(x, grads, 1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            got, grad = _run(x, grads, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(grad[k], want_grad[k]) for k in x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, grad = _run(x, grads, 1.0)
    for _ in range(3):
        for t in (*got, *grad.values()):
            t.fill_(7)
        graph.replay()
        _run(x, grads, 0.5)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(grad[k], want_grad[k]) for k in x)


def test_more_rows_than_a_line_of_a_launch(gpu_device):
    n = (1 << 26) + 77
    x = torch.ones(n, 8, dtype=torch.bfloat16, device="cuda")
    x[-1] = torch.arange(1, 9)
    w = torch.full((8,), 2.0, dtype=torch.bfloat16, device="cuda")
    y = training.rms_norm(x, w, eps=0.0)
    assert y[:-1].eq(2.0).all()
    want = 2 * x[-1].double() / x[-1].double().square().mean().sqrt()
    assert (y[-1].double() - want).abs().le(2.0 ** -8 * want * (1 + 2.0 ** -10)).all()


@pytest.mark.parametrize("tokens,h,dtype,stream,branch_norm,gate", [
    (1, 8, BF16, None, True, "token"), (15, 64, BF16, None, False, None), (16, 128, FP16, None, True, "channel"), (17, 128, BF16, FP32, True, "token"),
    (333, 104, BF16, FP32, False, "channel"), (7, 136, BF16, None, True, "channel"), (8, 256, FP16, FP32, True, "token"), (9, 256, BF16, None, False, None),
    (20000, 128, BF16, None, False, None), (10001, 200, FP16, None, True, "channel"), (50, 264, BF16, None, True, "channel"),
])
def test_short_rows(gpu_device, tokens, h, dtype, stream, branch_norm, gate):
    """Several rows to a wave, whose last may have none; and more rows than all workgroups take at once."""
    x, grads = _inputs(tokens, h, dtype, stream, branch_norm, gate)
    want, err, grad, grad_err = _formula(x, grads, 0.75)
    got, got_grad = _run(x, grads, 0.75)
    for g, w, e, what in zip(got, want, err, ("stream", "normed")):
        _close(g, w, e, what)
    for k, v in x.items():
        _close(got_grad[k], grad[k], grad_err[k], k)
