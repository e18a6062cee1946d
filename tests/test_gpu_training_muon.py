"""Newton-Schulz orthogonalisation, the Muon update and the AdamW update, against the formulas in 64 bits."""

import math

import pytest
import torch

from elasticmegatron_amd import training

pytestmark = pytest.mark.gpu

A, B, C = training.MUON_COEFFICIENTS
# How far the result may be off in norm: the products' roundings, and one rounding to bf16 where the result
# is bf16.
PRODUCTS, BF16 = 2e-3, 2.0 ** -9


def _newton_schulz(u, steps=5, coefficients=None, eps=1e-7):
    x = u.double()
    x = x / (torch.linalg.matrix_norm(x) + eps)
    for k in range(steps):
        a, b, c = coefficients[k] if coefficients else (A, B, C)
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x


def _matrix(rows, cols, spectrum="flat", seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    m = torch.randn(rows, cols, generator=gen, device="cuda", dtype=torch.float64)
    if spectrum == "flat":
        return m.float()
    n = min(rows, cols)
    q, _ = torch.linalg.qr(torch.randn(rows, n, generator=gen, device="cuda", dtype=torch.float64))
    p, _ = torch.linalg.qr(torch.randn(cols, n, generator=gen, device="cuda", dtype=torch.float64))
    i = torch.arange(1, n + 1, device="cuda", dtype=torch.float64)
    s = {"1/i": 1 / i, "1/i^2": i ** -2.0, "exp": torch.exp(-i / 20), "four": torch.where(i <= 4, 1.0, 1e-3),
         "one": (i == 1).double()}[spectrum]
    return ((q * s) @ p.t()).float()


def _off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (5, 1), (16, 16), (63, 65), (64, 64), (100, 37), (128, 384), (129, 127),
                                       (300, 1000), (1376, 512), (700, 700), (2668, 1000), (512, 4100), (2048, 2048)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shapes(gpu_device, rows, cols, dtype):
    u = _matrix(rows, cols).to(dtype)
    got = training.orthogonalise(u)
    assert got.dtype == torch.bfloat16 and got.shape == u.shape
    assert _off(got, _newton_schulz(u)) <= PRODUCTS + BF16


@pytest.mark.parametrize("spectrum", ["1/i", "1/i^2", "exp", "four", "one"])
@pytest.mark.parametrize("rows,cols", [(256, 256), (200, 600), (700, 300)])
def test_spectra(gpu_device, spectrum, rows, cols):
    """Small singular values grow by a in every step, and roundings with them."""
    u = _matrix(rows, cols, spectrum)
    assert _off(training.orthogonalise(u), _newton_schulz(u)) <= PRODUCTS + BF16


@pytest.mark.parametrize("rows,cols", [(33, 300), (64, 64), (100, 37), (128, 160), (301, 700), (700, 303), (260, 1300)])
def test_rank_one(gpu_device, rows, cols):
    """Every direction but one holds nothing but roundings: what the first two parts of an entry lose shows most."""
    for seed in range(1, 4):
        u = _matrix(rows, cols, "one", seed)
        assert _off(training.orthogonalise(u), _newton_schulz(u)) <= PRODUCTS + BF16


@pytest.mark.parametrize("scale", [1e-12, 1e-3, 1.0, 1e6, 1e15])
def test_scales(gpu_device, scale):
    """The norm takes out the scale; far below eps the result goes to zero with it."""
    u = _matrix(96, 160) * scale
    want = _newton_schulz(u)
    if want.abs().max() < 1e-4:  # entries far below the format's: absolute
        assert (training.orthogonalise(u).double() - want).abs().max() <= 1e-6
    else:
        assert _off(training.orthogonalise(u), want) <= PRODUCTS + BF16


def test_zeros_and_one_large_entry(gpu_device):
    assert not training.orthogonalise(torch.zeros(70, 90, device="cuda")).any()
    u = torch.zeros(70, 90, device="cuda")
    u[3, 4] = -5.0
    got = training.orthogonalise(u)
    assert _off(got, _newton_schulz(u)) <= PRODUCTS + BF16
    assert (got != 0).sum() == 1


def test_a_matrix_that_is_not_finite_spoils_itself_alone(gpu_device):
    u = torch.stack([_matrix(80, 100, seed=s) for s in range(3)])
    clean = training.orthogonalise(u)
    u[1, 4, 4] = math.nan
    got = training.orthogonalise(u)
    assert got[1].isnan().all()
    assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])


@pytest.mark.parametrize("steps", [1, 2, 3, 8])
def test_steps_and_their_coefficients(gpu_device, steps):
    u = _matrix(150, 210)
    own = [(2.0 - 0.1 * k, -1.5 + 0.1 * k, 0.5) for k in range(steps)]  # all keep 1 at 1
    assert _off(training.orthogonalise(u, steps=steps, coefficients=own), _newton_schulz(u, steps, own)) <= PRODUCTS + BF16


def test_stacks_and_sequences(gpu_device):
    u = torch.stack([_matrix(130, 70, seed=s) for s in range(5)])
    alone = torch.stack([training.orthogonalise(x) for x in u])
    assert torch.equal(training.orthogonalise(u), alone)
    assert torch.equal(torch.stack(training.orthogonalise(list(u))), alone)
    many = u.repeat(8, 1, 1)  # more than one native call takes
    assert torch.equal(training.orthogonalise(many), alone.repeat(8, 1, 1))
    assert training.orthogonalise([]) == []
    assert training.orthogonalise(u[:0]).shape == (0, 130, 70)
    assert training.orthogonalise(torch.zeros(0, 5, device="cuda")).shape == (0, 5)


def test_strides(gpu_device):
    u = _matrix(90, 140)
    want = training.orthogonalise(u)
    for shape, cut in (((90, 150), slice(0, 140)), ((90, 143), slice(3, 143))):
        wide = torch.full(shape, math.nan, device="cuda")
        wide[:, cut] = u
        assert torch.equal(training.orthogonalise(wide[:, cut]), want)
    assert torch.equal(training.orthogonalise(u.t().contiguous().t()), want)
    odd = torch.empty(90 * 140 + 1, device="cuda")[1:].view(90, 140).copy_(u)  # off 16 bytes
    assert torch.equal(training.orthogonalise(odd), want)


def _state(count, rows, cols, dtype):
    gen = torch.Generator(device="cuda").manual_seed(rows)
    r = lambda: torch.randn(count, rows, cols, generator=gen, device="cuda")  # noqa: E731
    return r() * 0.02, r() * 1e-3, (r() * 1e-3).to(dtype), torch.zeros(count, rows, cols, dtype=torch.bfloat16, device="cuda")


@pytest.mark.parametrize("count,rows,cols,dtype", [(1, 64, 64, torch.float32), (3, 100, 37, torch.bfloat16),
                                                   (2, 512, 1376, torch.float32), (2, 1001, 333, torch.float16),
                                                   (1, 1, 9, torch.float32), (40, 24, 40, torch.bfloat16)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step(gpu_device, count, rows, cols, dtype, nesterov):
    main, buf, grad, image = _state(count, rows, cols, dtype)
    lr, mu, decay, rms = 0.02, 0.9, 0.1, 0.2
    want_buf = mu * buf.double() + grad.double()
    u = grad.double() + mu * want_buf if nesterov else want_buf
    o = torch.stack([_newton_schulz(x) for x in u])
    rate = lr * rms * math.sqrt(max(rows, cols))
    want = main.double() * (1 - lr * decay) - rate * o
    scale_buf = (mu * buf.double()).abs() + grad.double().abs()
    before = main.clone()
    training.muon_step(main, buf, grad, model=image, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=decay, rms_scale=rms)
    assert (buf.double() - want_buf).abs().le(2.0 ** -22 * scale_buf).all()
    off = (main.double() - want).flatten(1).norm(dim=1)
    assert off.le(PRODUCTS * rate * o.flatten(1).norm(dim=1) + 2.0 ** -22 * before.double().flatten(1).norm(dim=1)).all()
    assert torch.equal(image, main.to(torch.bfloat16))


def test_muon_step_on_views_of_an_arena(gpu_device):
    """Matrices that lie anywhere in a state's arenas, without an image; neighbours stay as they are."""
    rows, cols = 50, 66
    n = rows * cols
    main, buf, grad, _ = _state(2, rows, cols, torch.float32)
    arenas = [torch.full((2 * n + 40,), 7.0, device="cuda") for _ in range(2)]
    places = (3, 3 + n + 9)
    views = [[a[p:p + n].view(rows, cols) for p in places] for a in arenas]
    for vs, t in zip(views, (main, buf)):
        for v, x in zip(vs, t):
            v.copy_(x)
    training.muon_step(*views, list(grad), lr=0.01)
    training.muon_step(main, buf, grad, lr=0.01)
    for vs, t, arena in zip(views, (main, buf), arenas):
        for v, x in zip(vs, t):
            assert torch.equal(v, x)
        outside = torch.ones_like(arena, dtype=torch.bool)
        for p in places:
            outside[p:p + n] = False
        assert (arena[outside] == 7.0).all()


def test_muon_replays_of_a_graph_and_another_stream(gpu_device):
    main, buf, grad, image = _state(2, 130, 260, torch.float32)
    eager = [t.clone() for t in (main, buf)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        training.muon_step(*[t.clone() for t in (main, buf)], grad, lr=0.01)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        training.muon_step(main, buf, grad, model=image, lr=0.01)
    for k in range(3):
        grad.mul_(-1.5)
        graph.replay()
        torch.cuda.synchronize()
        training.muon_step(*eager, grad, lr=0.01)
        assert torch.equal(main, eager[0]) and torch.equal(buf, eager[1])
        assert torch.equal(image, main.to(torch.bfloat16))


def _adam(n, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda: torch.randn(n, generator=gen, device="cuda")  # noqa: E731
    return r() * 0.02, r() * 1e-3, (r() * 1e-3).square(), (r() * 1e-3).to(dtype)


@pytest.mark.parametrize("n", [1, 3, 4, 5, 1023, 4096, 100001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("offset,with_model", [(0, True), (1, True), (0, False)])
def test_adamw_step(gpu_device, n, dtype, offset, with_model):
    main, m, v, g = (torch.cat([x.new_full((offset,), 3.0), x, x.new_full((2,), 3.0)])[offset:offset + n] for x in _adam(n, dtype))
    image = torch.zeros(n + offset, dtype=torch.bfloat16, device="cuda")[offset:] if with_model else None
    lr, b1, b2, eps, wd, step = 1e-2, 0.9, 0.95, 1e-8, 0.1, 7
    gd = g.double()
    wm, wv = b1 * m.double() + (1 - b1) * gd, b2 * v.double() + (1 - b2) * gd * gd
    move = lr * (wm / (1 - b1 ** step)) / ((wv / (1 - b2 ** step)).sqrt() + eps)
    want = main.double() * (1 - lr * wd) - move
    size_m = (b1 * m.double()).abs() + ((1 - b1) * gd).abs()
    room = 2.0 ** -21 * (main.double().abs() + move.abs() + lr * size_m / (wv.sqrt() + eps) * 2)
    training.adamw_step(main, m, v, g, model=image, lr=lr, beta1=b1, beta2=b2, eps=eps, weight_decay=wd, step=step)
    assert (m.double() - wm).abs().le(2.0 ** -22 * size_m).all()
    assert (v.double() - wv).abs().le(2.0 ** -21 * wv).all()
    assert (main.double() - want).abs().le(room).all()
    if with_model:
        assert torch.equal(image, main.to(torch.bfloat16))
    for x in (main, m, v):
        whole = x._base if x._base is not None else x
        assert (whole[:offset] == 3.0).all() and (whole[offset + n:] == 3.0).all()


def test_adamw_first_step_and_values_that_are_not_finite(gpu_device):
    """The first step moves by lr whatever the gradient's size; NaN stays where it is."""
    g = torch.tensor([1e-3, -1e-6, 0.0, math.nan, math.inf, 5.0], device="cuda")
    main, m, v = torch.ones(6, device="cuda"), torch.zeros(6, device="cuda"), torch.zeros(6, device="cuda")
    training.adamw_step(main, m, v, g, lr=0.5, eps=0.0, step=1)
    assert (main[[0, 1, 5]] - torch.tensor([0.5, 1.5, 0.5], device="cuda")).abs().max() < 1e-6
    assert main[2:5].isnan().all() and not main[[0, 1, 5]].isnan().any()
    empty = torch.empty(0, device="cuda")
    training.adamw_step(empty, empty.clone(), empty.clone(), empty.clone(), lr=0.1, step=1)
