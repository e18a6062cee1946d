"""Gradients of attention in fp16 where rows differ in size: each row of grad_q and each of grad_k and grad_v has the bits
that its own terms leave it, whatever the other rows are."""

import math

import pytest
import torch

from tests.test_gpu_training_attention import FP16, _bounds, _close, _offsets, _run

pytestmark = pytest.mark.gpu

U, F = 2.0 ** -11, 2.0 ** -24  # half a step of fp16 and of 32 bits, relative
P = 2.0 ** -31                 # of a probability in forward, absolute: half fp16's smallest number, under its scale of 2^7 or more
P_BACK = 2.0 ** -40            # in grad_v: under a scale of 2^15
# Of d, relative to the largest of its sum: half of fp16's smallest number, 2^-25, under a scale that brings a number which is at
# most 2^9 times that largest to 2^15: 2^-31.  Twice that for the error of the largest itself.
D = 2.0 ** -30


def _formula(q, k, v, g, q_at, k_at, causal, scale):
    """out, gradients and what bounds their errors but for the last rounding, in 64 bits."""
    dim, share = q.shape[2], q.shape[1] // k.shape[1]
    q, k, v, g = (t.double() for t in (q, k, v, g))
    out, err = ([torch.zeros_like(t) for t in (q, q, k, v)] for _ in range(2))
    for lo, hi, at, end in zip(q_at, q_at[1:], k_at, k_at[1:]):
        n, m = hi - lo, end - at
        if not n or not m:
            continue
        i, j = torch.arange(n, device=q.device)[:, None], torch.arange(m, device=q.device)[None]
        see = (j <= i + m - n) if causal else torch.ones(n, m, dtype=torch.bool, device=q.device)
        full = see.any(1, keepdim=True)
        for kv in range(k.shape[1]):
            b, c = k[at:end, kv], v[at:end, kv]
            largest, sizes = q.new_zeros(m, 1), q.new_zeros(1, dim)  # of d of a key; of the queries
            for h in range(kv * share, (kv + 1) * share):
                a, d = q[lo:hi, h], g[lo:hi, h]
                s = torch.where(see, (a @ b.t()) * scale, -math.inf)
                lse = torch.where(full, s.logsumexp(1, keepdim=True), 0.0)
                p = torch.where(see, (s - lse).exp(), 0.0)
                # dim products in 32 bits, and a few roundings of the exponents; its own, and the sum's.
                e_s = F * ((dim + 8) * (a.abs() @ b.abs().t()) * scale + 8 * torch.where(see, s.abs(), 0.0) + 8 * lse.abs() + 8)
                e_s = e_s + (p * e_s).sum(1, keepdim=True) + F * 64
                e_p = p * (e_s + U)
                o = p @ c
                e_o = (e_p + P * see) @ c.abs() + F * m * (p @ c.abs())
                out[0][lo:hi, h], err[0][lo:hi, h] = o, e_o
                delta, dp = (d * o).sum(1, keepdim=True), d @ c.t()
                # From the output with what its rounding left over, which is rounded itself (at the least to half of 2^-24).
                e_delta = (d.abs() * (e_o + (U * U + F * dim) * o.abs() + 2.0 ** -25)).sum(1, keepdim=True)
                ds = p * (dp - delta)
                e_ds = p * (F * dim * (d.abs() @ c.abs().t()) + e_delta + F * (dp.abs() + delta.abs())) + ds.abs() * (e_s + U)
                row = D * (ds.abs() + e_ds).amax(1, keepdim=True) * see
                out[1][lo:hi, h] = scale * (ds @ b)
                err[1][lo:hi, h] = scale * ((e_ds + row) @ b.abs() + F * m * (ds.abs() @ b.abs()))
                out[2][at:end, kv] += scale * (ds.t() @ a)
                err[2][at:end, kv] += scale * (e_ds.t() @ a.abs() + F * n * share * (ds.abs().t() @ a.abs()))
                largest = torch.maximum(largest, (ds.abs() + e_ds).amax(0)[:, None])
                sizes = sizes + a.abs().sum(0, keepdim=True)
                out[3][at:end, kv] += p.t() @ d
                err[3][at:end, kv] += (e_p + P_BACK * see).t() @ d.abs() + F * n * share * (p.t() @ d.abs())
            err[2][at:end, kv] += scale * D * largest * sizes
    return out, err


def _operands(queries, keys, heads, kv_heads, dim, spare, seed=0):
    """Small queries and large keys: gradients of queries whose d is small are then far above fp16's smallest numbers."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda rows, h, s: torch.randn(rows, h, dim, generator=gen, device="cuda") * s  # noqa: E731
    rows, key_rows = sum(queries) + spare, sum(keys) + spare
    return make(rows, heads, 0.1), make(key_rows, kv_heads, 24.0), make(key_rows, kv_heads, 1.0), make(rows, heads, 1.0)


CASES = [
    # queries, keys, heads, kv_heads, dim, causal
    ([200], None, 2, 2, 64, True),
    ([300], None, 4, 2, 128, True),
    ([257], None, 3, 3, 100, False),
    ([130], None, 16, 1, 128, True),          # heads split over workgroups
    ([40, 7], [3000, 900], 4, 2, 64, True),   # keys split over workgroups
    ([5, 60, 128], [700, 60, 128], 2, 1, 72, True),
]


@pytest.mark.parametrize("queries,keys,heads,kv_heads,dim,causal", CASES)
@pytest.mark.parametrize("small", [2.0 ** -8, 2.0 ** -18])
def test_rows_of_different_sizes(gpu_device, queries, keys, heads, kv_heads, dim, causal, small):
    """Gradients of most rows, and of the last third of all rows, are 2^-12 or 2^-22 of the others'; one row of values is larger than the rest."""
    keys = keys or queries
    q, k, v, g = _operands(queries, keys, heads, kv_heads, dim, 0)
    rows = torch.arange(g.shape[0], device="cuda")
    large = (rows % 7 == 3) & (rows < 2 * g.shape[0] // 3)
    g *= torch.where(large, 16.0, small)[:, None, None]
    v[v.shape[0] // 2] *= 4
    q, k, v, g = (t.to(FP16) for t in (q, k, v, g))
    q_at, k_at = _bounds(queries), _bounds(keys)
    got = _run(q, k, v, g, offsets=_offsets(q_at), key_offsets=_offsets(k_at), causal=causal)
    want, err = _formula(q, k, v, g, q_at, k_at, causal, 1 / math.sqrt(dim))
    for t, w, e, what in zip(got, want, err, ("out", "grad_q", "grad_k", "grad_v")):
        assert t.isfinite().all()
        _close(t, w, e, what)
    assert all(torch.equal(a, b) for a, b in zip(_run(q, k, v, g, offsets=_offsets(q_at), key_offsets=_offsets(k_at), causal=causal), got))


@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (8, 2, 128), (3, 1, 100)])
@pytest.mark.parametrize("listed", [False, True])
def test_documents_do_not_touch_each_other(gpu_device, heads, kv_heads, dim, listed):
    """Large numbers, infinities and NaN in one document, and in rows of none, leave the others' bits as they are."""
    queries = [70, 90, 40] + ([1, 2] * 40 if listed else [])
    q, k, v, g = _operands(queries, queries, heads, kv_heads, dim, 9)
    q, k, v, g = (t.to(FP16) for t in (q, k, v, g * 2.0 ** -10))
    kw = dict(offsets=_offsets(_bounds(queries)))
    want = _run(q, k, v, g, **kw)
    keep = torch.ones(g.shape[0], dtype=torch.bool, device="cuda")
    keep[70:160] = False
    gen = torch.Generator(device="cuda").manual_seed(3)
    for fill in (60000.0, -60000.0, math.inf, math.nan):
        bad = [t.clone() for t in (q, k, v, g)]
        for t in bad:
            for part in (t[70:160], t[sum(queries):]):
                sign = torch.randint(0, 2, part.shape, generator=gen, device="cuda") * 2 - 1
                part.copy_(fill * sign)
        got = _run(*bad, **kw)
        assert all(torch.equal(a[keep], b[keep]) for a, b in zip(got, want)), fill
