"""Matrices of one call that share memory: found exactly, against sets of their bytes (no GPU needed)."""

import random

import pytest

from elasticmegatron_amd.training._overlap import first_conflict, rows_of, share


def _bytes(m):
    return {m.base + i * m.stride + j for i in range(m.rows) for j in range(m.width)}


def _draw(rng, stride=None, **kw):
    width = rng.randint(1, 6)
    stride = rng.choice([width, width + rng.randint(0, 9)]) if stride is None else stride
    kw = dict(dict(what="main", index=0, written=True), **kw)
    return rows_of(rng.randint(0, 60), rng.randint(1, 7), max(stride, width), width, **kw)


@pytest.mark.parametrize("same_stride", [True, False])
def test_shared_bytes(same_stride):
    rng = random.Random(7)
    seen = set()
    for _ in range(5000):
        a = _draw(rng)
        b = _draw(rng, a.stride if same_stride else None)
        want = bool(_bytes(a) & _bytes(b))
        assert share(a, b) == share(b, a) == want, (a, b)
        seen.add((want, b.base < a.end and a.base < b.end))
    assert seen == {(True, True), (False, True), (False, False)}  # matrices between each other's rows among them


def test_conflicts_among_many():
    rng = random.Random(11)
    found = 0
    for _ in range(3000):
        many = [_draw(rng, what=what, index=i, written=what != "grad")
                for what in ("grad", "momentum_buffer", "main") for i in range(rng.randint(1, 3))]
        many = [m._replace(base=m.base + 200 * k, end=m.end + 200 * k) for m in many for k in [rng.randint(0, 6)]]
        allowed = lambda a, b: a.written != b.written and a.index == b.index and "momentum_buffer" not in (a.what, b.what)  # noqa: E731
        want = any((a.written or b.written) and not allowed(a, b) and _bytes(a) & _bytes(b)
                   for i, a in enumerate(many) for b in many[:i])
        got = first_conflict(many)
        assert (got is not None) == want
        if got:
            a, b = got
            assert _bytes(a) & _bytes(b) and (a.written or b.written)
            found += 1
    assert 300 < found < 2700


def test_many_that_are_only_read():
    """A broadcast gradient: thousands at one place, which no written matrix shares."""
    many = [rows_of(0, 4, 8, 8, "grad", i, False) for i in range(5000)]
    many += [rows_of(1000 + 100 * i, 4, 8, 8, "main", i, True) for i in range(5000)]
    assert first_conflict(many) is None
    assert first_conflict(many + [rows_of(1000, 1, 8, 8, "image", 1, True)]) is not None
