"""Which matrices in memory share an element with another one.

A matrix is its rows: ``rows`` runs of ``width`` bytes, ``stride`` bytes from one's start to the next one's
(``stride >= width``), the first at ``base``.  Matrices may lie between each other's rows.
"""

from __future__ import annotations

from typing import Iterable, NamedTuple, Optional, Tuple


class Rows(NamedTuple):
    base: int
    end: int  # past the last row
    rows: int
    stride: int
    width: int
    what: str     # the argument that it belongs to
    index: int    # its place there
    written: bool


def rows_of(base: int, rows: int, stride: int, width: int, what: str, index: int, written: bool) -> Rows:
    return Rows(base, base + (rows - 1) * stride + width, rows, stride, width, what, index, written)


def share(a: Rows, b: Rows) -> bool:
    """Whether a byte is in both."""
    if a.base > b.base:
        a, b = b, a
    if b.base >= a.end:
        return False
    if a.stride == b.stride:
        # Row i of b begins `at` bytes into row `first + i` of a, or into the gap after it.
        first, at = divmod(b.base - a.base, a.stride)
        return (at < a.width and first < a.rows) or (at + b.width > a.stride and first + 1 < a.rows)
    i = j = 0
    while i < a.rows and j < b.rows:
        x, y = a.base + i * a.stride, b.base + j * b.stride
        if x + a.width <= y:
            i += 1
        elif y + b.width <= x:
            j += 1
        else:
            return True
    return False


def first_conflict(matrices: Iterable[Rows]) -> Optional[Tuple[Rows, Rows]]:
    """Two matrices that share memory of which one is written, or None.  A matrix that is only read may share
    that of the written one of its own index, unless it is the momentum's: it is read before that is written."""
    ordered = sorted(matrices)
    end = -1
    for m in ordered:
        if m.base < end:
            break
        end = m.end
    else:
        return None  # one after the other, as they nearly always lie
    written, read = [], []
    for m in ordered:
        written = [x for x in written if x.end > m.base]
        read = [x for x in read if x.end > m.base] if m.written else read
        for x in (*written, *read) if m.written else written:
            if x.written != m.written and x.index == m.index and "momentum_buffer" not in (x.what, m.what):
                continue
            if share(x, m):
                return x, m
        (written if m.written else read).append(m)
    return None
