"""Host-only checks of how the tiles of the gated product and of its gradients
are dealt out to CTA pairs, through pax_selftest_feed_forward_items: every
column of every row block is computed exactly once.  No GPU needed."""
from __future__ import annotations

import ctypes
import random

import numpy as np
import pytest

import pax_b200


def items(which, M, D, F, units, most=1 << 17):
    """(tile width 1 or 2, rows of: pair, kind, row block, first column, columns)"""
    f = pax_b200.lib.pax_selftest_feed_forward_items
    f.argtypes = [ctypes.c_int] + [ctypes.c_longlong] * 3 + [ctypes.c_int, ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_int),
                                                             ctypes.c_int]
    f.restype = ctypes.c_int
    width, buf = ctypes.c_int(), (ctypes.c_int * (5 * most))()
    n = f(which, M, D, F, units, ctypes.byref(width), buf, most)
    return (width.value, np.frombuffer(buf, dtype=np.intc)[: 5 * n].reshape(n, 5)) if n >= 0 else (n, None)


def check(blocks, cols, part, slack):
    """Row blocks 0..blocks-1 have columns [0, cols) once each; tiles may reach up to `slack` columns beyond."""
    assert len(part) and part[:, 0].max() < blocks and (part[:, 2] > 0).all()
    unit = np.gcd.reduce(np.concatenate([part[:, 1], part[:, 2]]))
    times = np.zeros((blocks, -(-cols // unit) + slack // unit + 1), dtype=int)
    for mb, c, n in part:
        assert c >= 0 and c + n <= times.shape[1] * unit
        times[mb, c // unit: (c + n) // unit] += 1
    assert (times[:, : -(-cols // unit)] == 1).all() and (times <= 1).all()


def check_shape(which, M, D, F, units):
    w, it = items(which, M, D, F, units)
    assert w in (1, 2) and it[:, 0].min() >= 0 and it[:, 0].max() < units
    if which == 0:
        check(-(-M // 256), F, it[:, 2:], 128 * w)
        return w, len(it)
    x, g = it[it[:, 1] == 0][:, 2:], it[it[:, 1] == 1][:, 2:]
    check(-(-M // 256), D, x, 256 * w)
    edge = -(-F // (256 * w)) * 256 * w
    check(-(-D // 256), 2 * edge, g, 0)
    return w, len(it)


SHAPES = [(777, 1544, 4104), (4096, 4096, 11264), (2051, 2056, 5480), (4096, 4096, 8192), (130, 768, 2048), (1, 1, 1), (257, 255, 257),
          (1935, 3032, 320), (20000, 64, 64), (64, 20000, 72)]


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("units", [74, 66, 1])
@pytest.mark.parametrize("shape", SHAPES)
def test_every_column_once(which, shape, units):
    check_shape(which, *shape, units)


@pytest.mark.parametrize("which", [0, 1])
def test_every_column_once_at_random(which):
    rng = random.Random(11 + which)
    widths = set()
    for _ in range(250):
        M, D, F = (int(2 ** rng.uniform(0, 13.5)) for _ in range(3))
        widths.add(check_shape(which, M, D, F, rng.choice([74, 72, 37, 148]))[0])
    assert widths == {1, 2}


def test_bad_arguments():
    assert items(2, 8, 8, 8, 74)[0] == -1 and items(0, 0, 8, 8, 74)[0] == -1 and items(1, 8, 8, 8, 0)[0] == -1
    assert items(0, 8192, 64, 8192, 74, most=3)[0] == -1
