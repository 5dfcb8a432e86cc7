"""More of linear_recurrence, embedding, global norm and their gradients:
borders of tables, lists of tokens, gates and sizes that a launch's shares
meet at.  Tolerances as derived in test_gpu_sequence_ops.py."""

import numpy as np
import pytest
from test_gpu_sequence_ops import UNIT, close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cp():
    import macmetalpy_b200 as cp
    return cp


# ------------------------------------------------------------------ embedding gradient

def table_grad(ids, g, rows, scale):
    """(gradient, bound over u) in float64: sums of the tokens sorted by id.
    m additions and the scale's two roundings: (m + 2) u of the magnitudes."""
    order = np.argsort(ids, kind="stable")
    s = ids[order]
    first = np.flatnonzero(np.concatenate([[True], s[1:] != s[:-1]]))
    g = g[order].astype(np.float64)
    out, err = np.zeros((rows, g.shape[1])), np.zeros((rows, g.shape[1]))
    out[s[first]] = np.add.reduceat(g, first, 0) * scale
    count = np.diff(np.concatenate([first, [len(s)]]))
    err[s[first]] = (count[:, None] + 2) * np.add.reduceat(np.abs(g), first, 0) * abs(scale)
    return out, err


def check_table_grad(cp, ids, g, rows, calls=2):
    dt = str(g.dtype)
    want, err = table_grad(ids, g, rows, 1.7)
    I, G = cp.array(ids), cp.array(g)
    first = None
    for _ in range(calls):
        got = cp.embedding_grad(I, G, rows, 1.7, out=cp.full((rows, g.shape[1]), 5, dtype=dt)).get()
        close(got, want, err * UNIT[dt], dt)
        if first is None:
            first = got
        np.testing.assert_array_equal(got, first)  # equal calls, equal bits
    cp.synchronize()


# tables of 32 MB and more whose rows do not divide 32 MB
TABLES = [(50257, 768, "float16"), (1500000, 6, "float32"), (50257, 1000, "float16"), (100000, 300, "float32"),
          (131072, 100, "float32"), (40009, 333, "float64")]


@pytest.mark.parametrize("kind", ["uniform", "multiples"])
@pytest.mark.parametrize("rows,width,dt", TABLES)
def test_embedding_grad_large_tables(cp, rows, width, dt, kind):
    """The whole table, tokens anywhere, and at every word's edge of the bitmap
    of rows (all of them, where there are tokens enough)."""
    n = 16384
    rng = np.random.default_rng(rows + width)
    ids = rng.integers(0, rows, n)
    if kind == "multiples":
        ids = np.resize(np.arange(0, rows, 32), n) if rows <= 32 * n else ids // 32 * 32
    g = rng.standard_normal((n, width), dtype=np.float32).astype(dt)
    check_table_grad(cp, ids, g, rows, calls=3)
