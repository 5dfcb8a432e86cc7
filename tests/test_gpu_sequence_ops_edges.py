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


# ------------------------------------------------------------------ recurrence

# (outer, steps, inner) for every way rows reach the kernel, in clusters and in
# blocks alone: tensor copies, a lane's own copies, loads of two bytes (float16)
WAYS = [("float32", (1, 3000, 256)), ("float32", (1, 3000, 33)), ("float16", (1, 3000, 128)), ("float16", (1, 3000, 34)),
        ("float16", (1, 3000, 33)), ("float64", (1, 1500, 64)), ("float64", (1, 1500, 33)), ("float32", (230, 250, 32)),
        ("float16", (230, 250, 64)), ("float16", (230, 250, 33)), ("float16", (230, 250, 62)), ("float64", (230, 250, 32))]


@pytest.mark.parametrize("dt,shape", WAYS)
@pytest.mark.parametrize("decay", [16.0, 1024.0, 2.0 ** 15])
def test_recurrence_decays_past_the_range(cp, dt, shape, decay):
    """Decays whose product overflows within a span of steps or over the spans of
    a block (up to 112 steps, 56 for float64): a state of zero stays zero, from
    either end, and what is finite step by step is finite.  All values are
    exact: sums of powers of two, rounded to the arrays' dtype once."""
    last = {16.0: 4, 1024.0: 2, 2.0 ** 15: 2}[decay]
    if dt == "float64":
        decay, last = decay ** 12, 1  # 2^48, 2^120, 2^180 a step
    a = cp.full(shape, decay, dtype=dt)
    x = np.zeros(shape, dt)
    x[:, -last:, ::2] = 1
    want = np.zeros(shape)
    for k in range(last):
        want[:, shape[1] - last + k, ::2] = sum(decay ** j for j in range(k + 1))
    st = cp.empty((shape[0], shape[2]), dtype="float64" if dt == "float64" else "float32")
    h = cp.linear_recurrence(a, cp.array(x), state_out=st)
    np.testing.assert_array_equal(h.get(), want.astype(dt))
    np.testing.assert_array_equal(st.get(), want[:, -1])
    # backward: gradients of the first steps alone, seen from the last step on
    back, grad = want[:, ::-1], np.ascontiguousarray(x[:, ::-1])
    ones = np.ones(shape, dt)
    da, dx, _ = cp.linear_recurrence_grad(a, None, cp.array(ones), cp.array(grad))
    np.testing.assert_array_equal(dx.get(), back.astype(dt))
    back = back.copy()
    back[:, 0] = 0  # h before the first step is zero
    np.testing.assert_array_equal(da.get(), back.astype(dt))


def grow_as_computed(a, gated):
    """K of the recurrence's bound for float16 gates, from the instructions that
    make them: exp(-|z|) by ex2.approx within 2^-22.5 (2.8 u), its argument
    |z| log2(e) rounded once and by a constant rounded to 0.2 u (1.2 |z| u);
    1 + e u; rcp.approx 2^-23 (2 u); e r u: below 7 + 1.2 |z|.  The product
    (1 - f) x, the fma and the decays' product add u each, and a state passed
    on through three such products: 16 + 1.2 |z|.  |z| counts up to 104
    (exp(-104) is zero)."""
    assert a.dtype == np.float16 and gated
    return 16 + 1.2 * np.minimum(np.abs(a.astype(np.float64)), 104)


@pytest.mark.parametrize("spread", [1.0, 6.0, 20.0])
@pytest.mark.parametrize("shape", [(3, 1, 40), (2, 30, 33), (1, 700, 128), (2, 300, 66), (2, 130, 65), (230, 130, 64)])
def test_recurrence_float16_gates(cp, monkeypatch, shape, spread):
    import test_gpu_sequence_ops as base
    monkeypatch.setattr(base, "grow", grow_as_computed)
    rng = np.random.default_rng(int(spread) + shape[1])
    a = rng.normal(0, spread, shape).astype(np.float16)
    x, g = (rng.standard_normal(shape).astype(np.float16) for _ in "xg")
    h0 = rng.standard_normal((shape[0], shape[2])).astype(np.float32)
    hs, es, last, el = base.recurrence(a, x, h0, True)
    st = cp.empty(h0.shape, dtype="float32")
    h = cp.linear_recurrence(cp.array(a), cp.array(x), cp.array(h0), gated=True, state_out=st)
    close(h.get(), hs, es * UNIT["float16"], "float16")
    close(st.get(), last, el * UNIT["float16"], "float32")
    da, dx, dh0, ea, ex, e0 = base.recurrence_grad(a, x, h.get(), g, h0, None, True)
    got = cp.linear_recurrence_grad(cp.array(a), cp.array(x), h, cp.array(g), cp.array(h0), gated=True)
    close(got[0].get(), da, ea * UNIT["float16"], "float16")
    close(got[1].get(), dx, ex * UNIT["float16"], "float16")
    close(got[2].get(), dh0, e0 * UNIT["float16"], "float32")


MASKED = WAYS + [("float32", (3, 5, 40)), ("float16", (3, 14, 33)), ("float16", (3, 16, 64)), ("float64", (2, 9, 7)),
                 ("float32", (2, 300, 96)), ("float16", (1, 9000, 64)), ("float32", (100, 400, 64))]


def masked_inputs(dt, shape, seed):
    """Gates of ordinary sequences, about one step in nine padded (+inf or the
    type's highest value), and every 70 steps or so a new sequence (-inf or the
    type's lowest value)."""
    rng = np.random.default_rng(seed)
    big = np.finfo(dt).max
    z = rng.normal(0, 2, shape).astype(dt)
    steps = shape[1]
    pad, new = np.zeros(steps, bool), np.zeros(steps, bool)
    pad[rng.random(steps) < 0.11] = True
    new[rng.random(steps) < 0.014] = True
    new[steps // 2], pad[0], pad[-1] = True, True, steps > 9
    pad[new] = False
    z[:, pad], z[:, new] = np.inf, -np.inf
    z[:, pad, ::3], z[:, new, ::3] = big, -big
    sdt = "float64" if dt == "float64" else "float32"
    return (rng, z, rng.standard_normal(shape).astype(dt), rng.standard_normal((shape[0], shape[2])).astype(sdt),
            rng.standard_normal(shape).astype(dt), pad, new, sdt)


@pytest.mark.parametrize("dt,shape", MASKED)
def test_recurrence_not_finite_to_the_end_of_its_chain(cp, dt, shape):
    """An infinity or NaN in x, in a padded step too, or in the first state:
    nothing finite comes after it in its chain, through padded steps and new
    sequences (0 * inf is NaN); before it, and in other chains, every bit is
    as it was."""
    rng, z, x, h0, g, pad, new, sdt = masked_inputs(dt, shape, 1)

    def run(x, h0):
        st = cp.empty(h0.shape, dtype=sdt)
        h = cp.linear_recurrence(cp.array(z), cp.array(x), cp.array(h0), gated=True, state_out=st)
        return h.get(), st.get()
    clean, last = run(x, h0)
    assert np.isfinite(clean).all() and np.isfinite(last).all()
    bad, bh0, want = x.copy(), h0.copy(), np.zeros(shape, bool)
    at = {1: shape[1] // 3, 2: shape[1] - 1, 3: 0, 4: int(np.flatnonzero(pad)[-1])}
    for k, v in ((1, np.inf), (2, np.nan), (3, -np.inf), (4, np.nan)):
        bad[:, at[k], k::7] = v
        want[:, at[k]:, k::7] = True
    bh0[:, 5::7] = np.inf
    want[:, :, 5::7] = True
    h, st = run(bad, bh0)
    np.testing.assert_array_equal(~np.isfinite(h), want)
    np.testing.assert_array_equal(~np.isfinite(st), want[:, -1])
    np.testing.assert_array_equal(h[~want], clean[~want])
    np.testing.assert_array_equal(st[~want[:, -1]], last[~want[:, -1]])


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


@pytest.mark.parametrize("idt", ["int32", "int64"])
@pytest.mark.parametrize("dt", ["float16", "float32", "float64"])
def test_embedding_grad_more_tokens_than_a_cluster_sorts(cp, dt, idt):
    """65536 tokens (the cluster's last), one more, and ordinary batches: tables
    of one row to a million, frequent ids, padding, equal bits of equal calls."""
    for i, (n, rows, width) in enumerate([(65536, 5000, 24), (65537, 5000, 24), (65543, 1, 3), (131072, 50257, 16),
                                          (70001, 1000003, 9), (200003, 300, 40), (100000, 1 << 18, 4)]):
        rng = np.random.default_rng(i)
        ids = np.minimum(np.exp(rng.random(n) * np.log(rows + 1)) - 1, rows - 1).astype(idt)
        g = rng.standard_normal((n, width), dtype=np.float32).astype(dt)
        want, err = table_grad(ids, g, rows, 0.3)
        pad = int(ids[5]) if i % 2 else None
        if pad is not None:
            want[pad] = 0
        I, G = cp.array(ids), cp.array(g)
        got = cp.embedding_grad(I, G, rows, 0.3, padding_idx=pad, out=cp.full((rows, width), 5, dtype=dt)).get()
        close(got, want, err * UNIT[dt], dt)
        if pad is not None:
            assert not got[pad].any()
        np.testing.assert_array_equal(cp.embedding_grad(I, G, rows, 0.3, padding_idx=pad).get(), got)
    cp.synchronize()


@pytest.mark.parametrize("kind", ["one", "two", "all", "bad"])
def test_embedding_grad_many_tokens_of_a_kind(cp, kind):
    """One id, two in turn, each once, and ids out of range among others (which
    add nothing and are reported)."""
    n, rows, width = 90001, 120000, 20
    rng = np.random.default_rng(4)
    ids = {"one": np.full(n, 77), "two": np.arange(n) % 2 * (rows - 1), "all": rng.permutation(rows)[:n],
           "bad": rng.integers(0, rows, n)}[kind]
    g = rng.standard_normal((n, width), dtype=np.float32)
    sent, keep = ids.copy(), np.ones(n, bool)
    if kind == "bad":
        keep = rng.random(n) < 0.9
        sent[~keep] = np.resize([-1, rows, 2 ** 40], int((~keep).sum()))
    want, err = table_grad(ids[keep], g[keep], rows, 1.0)
    got = cp.embedding_grad(cp.array(sent), cp.array(g), rows).get()
    close(got, want, err * UNIT["float32"], "float32")
    if kind == "bad":
        with pytest.raises(RuntimeError, match="5"):
            cp.synchronize()
    cp.synchronize()


def test_embedding_grad_many_tokens_large_table(cp):
    rng = np.random.default_rng(2)
    check_table_grad(cp, rng.integers(0, 50257, 131072), rng.standard_normal((131072, 100), dtype=np.float32)
                     .astype(np.float16), 50257)
    check_table_grad(cp, np.resize(np.arange(0, 400009, 32), 70000), rng.standard_normal((70000, 50), dtype=np.float32),
                     400009)


@pytest.mark.parametrize("idt", ["int32", "int64"])
@pytest.mark.parametrize("n", [1, 3, 3000, 70000])
def test_bad_ids_of_empty_tables_are_reported(cp, n, idt):
    """Without a row every id is out of range, and without a column those that
    are beyond the rows, although there is nothing to write."""
    ids = cp.zeros((n,), dtype=idt)
    calls = [(True, lambda: cp.embedding(cp.zeros((0, 4), dtype="float32"), ids)),
             (True, lambda: cp.embedding_grad(ids, cp.ones((n, 4), dtype="float32"), 0)),
             (True, lambda: cp.embedding(cp.zeros((0, 0), dtype="float32"), ids)),
             (True, lambda: cp.embedding_grad(ids, cp.ones((n, 0), dtype="float32"), 0)),
             (False, lambda: cp.embedding(cp.zeros((2, 0), dtype="float32"), ids)),
             (False, lambda: cp.embedding_grad(ids, cp.ones((n, 0), dtype="float32"), 2)),
             (True, lambda: cp.embedding(cp.zeros((2, 0), dtype="float32"), ids + 2)),
             (True, lambda: cp.embedding_grad(ids - 1, cp.ones((n, 0), dtype="float32"), 2))]
    for k, (bad, call) in enumerate(calls):
        assert call().size in (0, 4 * n), k
        if bad:
            with pytest.raises(RuntimeError, match="5"):
                cp.synchronize()
        cp.synchronize()


# ------------------------------------------------------------------ clipping

@pytest.mark.parametrize("limit", [1.0, 1e-3, 1e-7, 1e-10, 1e-30, 1e-44])
def test_clip_by_a_coefficient_below_float32(cp, limit):
    """Huge gradients and a small limit: the coefficient passes float32's range
    (subnormal from 1e-38 on), the clipped arrays need not.  The norm's sum in
    float64 is within 2^-50 of 4100 terms; its root, the quotient, the
    coefficient's rounding to 32 bits and the product's: 2 u and the result's
    rounding."""
    rng = np.random.default_rng(6)
    arrays = [(rng.uniform(-3e38, 3e38, 4099)).astype(np.float32), np.float32([1e38, -1e25, 1.0]),
              np.float16([60000, -3, 1e-7])]
    norm = np.sqrt(sum((a.astype(np.float64) ** 2).sum() for a in arrays))
    A = [cp.array(a) for a in arrays]
    for out in (None, A):
        res, _ = cp.clip_by_global_norm(A, limit, out=out)
        for r, a in zip(res, arrays):
            want = a.astype(np.float64) * (limit / norm)
            close(r.get(), want, 2 * UNIT["float32"] * np.abs(want), str(a.dtype))


# ------------------------------------------------------------------ threads

def test_threads_with_launches_of_different_sizes(cp):
    """Calls from several threads at once whose launches of one kernel need
    different amounts of shared memory (steps below, at and above the spans of
    a block and of its ring; tokens of one to eight keys a thread)."""
    import threading

    from macmetalpy_b200 import _cuda_backend as cb

    rng = np.random.default_rng(9)
    work = []
    for steps, tokens in ((40, 2000), (200, 20000), (3000, 60000), (90, 9000)):
        a = rng.normal(2, 2, (2, steps, 96)).astype(np.float32)
        work.append((a, rng.standard_normal(a.shape, dtype=np.float32), rng.integers(0, 3000, tokens),
                     rng.standard_normal((tokens, 24), dtype=np.float32)))

    def one(w, to, times):
        a, x, ids, g = w
        cb.check(cb.lib.mmp_init(cb.CudaBackend().device))  # the device of a new thread
        A, X, I, G = cp.array(a), cp.array(x), cp.array(ids), cp.array(g)
        for _ in range(times):
            h = cp.linear_recurrence(A, X, gated=True)
            da, dx, _ = cp.linear_recurrence_grad(A, X, h, X, gated=True)
            to.append([r.get() for r in (h, da, dx, cp.embedding_grad(I, G, 3000))])

    alone, together, failed = [[] for _ in work], [[] for _ in work], []

    def guarded(w, to):
        try:
            one(w, to, 40)
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    for w, to in zip(work, alone):
        one(w, to, 1)
    threads = [threading.Thread(target=guarded, args=(w, to)) for w, to in zip(work, together)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for p, q in zip(alone, together):
        assert len(q) == 40
        for r in q:
            for got, want in zip(r, p[0]):
                np.testing.assert_array_equal(got, want)


# ------------------------------------------------------------------ captured

CAPTURE = """
import sys
sys.path.insert(0, {repo!r})
import ctypes
import numpy as np
import torch
import macmetalpy_b200 as cp
from macmetalpy_b200 import _cuda_backend as cb
cp.synchronize()
stream = torch.cuda.Stream()
cb.check(cb.lib.mmp_set_stream(ctypes.c_void_p(stream.cuda_stream)))
rng = np.random.default_rng(0)
n, width = 70000, 6
tables = [200, 5000, 50257 * 30]
ids = [cp.array(rng.integers(0, rows, n)) for rows in tables]
g = cp.array(rng.standard_normal((n, width)).astype("float32"))
out = [cp.empty((rows, width), dtype="float32") for rows in tables]
def step():
    for i, rows, o in zip(ids, tables, out):
        cp.embedding_grad(i, g, rows, 2.0, out=o)
def results():
    return [o.get() for o in out]
graphs = []
for _ in range(2):  # the first calls of this process: nothing is set up before the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    graphs.append(graph)
for k in range(6):
    for i, rows in zip(ids, tables):
        i.set(rng.integers(0, rows, n))
    g.set(rng.standard_normal((n, width)).astype("float32"))
    cp.cumsum(cp.ones(((k + 1) << 22,), dtype="float32"))  # grows and moves the library's own scan state
    step(); want = results()
    for o in out:
        o.fill(7)
    cp.synchronize()
    for _ in range(1 + k % 2):
        with torch.cuda.stream(stream):
            graphs[k % 2].replay()
    torch.cuda.synchronize()
    for p, q in zip(want, results()):
        np.testing.assert_array_equal(p, q)
    cp.synchronize()
print("captured")
"""


def test_many_tokens_captured_and_replayed(cp):
    """The gradient above 65536 tokens in two graphs, replayed in turn and twice
    in a row, sort keys of one pass and of several, other scans in between (a
    process of its own: the library keeps the stream it is given)."""
    import os
    import subprocess
    import sys

    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    p = subprocess.run([sys.executable, "-c", CAPTURE.format(repo=repo)], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and "captured" in p.stdout, p.stdout + p.stderr
