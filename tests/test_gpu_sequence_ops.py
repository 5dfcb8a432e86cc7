"""linear_recurrence, embedding, global norm and their gradients against plain
float64 implementations, with tolerances derived from the arithmetic.

Notation: u is the unit roundoff of the type that states and sums are held in
(2^-24 for float16 and float32 arrays, 2^-53 for float64), r that of the
array's own type (half a step relative to the value), s half its smallest
subnormal step (an absolute rounding error near zero).

Recurrence.  sigmoid: exp is within 2 ulp (4 u), the add and the division u
each, so f and 1 - f are within 10 u; with the product (1 - f) x, the fma and
the product of decays over a span (u a step), each step adds at most K = 16 u of
its terms' magnitudes, and what earlier steps left decays with f:
E_t = |f| E_{t-1} + K u (|f| H_{t-1} + |u_t|), H the recurrence of magnitudes.
float16 gates take CUDA's __expf, within 2 + 1.173 |z| ulp by its documented
bound: K = 16 + 2.4 |z|, where |z| counts up to 104 (exp(-104) is zero).
Sums of m terms in any order are within m u of the sum of magnitudes."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

UNIT = {"float16": 2.0 ** -24, "float32": 2.0 ** -24, "float64": 2.0 ** -53}
HALF = {"float16": 2.0 ** -11, "float32": 2.0 ** -24, "float64": 2.0 ** -53}
TINY = {"float16": 2.0 ** -25, "float32": 2.0 ** -150, "float64": 0.0}
DTYPES = ["float16", "float32", "float64"]


@pytest.fixture(scope="module")
def cp():
    import macmetalpy_b200 as cp
    return cp


def close(got, want, err, dt):
    """|got - want| <= err + the rounding of `want` to `dt`, NaN and infinities alike."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    fin = np.isfinite(want)
    np.testing.assert_array_equal(got[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)])
    tol = np.broadcast_to(err, want.shape)[fin] + HALF[dt] * np.abs(want[fin]) + TINY[dt]
    bad = np.abs(got[fin] - want[fin]) > tol
    assert not bad.any(), (int(bad.sum()), float(np.max(np.abs(got[fin] - want[fin]) - tol)))


def gates(a, gated):
    a = a.astype(np.float64)
    with np.errstate(over="ignore"):
        return (1 / (1 + np.exp(-a)), 1 / (1 + np.exp(a))) if gated else (a, np.ones_like(a))


def grow(a, gated):
    """K, per element."""
    return 16 + (2.4 * np.minimum(np.abs(a.astype(np.float64)), 104) if gated and a.dtype == np.float16 else np.zeros(a.shape))


def recurrence(a, x, h0, gated):
    """(h, error bound over u, last state) in float64, steps on axis 1 of (outer, steps, inner)."""
    f, rest = gates(a, gated)
    k = grow(a, gated)
    uu = rest * x.astype(np.float64)
    h = np.zeros(x[:, 0].shape if x.shape[1] else (x.shape[0], x.shape[2])) if h0 is None else h0.astype(np.float64)
    mag, e = np.abs(h), np.zeros_like(h)
    hs, es = np.empty(x.shape), np.empty(x.shape)
    for t in range(x.shape[1]):
        part = np.abs(f[:, t]) * mag + np.abs(uu[:, t])
        e = np.abs(f[:, t]) * e + k[:, t] * part
        h = f[:, t] * h + uu[:, t]
        mag = part
        hs[:, t], es[:, t] = h, e
    return hs, es, h, e


def recurrence_grad(a, x, h, g, h0, gs, gated):
    f, rest = gates(a, gated)
    kk = grow(a, gated)
    x, h, g = (v.astype(np.float64) for v in (x, h, g))
    n = x.shape[1]
    first = np.zeros((x.shape[0], x.shape[2])) if h0 is None else h0.astype(np.float64)
    c = np.zeros_like(first) if gs is None else gs.astype(np.float64)
    mag, e = np.abs(c), np.zeros_like(c)
    da, dx, ea, ex = (np.empty(x.shape) for _ in range(4))
    for t in range(n - 1, -1, -1):
        gt, gm = g[:, t] + c, np.abs(g[:, t]) + mag
        hp = h[:, t - 1] if t else first
        k = f[:, t] * rest[:, t] if gated else np.ones_like(gt)
        d = hp - x[:, t] if gated else hp
        dm = np.abs(hp) + np.abs(x[:, t]) if gated else np.abs(hp)
        da[:, t], dx[:, t] = gt * d * k, gt * rest[:, t]
        ea[:, t] = (e + 2 * kk[:, t] * gm) * dm * np.abs(k)
        ex[:, t] = (e + kk[:, t] * gm) * np.abs(rest[:, t])
        c = f[:, t] * gt
        e = np.abs(f[:, t]) * (e + kk[:, t] * gm)
        mag = np.abs(f[:, t]) * gm
    return da, dx, c, ea, ex, e


def rec_inputs(shape, dt, gated, seed, h0=True):
    rng = np.random.default_rng(seed)
    a = rng.normal(2.0, 2.0, shape) if gated else 1 / (1 + np.exp(-rng.normal(2.0, 2.0, shape)))
    st = (shape[0], shape[2])
    sdt = np.float64 if dt == "float64" else np.float32
    return (a.astype(dt), rng.standard_normal(shape).astype(dt),
            rng.standard_normal(st).astype(sdt) if h0 else None,
            rng.standard_normal(shape).astype(dt), rng.standard_normal(st).astype(sdt) if h0 else None)


# sizes round the edges of warps, vectors, tiles and time spans, and a few long ones
SHAPES = [(2, 300, 66), (1, 3000, 130), (200, 290, 96), (1, 1, 1), (1, 1, 2), (3, 2, 1), (2, 3, 5), (1, 16, 31), (2, 17, 32), (1, 31, 33), (2, 32, 64), (1, 33, 65),
          (3, 63, 100), (2, 64, 127), (1, 127, 128), (1, 129, 130), (5, 255, 7), (1, 257, 256), (40, 1, 96),
          (4, 511, 34), (2, 1025, 48), (1, 2047, 66), (1, 4099, 3), (70, 130, 2), (1, 9000, 40), (300, 5, 257)]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dt", DTYPES)
def test_recurrence(cp, dt, gated):
    for i, shape in enumerate(SHAPES):
        a, x, h0, _, _ = rec_inputs(shape, dt, gated, i, h0=i % 3 != 0)
        hs, es, last, el = recurrence(a, x, h0, gated)
        state = cp.empty((shape[0], shape[2]), dtype="float64" if dt == "float64" else "float32")
        h = cp.linear_recurrence(cp.array(a), cp.array(x), None if h0 is None else cp.array(h0), gated=gated,
                                 state_out=state)
        assert h.dtype == np.dtype(dt) and h.shape == shape
        close(h.get(), hs, es * UNIT[dt], dt)
        close(state.get(), last, el * UNIT[dt], str(state.dtype))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dt", DTYPES)
def test_recurrence_grad(cp, dt, gated):
    for i, shape in enumerate(SHAPES):
        a, x, h0, g, gs = rec_inputs(shape, dt, gated, 100 + i, h0=i % 3 != 0)
        h = recurrence(a, x, h0, gated)[0].astype(dt)
        da, dx, dh0, ea, ex, e0 = recurrence_grad(a, x, h, g, h0, gs, gated)
        got = cp.linear_recurrence_grad(cp.array(a), cp.array(x) if gated else None, cp.array(h), cp.array(g),
                                        None if h0 is None else cp.array(h0), gated=gated,
                                        grad_state=None if gs is None else cp.array(gs))
        close(got[0].get(), da, ea * UNIT[dt], dt)
        close(got[1].get(), dx, ex * UNIT[dt], dt)
        if h0 is None:
            assert got[2] is None
        else:
            close(got[2].get(), dh0, e0 * UNIT[dt], "float64" if dt == "float64" else "float32")


@pytest.mark.parametrize("gated", [False, True])
def test_recurrence_grad_by_differences(cp, gated):
    """The gradient of L = sum(w h) + sum(v state) against central differences
    of the float64 forward pass.  Step 1e-5: the third-order term is below
    1e-10 of values of order 1, the rounding 1e-16 / 1e-5 a value: 1e-8 covers
    sums over 24 steps of order 1."""
    shape = (2, 24, 3)
    a, x, h0, w, v = rec_inputs(shape, "float64", gated, 5)

    def loss(a, x, h0):
        st = cp.empty(h0.shape, dtype="float64")
        h = cp.linear_recurrence(cp.array(a), cp.array(x), cp.array(h0), gated=gated, state_out=st).get()
        return float((h * w).sum() + (st.get() * v).sum())

    h = cp.linear_recurrence(cp.array(a), cp.array(x), cp.array(h0), gated=gated)
    got = [r.get() for r in cp.linear_recurrence_grad(cp.array(a), cp.array(x), h, cp.array(w), cp.array(h0),
                                                      gated=gated, grad_state=cp.array(v))]
    rng = np.random.default_rng(0)
    for k, val in enumerate((a, x, h0)):
        for _ in range(12):
            at = tuple(rng.integers(0, n) for n in val.shape)
            args = [a, x, h0]
            hi, lo = val.copy(), val.copy()
            hi[at] += 1e-5
            lo[at] -= 1e-5
            args[k] = hi
            up = loss(*args)
            args[k] = lo
            down = loss(*args)
            assert abs((up - down) / 2e-5 - got[k][at]) <= 1e-8 * 10, (k, at)


@pytest.mark.parametrize("dt", DTYPES)
def test_recurrence_gate_limits(cp, dt):
    """Gates of +-inf, of the type's lowest and highest value: the state kept
    or replaced exactly; no NaN; whole rows of one kind."""
    big = float(np.finfo(dt).max)
    kinds = np.array([np.inf, -np.inf, big, -big, 0.0, np.inf, np.inf, -np.inf], np.float64)
    rng = np.random.default_rng(1)
    steps, width = 67, 40
    a = kinds[rng.integers(0, len(kinds), (3, steps, width))].astype(dt)
    a[0] = np.inf       # every step padded
    a[1] = -big         # every step a start
    x = rng.standard_normal((3, steps, width)).astype(dt)
    h0 = rng.standard_normal((3, width)).astype("float64" if dt == "float64" else "float32")
    h = cp.linear_recurrence(cp.array(a), cp.array(x), cp.array(h0), gated=True)
    hs, es, _, _ = recurrence(a, x, h0, True)
    close(h.get(), hs, es * UNIT[dt], dt)
    np.testing.assert_array_equal(h.get()[0], np.broadcast_to(h0[0].astype(dt), (steps, width)))
    np.testing.assert_array_equal(h.get()[1], x[1])
    g = rng.standard_normal((3, steps, width)).astype(dt)
    da, dx, dh0, ea, ex, e0 = recurrence_grad(a, x, hs.astype(dt), g, h0, None, True)
    got = cp.linear_recurrence_grad(cp.array(a), cp.array(x), cp.array(hs.astype(dt)), cp.array(g), cp.array(h0),
                                    gated=True)
    close(got[0].get(), da, ea * UNIT[dt], dt)
    close(got[1].get(), dx, ex * UNIT[dt], dt)
    close(got[2].get(), dh0, e0 * UNIT[dt], "float64" if dt == "float64" else "float32")


# (outer, steps, inner): rows copied as tensors in blocks alone and in clusters,
# one wave and several, and as many blocks as take clusters of eight in several
LONG = [(1, 5000, 256), (3, 2500, 512), (2, 1500, 1000), (40, 200, 512), (6, 1000, 1024), (1, 10800, 1248),
        (1, 700, 4000)]


@pytest.mark.parametrize("dt,gated", [("float16", True), ("float32", False), ("float32", True), ("float64", True)])
@pytest.mark.parametrize("shape", LONG)
def test_recurrence_long(cp, dt, gated, shape):
    if dt == "float64" and shape[1] * shape[0] * shape[2] > 2 ** 22:
        shape = (shape[0], shape[1] // 8, shape[2])
    a, x, h0, g, gs = rec_inputs(shape, dt, gated, shape[1])
    hs, es, last, el = recurrence(a, x, h0, gated)
    state = cp.empty(h0.shape, dtype=str(h0.dtype))
    h = cp.linear_recurrence(cp.array(a), cp.array(x), cp.array(h0), gated=gated, state_out=state)
    close(h.get(), hs, es * UNIT[dt], dt)
    close(state.get(), last, el * UNIT[dt], str(state.dtype))
    del hs, es
    da, dx, dh0, ea, ex, e0 = recurrence_grad(a, x, h.get(), g, h0, gs, gated)
    got = cp.linear_recurrence_grad(cp.array(a), cp.array(x), h, cp.array(g), cp.array(h0), gated=gated,
                                    grad_state=cp.array(gs))
    close(got[0].get(), da, ea * UNIT[dt], dt)
    close(got[1].get(), dx, ex * UNIT[dt], dt)
    close(got[2].get(), dh0, e0 * UNIT[dt], str(h0.dtype))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape", [(3, 701, 257), (6, 640, 258), (2, 1000, 512)])
def test_recurrence_gated_in_clusters(cp, dt, shape):
    """25 to 32 blocks of chains, in clusters of eight, for each way rows are
    copied; gates that keep and that replace the state; equal calls give equal
    bits."""
    a, x, h0, g, gs = rec_inputs(shape, dt, True, 700)
    a[:, 350], a[:, 353] = np.inf, -np.inf
    hs, es, last, el = recurrence(a, x, h0, True)
    sdt = "float64" if dt == "float64" else "float32"
    state = cp.empty((shape[0], shape[2]), dtype=sdt)
    h = cp.linear_recurrence(cp.array(a), cp.array(x), cp.array(h0), gated=True, state_out=state)
    close(h.get(), hs, es * UNIT[dt], dt)
    close(state.get(), last, el * UNIT[dt], sdt)
    again = cp.linear_recurrence(cp.array(a), cp.array(x), cp.array(h0), gated=True)
    np.testing.assert_array_equal(again.get(), h.get())
    h = hs.astype(dt)
    da, dx, dh0, ea, ex, e0 = recurrence_grad(a, x, h, g, h0, gs, True)
    got = cp.linear_recurrence_grad(cp.array(a), cp.array(x), cp.array(h), cp.array(g), cp.array(h0), gated=True,
                                    grad_state=cp.array(gs))
    close(got[0].get(), da, ea * UNIT[dt], dt)
    close(got[1].get(), dx, ex * UNIT[dt], dt)
    close(got[2].get(), dh0, e0 * UNIT[dt], sdt)


def test_recurrence_decays_above_one(cp):
    """Spans whose decays multiply past float32's range: a state of zero stays
    zero, and what is finite step by step is finite."""
    steps, width = 3000, 64
    a = np.full((1, steps, width), 2.0, np.float32)
    x = np.zeros((1, steps, width), np.float32)
    x[0, -30:, ::2] = 1.0
    h = cp.linear_recurrence(cp.array(a), cp.array(x)).get()
    np.testing.assert_array_equal(h[0, :-30], 0)
    np.testing.assert_array_equal(h[0, :, 1::2], 0)
    # 2^k - 1: exact up to k = 24; each step after that rounds once, 2^-24 of a
    # value that its error has grown along with, so six roundings at most
    want = 2.0 ** np.arange(1, 31) - 1
    np.testing.assert_array_equal(h[0, -30:-6, 0], want[:24])
    assert (np.abs(h[0, -6:, 0] - want[24:]) <= 6 * 2.0 ** -24 * want[24:]).all()


def test_recurrence_offsets_past_32_bits(cp):
    """More than 2^31 elements: with decay zero h is x, wherever it lies."""
    steps, width = (1 << 21) + 37, 1032
    x = (cp.arange(steps, dtype="int32") % 1021).astype("float16")
    x = (x.reshape(1, steps, 1) + cp.zeros((1, 1, width), dtype="float16"))
    a = cp.zeros((1, 1, width), dtype="float16").broadcast_to((1, steps, width))
    h = cp.linear_recurrence(a, x)
    assert bool(cp.array_equal(h, x))
    _, dx, _ = cp.linear_recurrence_grad(a, None, h, x, out=(h, cp.empty(x.shape, dtype="float16")))
    assert bool(cp.array_equal(dx, x))


def test_recurrence_nan_stays_in_its_chain(cp):
    a, x, h0, g, _ = rec_inputs((2, 300, 70), "float32", True, 3)
    x[0, 100, 7] = np.nan
    a[1, 200, 69] = np.nan
    h = cp.linear_recurrence(cp.array(a), cp.array(x), cp.array(h0), gated=True).get()
    want = np.zeros_like(x, bool)
    want[0, 100:, 7] = True
    want[1, 200:, 69] = True
    np.testing.assert_array_equal(np.isnan(h), want)


@pytest.mark.parametrize("dt", ["float16", "float32"])
@pytest.mark.parametrize("axis", [0, 1, 2, 3, -1])
def test_recurrence_axes_and_views(cp, dt, axis):
    """Every axis; slices of one larger array, reversed, transposed and
    broadcast operands give what their copies give."""
    rng = np.random.default_rng(axis + 4)
    base = (1 / (1 + np.exp(-rng.normal(2, 1, (4, 37, 6, 22))))).astype(dt)
    A = cp.array(base)
    a, x = base[..., :10], base[..., 11:21]
    ax = axis % 4
    three = lambda v: np.moveaxis(v, ax, -1).reshape(1, -1, v.shape[ax]).transpose(0, 2, 1)  # noqa: E731
    hs, es, _, _ = recurrence(three(a), three(x), None, False)
    got = cp.linear_recurrence(A[..., :10], A[..., 11:21], axis=axis).get()
    close(three(got), hs, es * UNIT[dt], dt)
    same = cp.linear_recurrence(cp.array(a), cp.array(x), axis=axis).get()
    close(three(same), hs, es * UNIT[dt], dt)
    ra, rx = a[:, ::-1], x[:, ::-1]
    hs, es, _, _ = recurrence(three(ra), three(rx), None, False)
    rev = cp.linear_recurrence(A[:, ::-1, :, :10], A[:, ::-1, :, 11:21], axis=axis).get()
    close(three(rev), hs, es * UNIT[dt], dt)
    oa = np.broadcast_to(base[:1, :1, :1, :10], (4, 37, 6, 10))
    hs, es, _, _ = recurrence(three(oa), three(x), None, False)
    one = cp.array(base[:1, :1, :1, :10]).broadcast_to((4, 37, 6, 10))
    close(three(cp.linear_recurrence(one, A[..., 11:21], axis=axis).get()), hs, es * UNIT[dt], dt)


@pytest.mark.parametrize("dt", ["float16", "float32"])
def test_recurrence_time_major_and_skipped_steps(cp, dt):
    """Memory in (steps, batch, width) order, every second step of an odd
    number, every second batch entry, one step and one batch entry."""
    rng = np.random.default_rng(6)
    base = rng.standard_normal((61, 4, 192)).astype(dt)
    B = cp.array(base)
    views = [lambda v: v[..., :96].transpose(1, 0, 2), lambda v: v[..., :96][::2].transpose(1, 0, 2),
             lambda v: v[:, ::2, :64].transpose(1, 0, 2), lambda v: v[:1, :, :64].transpose(1, 0, 2),
             lambda v: v[:, 1:2, :64].transpose(1, 0, 2), lambda v: v[::-1, :, :64].transpose(1, 0, 2),
             lambda v: v[1::2], lambda v: v[3:4]]
    for f in views:
        a, x = f(base), f(base[..., 96:] if f(base).shape[2] < 192 else base)
        hs, es, _, _ = recurrence(a, x, None, True)
        va, vx = f(B), f(B[..., 96:] if f(base).shape[2] < 192 else B)
        h = cp.linear_recurrence(va, vx, gated=True)
        close(h.get(), hs, es * UNIT[dt], dt)
        da, dx, _, ea, ex, _ = recurrence_grad(a, x, h.get(), x, None, None, True)
        got = cp.linear_recurrence_grad(va, vx, h, vx, gated=True)
        close(got[0].get(), da, ea * UNIT[dt], dt)
        close(got[1].get(), dx, ex * UNIT[dt], dt)


@pytest.mark.parametrize("off", range(1, 8))
@pytest.mark.parametrize("dt", ["float16", "float32"])
def test_recurrence_unaligned_views(cp, dt, off):
    """Views that start off a 16-byte boundary, and rows an odd stride apart."""
    rng = np.random.default_rng(off)
    base = (1 / (1 + np.exp(-rng.normal(2, 1, (3, 50, 150 + off))))).astype(dt)
    A = cp.array(base)
    w = 64
    a, x, g = base[..., off:off + w], base[..., off + w:off + 2 * w], base[..., :w]
    va, vx, vg = A[..., off:off + w], A[..., off + w:off + 2 * w], A[..., :w]
    hs, es, _, _ = recurrence(a, x, None, True)
    h = cp.linear_recurrence(va, vx, gated=True)
    close(h.get(), hs, es * UNIT[dt], dt)
    da, dx, _, ea, ex, _ = recurrence_grad(a, x, h.get(), g, None, None, True)
    got = cp.linear_recurrence_grad(va, vx, h, vg, gated=True)
    close(got[0].get(), da, ea * UNIT[dt], dt)
    close(got[1].get(), dx, ex * UNIT[dt], dt)


@pytest.mark.parametrize("dt", ["float16", "float32"])
def test_recurrence_outputs_in_place(cp, dt):
    """out= over the inputs gives the same bits; into a strided view, or over a
    shifted view of an input (rows that start elsewhere may be copied in other
    spans): within the bound; rows of the larger array outside the view stay
    as they were."""
    shape = (2, 150, 70)
    a, x, h0, g, gs = rec_inputs(shape, dt, True, 9)
    hs, es, _, _ = recurrence(a, x, h0, True)
    want = cp.linear_recurrence(cp.array(a), cp.array(x), cp.array(h0), gated=True).get()
    for over in (0, 1):
        A, X = cp.array(a), cp.array(x)
        r = cp.linear_recurrence(A, X, cp.array(h0), gated=True, out=(A, X)[over])
        assert r is (A, X)[over]
        np.testing.assert_array_equal(r.get(), want)
    big = cp.full((2, 152, 80), 7, dtype=dt)
    r = cp.linear_recurrence(cp.array(a), cp.array(x), cp.array(h0), gated=True, out=big[:, 1:151, 5:75])
    close(r.get(), hs, es * UNIT[dt], dt)
    host = np.full((2, 152, 80), 7, dt)
    host[:, 1:151, 5:75] = r.get()
    np.testing.assert_array_equal(big.get(), host)
    X = cp.zeros((2, 151, 70), dtype=dt)
    X[:, :150] = cp.array(x)
    r = cp.linear_recurrence(cp.array(a), X[:, :150], cp.array(h0), gated=True, out=X[:, 1:])
    close(r.get(), hs, es * UNIT[dt], dt)
    dg = [v.get() for v in cp.linear_recurrence_grad(cp.array(a), cp.array(x), cp.array(want), cp.array(g),
                                                     cp.array(h0), gated=True, grad_state=cp.array(gs))]
    A, X, H, G, S = cp.array(a), cp.array(x), cp.array(want), cp.array(g), cp.array(gs)
    r = cp.linear_recurrence_grad(A, X, H, G, cp.array(h0), gated=True, grad_state=S, out=(A, X, S))
    for v, w in zip(r, dg):
        np.testing.assert_array_equal(v.get(), w)
    A, X, H, G = cp.array(a), cp.array(x), cp.array(want), cp.array(g)
    H0 = cp.array(h0)
    r = cp.linear_recurrence_grad(A, X, H, G, H0, gated=True, grad_state=cp.array(gs), out=(H, G, H0))
    for v, w in zip(r, dg):
        np.testing.assert_array_equal(v.get(), w)


def test_recurrence_state_is_carried_exactly(cp):
    """A sequence cut anywhere, the state passed on in place, equals the whole;
    so does one token at a time.  Both sides differ by the order of the decays'
    products only, which the bound of the whole covers twice."""
    shape = (3, 90, 33)
    for dt in ("float16", "float32"):
        a, x, h0, _, _ = rec_inputs(shape, dt, True, 11)
        hs, es, last, el = recurrence(a, x, h0, True)
        for cut in (1, 37, 90):
            s = cp.array(h0)
            got = [cp.linear_recurrence(cp.array(a[:, i:i + cut]), cp.array(x[:, i:i + cut]), s, gated=True,
                                        state_out=s).get() for i in range(0, 90, cut)]
            close(np.concatenate(got, 1), hs, es * UNIT[dt], dt)
            close(s.get(), last, el * UNIT[dt], "float32")


def test_recurrence_empty(cp):
    for shape in ((0, 5, 3), (2, 0, 3), (2, 5, 0)):
        z = cp.zeros(shape, dtype="float32")
        st = cp.full((shape[0], shape[2]), 9, dtype="float32")
        h0 = np.arange(shape[0] * shape[2], dtype=np.float32).reshape(shape[0], shape[2])
        h = cp.linear_recurrence(z, z, cp.array(h0), state_out=st)
        assert h.shape == shape
        np.testing.assert_array_equal(st.get(), h0)
        r = cp.linear_recurrence_grad(z, z, z, z, cp.array(h0), grad_state=cp.array(h0))
        np.testing.assert_array_equal(r[2].get(), h0)


def test_recurrence_is_cumsum_at_decay_one(cp):
    x = np.random.default_rng(0).integers(-9, 10, (3, 700, 45)).astype(np.float32)  # sums are exact
    got = cp.linear_recurrence(cp.ones((3, 700, 45), dtype="float32"), cp.array(x))
    np.testing.assert_array_equal(got.get(), np.cumsum(x, 1))
    np.testing.assert_array_equal(got.get(), cp.cumsum(cp.array(x), axis=1).get())


def test_recurrence_lazy_mixed_and_repeat(cp):
    """Lazy operands, promotion of float16 with float32, equal bits of equal calls."""
    a, x, _, _, _ = rec_inputs((2, 600, 130), "float16", True, 4, h0=False)
    A, X = cp.array(a), cp.array(x)
    r1 = cp.linear_recurrence(A * 1.0, X.astype("float32"), gated=True)
    assert r1.dtype == np.float32
    hs, es, _, _ = recurrence(a, x, None, True)
    close(r1.get(), hs, es * UNIT["float32"], "float32")
    for _ in range(3):
        np.testing.assert_array_equal(cp.linear_recurrence(A, X.astype("float32"), gated=True).get(), r1.get())


# ------------------------------------------------------------------ embedding

EMB = [(1, 1, 1), (2, 3, 1), (5, 7, 3), (31, 1, 64), (33, 100, 65), (64, 50, 128), (257, 1000, 100), (1000, 37, 257),
       (1024, 4096, 8), (1025, 300, 40), (3000, 5000, 30), (4097, 2, 17), (9000, 20000, 24), (40000, 300, 12)]


def ids_of(rng, n, rows, dt):
    return np.minimum(np.exp(rng.random(n) * np.log(rows + 1)) - 1, rows - 1).astype(dt)


@pytest.mark.parametrize("idt", ["int32", "int64"])
@pytest.mark.parametrize("dt", DTYPES)
def test_embedding(cp, dt, idt):
    for i, (n, rows, width) in enumerate(EMB):
        rng = np.random.default_rng(i)
        w = rng.standard_normal((rows, width)).astype(dt)
        ids = ids_of(rng, n, rows, idt)
        got = cp.embedding(cp.array(w), cp.array(ids), 3.3)
        assert got.dtype == np.dtype(dt)
        want = w[ids].astype(np.float64) * 3.3
        close(got.get(), want, 2 * UNIT[dt] * np.abs(want), dt)
        np.testing.assert_array_equal(cp.embedding(cp.array(w), cp.array(ids)).get(), w[ids])
    cp.synchronize()


def grad_of(ids, g, rows, scale, pad=None):
    """(gradient, bound over u) in float64."""
    g = g.astype(np.float64)
    out, mag = np.zeros((rows, g.shape[1])), np.zeros((rows, g.shape[1]))
    np.add.at(out, ids, g)
    np.add.at(mag, ids, np.abs(g))
    count = np.bincount(ids, minlength=rows)[:, None]
    if pad is not None:
        out[pad] = mag[pad] = 0
    return out * scale, (count + 2) * mag * abs(scale)


@pytest.mark.parametrize("idt", ["int32", "int64"])
@pytest.mark.parametrize("dt", DTYPES)
def test_embedding_grad(cp, dt, idt):
    for i, (n, rows, width) in enumerate(EMB):
        rng = np.random.default_rng(50 + i)
        ids = ids_of(rng, n, rows, idt)
        g = rng.standard_normal((n, width)).astype(dt)
        pad = int(ids[0]) if i % 2 else None
        want, err = grad_of(ids, g, rows, 1.7, pad)
        out = cp.full((rows, width), 5, dtype=dt)
        got = cp.embedding_grad(cp.array(ids), cp.array(g), rows, 1.7, padding_idx=pad, out=out)
        assert got is out
        close(got.get(), want, err * UNIT[dt], dt)
        np.testing.assert_array_equal(got.get()[np.bincount(ids, minlength=rows) == 0], 0)
        again = cp.embedding_grad(cp.array(ids), cp.array(g), rows, 1.7, padding_idx=pad)
        np.testing.assert_array_equal(again.get(), got.get())
    cp.synchronize()


@pytest.mark.parametrize("dt", ["float16", "float32"])
@pytest.mark.parametrize("kind", ["one", "all", "last", "two"])
def test_embedding_grad_heavy_ids(cp, dt, kind):
    """One id for every token, every id once, the last row only, two ids in turn."""
    for n in (31, 1000, 5000, 20001):
        rows, width = 30000, 48
        rng = np.random.default_rng(n)
        ids = {"one": np.full(n, 17), "all": rng.permutation(rows)[:n], "last": np.full(n, rows - 1),
               "two": np.arange(n) % 2 * (rows - 1)}[kind].astype(np.int64)
        g = rng.standard_normal((n, width)).astype(dt)
        want, err = grad_of(ids, g, rows, 0.5)
        got = cp.embedding_grad(cp.array(ids), cp.array(g), rows, 0.5).get()
        close(got, want, err * UNIT[dt], dt)


def test_embedding_grad_wide_ids(cp):
    """A table of more than 2^18 and 2^24 rows (longer sort keys)."""
    for rows in ((1 << 18) + 3, (1 << 24) + 11):
        rng = np.random.default_rng(rows)
        ids = np.concatenate([rng.integers(0, rows, 3000), [0, rows - 1, rows - 1]]).astype(np.int32)
        g = rng.standard_normal((len(ids), 2)).astype(np.float32)
        want, err = grad_of(ids, g, rows, 1.0)
        close(cp.embedding_grad(cp.array(ids), cp.array(g), rows).get(), want, err * UNIT["float32"], "float32")


def test_embedding_shapes_views_and_empty(cp):
    rng = np.random.default_rng(8)
    big = rng.standard_normal((50, 90)).astype(np.float32)
    B = cp.array(big)
    ids = rng.integers(0, 20, (3, 4, 5)).astype(np.int16)
    got = cp.embedding(B[10:50:2, 7:71], cp.array(ids), 2.0)
    np.testing.assert_array_equal(got.get(), big[10:50:2, 7:71][ids] * 2)
    np.testing.assert_array_equal(cp.embedding(B[:, ::3], cp.array(ids)).get(), big[:, ::3][ids])
    np.testing.assert_array_equal(cp.embedding(B.T, cp.array(ids)).get(), big.T[ids])
    assert cp.embedding(B, cp.array(3, dtype="int64")).shape == (90,)
    assert cp.embedding(B, cp.zeros((0,), dtype="int64")).shape == (0, 90)
    g = rng.standard_normal((3, 4, 5, 96)).astype(np.float32)
    G = cp.array(g)
    want, err = grad_of(ids.reshape(-1), g[..., 3:93].reshape(-1, 90), 20, 1.0)
    close(cp.embedding_grad(cp.array(ids), G[..., 3:93], 20).get(), want, err * UNIT["float32"], "float32")
    z = cp.embedding_grad(cp.zeros((0,), dtype="int64"), cp.zeros((0, 6), dtype="float32"), 4)
    np.testing.assert_array_equal(z.get(), np.zeros((4, 6), np.float32))
    assert cp.embedding_grad(cp.array(ids), cp.zeros((3, 4, 5, 0), dtype="float32"), 20).shape == (20, 0)
    wide = cp.full((22, 90), 3, dtype="float32")
    r = cp.embedding_grad(cp.array(ids), G[..., 3:93], 20, out=wide[1:21])
    close(r.get(), want, err * UNIT["float32"], "float32")
    np.testing.assert_array_equal(wide.get()[[0, 21]], np.full((2, 90), 3, np.float32))
    cp.synchronize()


def test_embedding_offsets_past_32_bits(cp):
    """Tables of more than 2^31 elements, few tokens and many."""
    rows, width = (1 << 21) + 5, 1032
    w = cp.zeros((rows, width), dtype="float16")
    w[rows - 1] = 3
    w[rows - 2, 1000:] = 5
    ids = np.array([rows - 1, 0, rows - 2, rows - 1], np.int64)
    got = cp.embedding(w, cp.array(ids), 2.0).get()
    want = np.zeros((4, width), np.float16)
    want[[0, 3]] = 6
    want[2, 1000:] = 10
    np.testing.assert_array_equal(got, want)
    for n in (4, 4000):
        many = np.resize(ids, n)
        out = cp.embedding_grad(cp.array(many), cp.ones((n, width), dtype="float16"), rows, out=w)
        count = np.bincount(many, minlength=rows)
        assert float(cp.sum(out[1:rows - 2].astype("float32")).get()) == 0
        np.testing.assert_array_equal(out[[0, rows - 2, rows - 1]].get(),
                                      np.repeat(count[[0, rows - 2, rows - 1], None], width, 1))
    cp.synchronize()


def test_embedding_ids_out_of_range(cp):
    """A bad id gives zeros (lookup) or adds nothing (gradient), and the next
    synchronize raises once."""
    w = np.arange(12, dtype=np.float32).reshape(4, 3) + 1
    ids = np.array([0, 4, 3, -1, 2 ** 40], np.int64)
    got = cp.embedding(cp.array(w), cp.array(ids)).get()
    np.testing.assert_array_equal(got, np.stack([w[0], 0 * w[0], w[3], 0 * w[0], 0 * w[0]]))
    with pytest.raises(RuntimeError, match="5"):
        cp.synchronize()
    cp.synchronize()
    for reps in (1, 2000):  # a few tokens and many
        many = np.tile(ids, reps)
        g = np.ones((len(many), 3), np.float32)
        got = cp.embedding_grad(cp.array(many), cp.array(g), 4).get()
        want = np.zeros((4, 3), np.float32)
        want[[0, 3]] = reps
        np.testing.assert_array_equal(got, want)
        with pytest.raises(RuntimeError, match="5"):
            cp.synchronize()
    cp.synchronize()


def test_embedding_grad_nan_stays_in_its_row(cp):
    ids = np.random.default_rng(0).integers(0, 50, 4000)
    g = np.ones((4000, 20), np.float32)
    g[123, 4] = np.nan
    g[7, 5] = np.inf
    got = cp.embedding_grad(cp.array(ids), cp.array(g), 50).get()
    bad = ~np.isfinite(got)
    want = np.zeros_like(bad)
    want[ids[123], 4] = want[ids[7], 5] = True
    np.testing.assert_array_equal(bad, want)


# ------------------------------------------------------------------ global norm

def norm_lists(seed, kinds):
    rng = np.random.default_rng(seed)
    sizes = [(1,), (3, 5), (0,), (16384,), (16385,), (127, 129), (), (100003,), (2, 3, 4)]
    return [np.asarray(rng.standard_normal(s)).astype(kinds[i % len(kinds)]) for i, s in enumerate(sizes)]


@pytest.mark.parametrize("kinds", [["float16"], ["float32"], ["float64"], ["float16", "float32"],
                                   ["float64", "float16", "float32"]])
def test_clip_by_global_norm(cp, kinds):
    arrays = norm_lists(1, kinds)
    want = np.sqrt(sum((a.astype(np.float64) ** 2).sum() for a in arrays))
    ndt = "float64" if "float64" in kinds else "float32"
    # n u over the float64 sum of about 2^18 terms, and the rounding of the result
    close(cp.global_norm([cp.array(a) for a in arrays]).get(), want, 2.0 ** 19 * 2.0 ** -53 * want, ndt)
    for limit in (0.37, want * 0.999, want * 1.001, 1e9, 0.0):
        A = [cp.array(a) for a in arrays]
        res, norm = cp.clip_by_global_norm(A, limit)
        assert norm.dtype == np.dtype(ndt) and norm.shape == ()
        coef = 1.0 if want <= limit else limit / want
        for r, a in zip(res, arrays):
            assert r.dtype == a.dtype and r.shape == a.shape
            v = a.astype(np.float64) * coef
            close(r.get(), v, (0 if coef == 1 else 2 * UNIT[str(a.dtype)] + 2.0 ** -30 * (ndt == "float32")) * np.abs(v)
                  + (0 if coef == 1 else 2.0 ** -34 * np.abs(v) * (str(a.dtype) == "float64")), str(a.dtype))
            if coef == 1:
                np.testing.assert_array_equal(r.get(), a)
        r2, n2 = cp.clip_by_global_norm(A, limit, out=A)
        assert all(p is q for p, q in zip(r2, A))
        assert float(n2) == float(norm)
        for p, q in zip(r2, res):
            np.testing.assert_array_equal(p.get(), q.get())


def test_global_norm_limits(cp):
    assert float(cp.global_norm([])) == 0.0
    assert float(cp.global_norm([cp.zeros((0,), dtype="float16")])) == 0.0
    big = np.full(1000, 3e30, np.float32)  # squares pass float32's range
    got = float(cp.global_norm([cp.array(big)]))
    want = 3e30 * np.sqrt(1000)
    assert abs(got - want) <= 2.0 ** -22 * want
    small = np.full(1000, 1e-30, np.float32)
    assert abs(float(cp.global_norm([cp.array(small)])) - 1e-30 * np.sqrt(1000)) <= 2.0 ** -22 * 1e-28
    z = cp.zeros((5,), dtype="float32")
    r, n = cp.clip_by_global_norm([z], 0.0)
    assert float(n) == 0 and not r[0].get().any()
    bad = np.array([1, np.inf, -2], np.float32)
    r, n = cp.clip_by_global_norm([cp.array(bad), cp.ones((3,), dtype="float16")], 1.0)
    assert np.isinf(float(n))
    np.testing.assert_array_equal(r[0].get(), np.array([0, np.nan, -0.0], np.float32))
    np.testing.assert_array_equal(r[1].get(), np.zeros(3, np.float16))
    r, n = cp.clip_by_global_norm([cp.array(np.array([1, np.nan], np.float32)), cp.ones((3,), dtype="float16")], 1.0)
    assert np.isnan(float(n)) and np.isnan(r[0].get()).all() and np.isnan(r[1].get()).all()


def test_global_norm_many_arrays(cp):
    """More arrays than one launch's table holds; unaligned views; equal bits
    of equal calls."""
    rng = np.random.default_rng(2)
    base = rng.standard_normal(60000).astype(np.float32)
    B = cp.array(base)
    cuts = np.concatenate([[0], np.sort(rng.integers(0, 60000, 1299)), [60000]])
    parts = [B[i:j] for i, j in zip(cuts, cuts[1:])]
    want = np.sqrt((base.astype(np.float64) ** 2).sum())
    norms = [float(cp.global_norm(parts)) for _ in range(3)]
    assert norms[0] == norms[1] == norms[2]
    assert abs(norms[0] - want) <= 2.0 ** -23 * want
    res, _ = cp.clip_by_global_norm(parts, 1.0)
    v = base.astype(np.float64) / want
    close(np.concatenate([r.get() for r in res]), v, 4 * UNIT["float32"] * np.abs(v), "float32")
    cp.clip_by_global_norm(parts, 1.0, out=parts)
    np.testing.assert_array_equal(B.get(), np.concatenate([r.get() for r in res]))


def test_clip_outputs_that_overlap(cp):
    """The same array twice (tied weights) is scaled once; outputs over other
    inputs and strided outputs get what separate ones get."""
    x = np.random.default_rng(3).standard_normal(5000).astype(np.float32)
    X = cp.array(x)
    n = np.sqrt(2 * (x.astype(np.float64) ** 2).sum())
    r, norm = cp.clip_by_global_norm([X, X], 1.0, out=[X, X])
    v = x.astype(np.float64) / n
    close(X.get(), v, 4 * UNIT["float32"] * np.abs(v), "float32")
    a, b = cp.array(x[:2000]), cp.array(x[2000:4000])
    want, _ = cp.clip_by_global_norm([a, b], 1.0)
    want = [w.get() for w in want]
    cp.clip_by_global_norm([a, b], 1.0, out=[b, a])
    np.testing.assert_array_equal(b.get(), want[0])
    np.testing.assert_array_equal(a.get(), want[1])
    wide = cp.full((2000, 3), 4, dtype="float32")
    a = cp.array(x[:2000])
    r, _ = cp.clip_by_global_norm([a], 1.0, out=[wide[:, 1]])
    np.testing.assert_array_equal(wide.get()[:, 1], cp.clip_by_global_norm([a], 1.0)[0][0].get())
    np.testing.assert_array_equal(wide.get()[:, ::2], np.full((2000, 2), 4, np.float32))
    t = cp.array(x[:2000].reshape(40, 50)).T
    r, _ = cp.clip_by_global_norm([t], 1.0, out=[t])
    w = x[:2000].reshape(40, 50).T.astype(np.float64)
    w = w / np.sqrt((w ** 2).sum())
    close(t.get(), w, 4 * UNIT["float32"] * np.abs(w), "float32")


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("dt", ["float32", "float64"])
def test_a_training_step(cp, dt):
    """Tokens through the lookup, a projection to gates and candidates, the
    gated recurrence and a squared loss, back to every gradient, clipped: each
    gradient against central differences of the float64 loss."""
    rng = np.random.default_rng(0)
    rows, d, batch, steps = 11, 6, 2, 9
    table, proj = rng.standard_normal((rows, d)), rng.standard_normal((d, 2 * d))
    ids = rng.integers(0, rows, (batch, steps))
    target = rng.standard_normal((batch, steps, d))
    scale = 1.5

    def step(table, proj, dt):
        T, P = cp.array(table.astype(dt)), cp.array(proj.astype(dt))
        e = cp.embedding(T, cp.array(ids), scale)
        zx = e @ P
        z, x = zx[..., :d], zx[..., d:]
        h = cp.linear_recurrence(z, x, gated=True)
        diff = h - cp.array(target.astype(dt))
        loss = float(cp.sum(diff * diff).get())
        dzx = cp.empty((batch, steps, 2 * d), dtype=dt)
        cp.linear_recurrence_grad(z, x, h, 2 * diff, gated=True, out=(dzx[..., :d], dzx[..., d:]))
        flat = dzx.reshape(batch * steps, 2 * d)
        dP = e.reshape(batch * steps, d).T @ flat
        dT = cp.embedding_grad(cp.array(ids), dzx @ P.T, rows, scale)
        return loss, dT, dP

    loss, dT, dP = step(table, proj, dt)
    grads = [dT.get(), dP.get()]
    for k, val in enumerate((table, proj)):
        for _ in range(10):
            at = tuple(rng.integers(0, n) for n in val.shape)
            two = []
            for s in (1e-5, -1e-5):
                args = [table.copy(), proj.copy()]
                args[k][at] += s
                two.append(step(*args, "float64")[0])
            diff = (two[0] - two[1]) / 2e-5
            # differences of a loss of order 10^2: 1e-14 / 1e-5 rounding and a
            # cubic term 1e-10 times third derivatives of order 10^3; float32
            # gradients: some 100 roundings of terms of order 10^2 at 2^-24
            tol = 1e-5 if dt == "float64" else 100 * 100 * 2.0 ** -24
            assert abs(diff - grads[k][at]) <= tol * max(1.0, abs(diff)), (k, at)
    n = np.sqrt(sum((g.astype(np.float64) ** 2).sum() for g in grads))
    clipped, norm = cp.clip_by_global_norm([dT, dP], 0.5, out=[dT, dP])
    assert abs(float(norm) - n) <= 2.0 ** -22 * n
    for c, g in zip(clipped, grads):
        close(c.get(), g.astype(np.float64) * (0.5 / n), 4 * UNIT[dt] * np.abs(g) * (0.5 / n), dt)


def test_decode_follows_training(cp):
    """One token at a time from the lookup through the recurrence gives what
    the whole sequence gives (each within its own bound)."""
    rng = np.random.default_rng(4)
    rows, d, steps = 40, 50, 12
    table = rng.standard_normal((rows, d)).astype(np.float16)
    gate = rng.standard_normal((rows, d)).astype(np.float16)
    ids = rng.integers(0, rows, (3, steps))
    T, G = cp.array(table), cp.array(gate)
    whole = cp.linear_recurrence(cp.embedding(G, cp.array(ids)), cp.embedding(T, cp.array(ids)), gated=True).get()
    hs, es, _, _ = recurrence(gate[ids], table[ids], None, True)
    close(whole, hs, es * UNIT["float16"], "float16")
    s = cp.zeros((3, d), dtype="float32")
    for t in range(steps):
        i = cp.array(ids[:, t:t + 1])
        h = cp.linear_recurrence(cp.embedding(G, i), cp.embedding(T, i), s, gated=True, state_out=s)
        close(h.get()[:, 0], hs[:, t], es[:, t] * UNIT["float16"], "float16")


def test_from_several_threads(cp):
    """Calls from several threads at once (each gets its own results)."""
    import threading

    from macmetalpy_b200 import _cuda_backend as cb

    rng = np.random.default_rng(9)
    work = []
    for k in range(4):
        a, x, _, _, _ = rec_inputs((2, 400 + k, 96), "float32", True, 40 + k)
        ids, g = rng.integers(0, 3000, 5000 + k), rng.standard_normal((5000 + k, 24)).astype(np.float32)
        work.append((a, x, ids, g))

    def one(w, to):
        a, x, ids, g = w
        cb.check(cb.lib.mmp_init(cb.CudaBackend().device))  # the device of a new thread
        for _ in range(5):
            h = cp.linear_recurrence(cp.array(a), cp.array(x), gated=True)
            d = cp.embedding_grad(cp.array(ids), cp.array(g), 3000)
            _, n = cp.clip_by_global_norm([h, d], 1.0)
            to.append((h.get(), d.get(), float(n)))

    alone, together = [[] for _ in work], [[] for _ in work]
    for w, to in zip(work, alone):
        one(w, to)
    threads = [threading.Thread(target=one, args=(w, to)) for w, to in zip(work, together)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for p, q in zip(alone, together):
        assert len(q) == 5
        for r in q:
            np.testing.assert_array_equal(r[0], p[0][0])
            np.testing.assert_array_equal(r[1], p[0][1])
            assert r[2] == p[0][2]


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
f = lambda *s, dt="float32": cp.array(rng.standard_normal(s).astype(dt))
z, x, g = f(2, 700, 128, dt="float16"), f(2, 700, 128, dt="float16"), f(2, 700, 128, dt="float16")
h, da, dx = (cp.empty((2, 700, 128), dtype="float16") for _ in range(3))
s = cp.zeros((2, 128), dtype="float32")
ids = [cp.array(rng.integers(0, 500, n)) for n in (300, 3000)]
gr = [f(n, 40) for n in (300, 3000)]
dw = [cp.empty((500, 40), dtype="float32") for _ in ids]
e = cp.empty((300, 40), dtype="float32")
clipped = [cp.empty((500, 40), dtype="float32") for _ in ids]
norm = cp.empty((), dtype="float32")
def step():
    cp.linear_recurrence(z, x, s, gated=True, out=h, state_out=s)
    cp.linear_recurrence_grad(z, x, h, g, gated=True, out=(da, dx))
    for i, r, d in zip(ids, gr, dw):
        cp.embedding_grad(i, r, 500, 2.0, out=d)
    cp.embedding(dw[0], ids[0], 0.5, out=e)
    cp.clip_by_global_norm(dw, 1.0, out=clipped, norm_out=norm)
def results():
    return [a.get() for a in (h, da, dx, s, e, norm, *dw, *clipped)]
step(); step(); cp.synchronize()
graphs = []
for _ in range(2):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    graphs.append(graph)
for k in range(4):
    new = [rng.standard_normal(a.shape).astype(a.dtype) for a in (z, x, g, *gr)]
    for a, v in zip((z, x, g, *gr), new):
        a.set(v)
    for i in ids:
        i.set(rng.integers(0, 500, i.shape))
    s0 = rng.standard_normal((2, 128)).astype("float32")
    s.set(s0); cp.synchronize()
    step(); want = results()
    s.set(s0); cp.synchronize()
    with torch.cuda.stream(stream):
        graphs[k % 2].replay()
    torch.cuda.synchronize()
    for p, q in zip(want, results()):
        np.testing.assert_array_equal(p, q)
cp.synchronize()
print("captured")
"""


def test_captured_and_replayed(cp):
    """Every operator captured into two graphs on a foreign stream and replayed
    on new inputs gives what the plain calls give (a process of its own: the
    library keeps the stream it is given)."""
    import os
    import subprocess
    import sys

    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    p = subprocess.run([sys.executable, "-c", CAPTURE.format(repo=repo)], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and "captured" in p.stdout, p.stdout + p.stderr
