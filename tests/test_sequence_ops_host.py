"""Refusals of the sequence operators, and the host-side rules on views and
overlaps: no GPU and no library call (arrays over made-up addresses)."""

import ctypes

import numpy as np
import pytest

from macmetalpy_b200 import _cuda_backend as cb
from macmetalpy_b200 import sequence_ops as so
from macmetalpy_b200.ndarray import ndarray


class Buf:
    def __init__(self, ptr, nbytes):
        self.ptr, self.nbytes = ptr, nbytes


_next = [1 << 20]


def arr(shape, dt="float32", strides=None, offset=0, buf=None):
    n = int(np.prod(shape, dtype=np.int64)) * np.dtype(dt).itemsize
    if buf is None:
        buf = Buf(_next[0], n)
        _next[0] += (n + 4096) // 256 * 256
    return ndarray(buf, shape, dt, strides=strides, offset=offset)


@pytest.fixture(autouse=True)
def no_device(monkeypatch):
    """Any use of the device from here on is a failure of the test."""
    def fail(*a, **k):
        raise AssertionError("the device was reached")
    monkeypatch.setattr(ndarray, "_empty", classmethod(lambda cls, shape, dt: arr(tuple(shape), dt)))
    monkeypatch.setattr(ndarray, "_empty0", classmethod(lambda cls, dt: arr((), dt)))
    monkeypatch.setattr(ndarray, "_contiguous_copy", lambda self: arr(self._shape, self._dtype))

    class Lib:
        def __getattr__(self, name):
            return fail
    monkeypatch.setattr(so._cb, "lib", Lib())


def test_recurrence_refusals():
    a, x = arr((2, 5, 3)), arr((2, 5, 3))
    with pytest.raises(ValueError, match="shape"):
        so.linear_recurrence(a, arr((2, 5, 4)))
    with pytest.raises(TypeError, match="floating"):
        so.linear_recurrence(arr((2, 5, 3), "int32"), arr((2, 5, 3), "int32"))
    with pytest.raises(np.exceptions.AxisError):
        so.linear_recurrence(a, x, axis=3)
    with pytest.raises(np.exceptions.AxisError):
        so.linear_recurrence(arr((5,)), arr((5,)))  # the default axis is -2
    with pytest.raises(ValueError, match="axis"):
        so.linear_recurrence(arr(()), arr(()))
    with pytest.raises(ValueError, match="h0"):
        so.linear_recurrence(a, x, arr((2, 5)))
    with pytest.raises(TypeError, match="floating"):
        so.linear_recurrence(a, x, arr((2, 3), "int64"))
    with pytest.raises(ValueError, match="out"):
        so.linear_recurrence(a, x, out=arr((2, 5, 3), "float16"))
    with pytest.raises(TypeError, match="out"):
        so.linear_recurrence(a, x, out=np.zeros((2, 5, 3), np.float32))
    with pytest.raises(ValueError, match="state_out"):
        so.linear_recurrence(arr((2, 5, 3), "float16"), arr((2, 5, 3), "float16"), state_out=arr((2, 3), "float16"))
    with pytest.raises(AssertionError, match="reached"):  # and a right call gets there
        so.linear_recurrence(a, x, arr((2, 3)), out=arr((2, 5, 3)), state_out=arr((2, 3)))


def test_recurrence_grad_refusals():
    a, x, h, g = (arr((2, 5, 3)) for _ in range(4))
    with pytest.raises(ValueError, match="x is needed"):
        so.linear_recurrence_grad(a, None, h, g, gated=True)
    with pytest.raises(ValueError, match="differ"):
        so.linear_recurrence_grad(a, x, h, arr((2, 5)))
    with pytest.raises(ValueError, match="grad_state"):
        so.linear_recurrence_grad(a, x, h, g, grad_state=arr((3, 2)))
    with pytest.raises(ValueError, match="tuple of 2"):
        so.linear_recurrence_grad(a, x, h, g, out=(a, x, arr((2, 3))))
    with pytest.raises(ValueError, match="tuple of 3"):
        so.linear_recurrence_grad(a, x, h, g, arr((2, 3)), out=(a, x))
    with pytest.raises(AssertionError, match="reached"):
        so.linear_recurrence_grad(a, None, h, g)


def test_embedding_refusals():
    w, ids = arr((10, 4)), arr((3,), "int64")
    with pytest.raises(ValueError, match="2-D"):
        so.embedding(arr((10,)), ids)
    with pytest.raises(TypeError, match="integers"):
        so.embedding(w, arr((3,), "float32"))
    with pytest.raises(TypeError, match="floating"):
        so.embedding(arr((10, 4), "int32"), ids)
    with pytest.raises(ValueError, match="out"):
        so.embedding(w, ids, out=arr((3, 5)))
    with pytest.raises(ValueError, match="grad"):
        so.embedding_grad(ids, arr((4, 4)), 10)
    with pytest.raises(ValueError, match="num_rows"):
        so.embedding_grad(ids, arr((3, 4)), -1)
    with pytest.raises(IndexError, match="padding_idx"):
        so.embedding_grad(ids, arr((3, 4)), 10, padding_idx=10)
    with pytest.raises(ValueError, match="out"):
        so.embedding_grad(ids, arr((3, 4)), 10, out=arr((10, 4), "float16"))
    with pytest.raises(AssertionError, match="reached"):
        so.embedding_grad(ids, arr((3, 4)), 10, padding_idx=-1, out=arr((10, 4)))


def test_norm_refusals():
    with pytest.raises(TypeError, match="list"):
        so.global_norm(arr((3,)))
    with pytest.raises(TypeError, match="floating"):
        so.global_norm([arr((3,), "int32")])
    with pytest.raises(ValueError, match="out"):
        so.global_norm([arr((3,))], out=arr((), "float64"))
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            so.clip_by_global_norm([arr((3,))], bad)
    with pytest.raises(ValueError, match="list of 1"):
        so.clip_by_global_norm([arr((3,))], 1.0, out=[])
    with pytest.raises(ValueError, match="out"):
        so.clip_by_global_norm([arr((3,))], 1.0, out=[arr((3,), "float16")])
    a = arr((3,))
    with pytest.raises(ValueError, match="overlaps"):
        so.clip_by_global_norm([a], 1.0, norm_out=ndarray(a._buffer, (), "float32"))


def test_block_distributed_arrays_are_refused():
    class DistArray:
        pass
    with pytest.raises(TypeError, match="distributed"):
        so.linear_recurrence(DistArray(), DistArray())
    with pytest.raises(TypeError, match="distributed"):
        so.embedding(DistArray(), arr((3,), "int64"))
    with pytest.raises(TypeError, match="distributed"):
        so.global_norm([DistArray()])


def test_strides3():
    a = arr((4, 7, 6, 5))
    assert so._strides3(a, 0) == (0, 210)
    assert so._strides3(a, 1) == (210, 30)
    assert so._strides3(a, 2) == (30, 5)
    assert so._strides3(a, 3) == (5, 1)
    buf = a._buffer
    half = ndarray(buf, (4, 7, 2, 5), "float32", strides=(210, 30, 5, 1))
    assert so._strides3(half, 1) == (210, 30)      # inner 2 x 5 contiguous
    assert so._strides3(half, 2) == (30, 5)
    cols = ndarray(buf, (4, 7, 6, 3), "float32", strides=(210, 30, 5, 1))
    assert so._strides3(cols, 1) is None            # inner 6 x 3 is not
    assert so._strides3(cols, 2) == (30, 5)
    every = ndarray(buf, (4, 7, 3, 5), "float32", strides=(210, 30, 10, 1))
    assert so._strides3(every, 2) == (30, 10)
    odd = ndarray(buf, (2, 7, 6, 5), "float32", strides=(420, 30, 5, 1))
    assert so._strides3(odd, 2) is None             # outer axes of two strides
    rev = ndarray(buf, (4, 7, 30), "float32", strides=(210, -30, 1), offset=180)
    assert so._strides3(rev, 1) == (210, -30)
    assert so._strides3(ndarray(buf, (4, 7, 30), "float32", strides=(0, 0, 0)), 1) is None
    assert so._strides3(ndarray(buf, (4, 7, 30), "float32", strides=(0, 30, 1)), 1) == (0, 30)


def test_overlap_and_spans():
    buf = Buf(4096, 4000)
    a = ndarray(buf, (10, 10), "float32")
    assert so._span(a) == (4096, 4496)
    b = ndarray(buf, (10, 10), "float32", offset=100)
    assert not so._overlap(a, b)
    assert so._overlap(a, ndarray(buf, (10, 10), "float32", offset=99))
    rev = ndarray(buf, (10,), "float32", strides=(-1,), offset=9)
    assert so._span(rev) == (4096, 4136)
    assert so._same(a, ndarray(buf, (10, 10), "float32"))
    assert not so._same(a, ndarray(buf, (10, 10), "float32", strides=(1, 10)))


def test_out3_rules():
    a, x = arr((2, 5, 3)), arr((2, 5, 3))
    pick = lambda out: so._out3(out, (2, 5, 3), a._dtype, 1, "t", "out", (a, x), (True, False))[0]  # noqa: E731
    assert pick(a) is a                       # an input it may be
    assert pick(x) is not x                   # one it may not be
    big = Buf(1 << 30, 4000)
    free = ndarray(big, (2, 5, 3), "float32", strides=(100, 10, 1))
    assert pick(free) is free
    assert pick(ndarray(big, (2, 5, 3), "float32", strides=(0, 10, 1))) is not None
    flat = ndarray(big, (2, 5, 3), "float32", strides=(0, 10, 1))
    assert pick(flat) is not flat             # two rows in one place
    cols = ndarray(big, (2, 5, 3), "float32", strides=(100, 10, 2))
    assert pick(cols) is not cols             # columns not adjacent


def test_norm_output_rules():
    a, b = arr((100,)), arr((100,))
    for outs, kept in (([a, b], [True, True]), ([b, a], [False, False]),
                       ([arr((100,)), arr((100,))], [True, True])):
        mine = list(outs)
        so._norm_outs(mine, [a, b])
        assert [m is o for m, o in zip(mine, outs)] == kept
    mine = [a, a]
    so._norm_outs(mine, [a, a])
    assert mine[0] is not a and mine[1] is not a
    c = arr((100,))
    mine = [c, c]
    so._norm_outs(mine, [a, b])
    assert mine[0] is c and mine[1] is not c
    part = ndarray(a._buffer, (50,), "float32", offset=10)
    mine = [part]
    so._norm_outs(mine, [ndarray(a._buffer, (50,), "float32")])
    assert mine[0] is not part


def test_c_entries_refuse():
    """The C ABI's own checks (before any device use)."""
    L = ctypes.CDLL(cb.LIB_PATH)
    for name in ("mmp_recurrence", "mmp_recurrence_grad", "mmp_embedding", "mmp_embedding_grad", "mmp_global_norm"):
        fn = getattr(L, name)
        fn.restype, fn.argtypes = cb.SIGNATURES[name]
    P = ctypes.c_void_p(4096)
    assert L.mmp_recurrence(5, 0, 1, 1, 1, P, 1, 1, P, 1, 1, None, P, 1, 1, None) == -2      # int32
    assert L.mmp_recurrence(10, 0, -1, 1, 1, P, 1, 1, P, 1, 1, None, P, 1, 1, None) == -2
    assert L.mmp_recurrence(10, 0, 1, 1, 1, None, 1, 1, P, 1, 1, None, P, 1, 1, None) == -2
    assert L.mmp_recurrence(10, 0, 1 << 40, 1, 1 << 40, P, 1, 1, P, 1, 1, None, P, 1, 1, None) == -2
    assert L.mmp_recurrence(10, 0, 0, 1, 1, None, 1, 1, None, 1, 1, None, None, 1, 1, None) == 0  # nothing to do
    assert L.mmp_recurrence_grad(10, 1, 1, 1, 1, P, 1, 1, None, 1, 1, P, 1, 1, P, 1, 1, None, None, P, 1, 1, P, 1, 1,
                                 None) == -2                                                  # gated without x
    assert L.mmp_embedding(10, P, 4, 4, 4, 3, P, 1, 1.0, P) == -2                             # int16 ids
    assert L.mmp_embedding(10, P, -4, 4, 4, 5, P, 1, 1.0, P) == -2
    assert L.mmp_embedding(10, P, 1 << 31, 4, 4, 5, P, 1, 1.0, P) == -2
    assert L.mmp_embedding(10, None, 4, 4, 4, 5, None, 0, 1.0, None) == 0
    assert L.mmp_embedding_grad(10, 5, None, 3, P, 4, 4, 4, 1.0, -1, P) == -2
    assert L.mmp_embedding_grad(6, 5, P, 3, P, 4, 4, 4, 1.0, -1, P) == -2
    assert L.mmp_embedding_grad(10, 5, None, 0, None, 4, 0, 4, 1.0, -1, None) == 0
    assert L.mmp_global_norm(-1, None, None, None, None, 1.0, 10, P) == -2
    assert L.mmp_global_norm(1, None, None, None, None, 1.0, 10, P) == -2
    one = (ctypes.c_int * 1)(5)
    ptr, size = (ctypes.c_void_p * 1)(4096), (ctypes.c_int64 * 1)(3)
    assert L.mmp_global_norm(1, one, ptr, None, size, 1.0, 10, P) == -2                       # int32
    one[0] = 10
    assert L.mmp_global_norm(1, one, ptr, None, size, 1.0, 9, P) == -2                        # half norm
    size[0] = -3
    assert L.mmp_global_norm(1, one, ptr, None, size, 1.0, 10, P) == -2


class Recorder:
    """The library's calls with their arguments; each returns 0."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


def test_recurrence_grad_without_gates_leaves_x_alone(monkeypatch):
    """x is not read there, so its dtype has no part in the result's."""
    lib = Recorder()
    monkeypatch.setattr(so._cb, "lib", lib)
    a, h, g = (arr((2, 5, 3)) for _ in range(3))
    for x in (arr((2, 5, 3), "float64"), arr((2, 5, 3), "int32"), None):
        da, dx, _ = so.linear_recurrence_grad(a, x, h, g)
        assert da.dtype == dx.dtype == np.float32
        so.linear_recurrence_grad(a, x, h, g, out=(arr((2, 5, 3)), arr((2, 5, 3))))
    assert [c[1][0] for c in lib.calls] == [so.MMP_CODES[np.dtype("float32")]] * 6
    with pytest.raises(ValueError, match="differ"):
        so.linear_recurrence_grad(a, arr((2, 5, 4)), h, g)


def test_host_data_that_would_be_distributed_is_refused(monkeypatch):
    """Above the shard threshold of a multi-rank job asarray() of host data
    gives a block-distributed array."""
    from macmetalpy_b200 import creation

    class DistArray:
        pass
    monkeypatch.setattr(creation, "asarray", lambda obj: DistArray())
    with pytest.raises(TypeError, match="distributed"):
        so.linear_recurrence(np.zeros((2, 5, 3)), np.zeros((2, 5, 3)))
    with pytest.raises(TypeError, match="distributed"):
        so.embedding(arr((4, 3)), [1, 2])
    with pytest.raises(TypeError, match="distributed"):
        so.global_norm([np.zeros(3)])
