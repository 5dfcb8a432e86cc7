"""Operators of sequence models, beside the array operations they extend.

* :func:`linear_recurrence` is ``cumsum`` with a decay (``reductions.py:661-681``
  has the plain sum): ``h_t = f_t h_{t-1} + u_t`` along an axis, with its
  gradient :func:`linear_recurrence_grad`;
* :func:`embedding` is ``take`` of rows with a scale (``indexing.py:24-60``), with
  the gradient of the table :func:`embedding_grad`;
* :func:`global_norm` and :func:`clip_by_global_norm` are the norm over a list of
  arrays and ``clip`` by it.

They take float16, float32 and float64 arrays.  States, sums and norms are held
in float32 or more whatever the arrays' dtype, and every output is rounded once.
Everything runs on the library stream and is asynchronous, like every other
operation of this package.  ``out=`` arrays are written in place; results are
the same bits for equal calls.
"""

from __future__ import annotations

import array
import bisect
import itertools
import math
import operator

import numpy as np

from . import _cuda_backend as _cb
from ._dtypes import MMP_CODES, resolve_dtype
from .ndarray import _c_contiguous_strides, ndarray

__all__ = ["linear_recurrence", "linear_recurrence_grad", "embedding", "embedding_grad", "global_norm",
           "clip_by_global_norm"]

_F32, _F64 = np.dtype(np.float32), np.dtype(np.float64)
_I32, _I64 = np.dtype(np.int32), np.dtype(np.int64)


def _arr(x, what: str) -> ndarray:
    if x.__class__ is ndarray:
        return x
    if x.__class__.__name__ != "DistArray":
        from .creation import asarray
        x = asarray(x)  # of host data on a multi-rank job, this too can be block-distributed
        if x.__class__.__name__ != "DistArray":
            return x
    raise TypeError(f"{what}: block-distributed arrays are not supported")


def _floating(dt, what: str):
    if dt.kind != "f":
        raise TypeError(f"{what} needs floating-point arrays, got {dt}")
    return dt


def _cast(a: ndarray, dt) -> ndarray:
    return a if a._dtype == dt else a.astype(dt)


def _check_out(out, shape, dt, what: str, name: str = "out"):
    if out.__class__ is not ndarray:
        raise TypeError(f"{what}: {name} must be an array of this package, got {type(out).__name__}")
    if out._shape != shape or out._dtype != dt:
        raise ValueError(f"{what}: {name} has shape {out._shape} and dtype {out._dtype}, needs {shape} and {dt}")
    out._materialize_if_lazy()


def _span(a: ndarray):
    """First and last byte address of the array's elements (end exclusive)."""
    lo = hi = 0
    for n, s in zip(a._shape, a._strides):
        if s < 0:
            lo += (n - 1) * s
        else:
            hi += (n - 1) * s
    e = a._dtype.itemsize
    p = a._ptr
    return p + lo * e, p + (hi + 1) * e


def _overlap(a: ndarray, b: ndarray) -> bool:
    if a._buffer is not b._buffer or a.size == 0 or b.size == 0:  # a buffer is one allocation
        return False
    a0, a1 = _span(a)
    b0, b1 = _span(b)
    return a0 < b1 and b0 < a1


def _same(a: ndarray, b: ndarray) -> bool:
    """The very same elements in the same places."""
    return a._ptr == b._ptr and a._shape == b._shape and a._strides == b._strides and a._dtype == b._dtype


# ------------------------------------------------------------------ recurrence

def _split(shape, axis):
    if len(shape) == 3 and axis == 1:
        return shape
    return math.prod(shape[:axis]), shape[axis], math.prod(shape[axis + 1:])


def _strides3(a: ndarray, axis: int):
    """(outer, step) element strides of ``a`` seen as (outer, steps, inner)
    with inner contiguous, or None if no such strides exist."""
    shape, st = a._shape, a._strides
    if len(shape) == 3 and axis == 1 and (st[2] == 1 or shape[2] == 1):  # (batch, steps, width)
        return (st[0] if shape[0] != 1 else 0), st[1]
    run = 1
    for n, s in zip(reversed(shape[axis + 1:]), reversed(st[axis + 1:])):
        if n != 1 and s != run:
            return None
        run *= n
    so = 0
    last = None  # (size, stride) of the last axis of more than one entry
    for n, s in zip(reversed(shape[:axis]), reversed(st[:axis])):
        if n == 1:
            continue
        if last is None:
            so = s
        elif s != last[0] * last[1]:
            return None
        last = (n, s)
    return so, st[axis]


def _view3(a: ndarray, axis: int):
    """(array, outer stride, step stride), of a contiguous copy where needed."""
    a._materialize_if_lazy()
    r = _strides3(a, axis)
    if r is None:
        a = a._contiguous_copy()
        r = _strides3(a, axis)
    return a, r[0], r[1]


def _out3(out, shape, dt, axis, what, name, inputs, same_ok):
    """The array the kernel writes for ``out`` (a new one where ``out`` is None,
    has no fitting strides or overlaps an input it may not), with its strides."""
    if out is not None:
        _check_out(out, shape, dt, what, name)
        r = _strides3(out, axis)
        ok = r is not None and (0 not in out._strides or all(s != 0 or n <= 1
                                                             for n, s in zip(out._shape, out._strides)))
        if ok:
            for b, same in zip(inputs, same_ok):
                if out._buffer is b._buffer and _overlap(out, b) and not (same and _same(out, b)):
                    break
            else:
                return out, r[0], r[1]
    new = ndarray._empty(shape, dt)
    so, st = _strides3(new, axis)
    return new, so, st


def _axis(axis, ndim, what):
    if ndim == 0:
        raise ValueError(f"{what} needs at least one axis")
    axis = int(axis)
    if not -ndim <= axis < ndim:
        raise np.exceptions.AxisError(axis, ndim)
    return axis % ndim


def _state(s, shape, dt, what, name):
    """A contiguous state array in ``dt``."""
    s = _arr(s, what)
    if s._shape != shape:
        raise ValueError(f"{what}: {name} has shape {s._shape}, needs {shape}")
    if s._dtype != dt:
        _floating(s._dtype, what)
        s = s.astype(dt)
    return s if s._buffer is not None and s._strides == _c_contiguous_strides(shape) else s._ensure_contiguous()


def _p(a):
    return None if a is None else a._ptr


def linear_recurrence(a, x, h0=None, *, axis=-2, gated=False, out=None, state_out=None):
    """First-order linear recurrence along ``axis``: ``h_t = f_t * h_{t-1} + u_t``.

    ``gated=False``: ``f = a`` and ``u = x`` (``a = 1`` is ``cumsum``).
    ``gated=True``: ``a`` holds logits, ``f = sigmoid(a)`` and ``u = (1 - f) * x``;
    a logit of ``+inf`` (a padded step) keeps the state as it is, one of
    ``-inf`` (the first step of the next sequence in a packed row) replaces it,
    both exactly, where ``x`` and the state are finite.  The products are made:
    an infinity or NaN in a padded step's ``x`` (``where`` puts zeros there) or in
    the state before a new sequence gives NaN, as ``0 * inf`` is, and what is NaN
    stays so to the end of its row.

    ``a`` and ``x`` have one shape, ``(..., steps, ...)``; the default axis is that
    of ``(batch, steps, width)``.  Slices of one larger array are read in place.
    ``h0`` (zeros if None) is the state before the first step, of the shape
    without ``axis``.  The state is float32 (float64 for float64 arrays) whatever
    the arrays' dtype: ``state_out``, an array of that dtype, receives the state
    after the last step, and may be ``h0`` itself, so a loop over tokens or
    segments carries it without a rounding in between::

        s = cp.zeros((batch, width), dtype="float32")
        for ...:
            h = cp.linear_recurrence(gate, x, s, gated=True, state_out=s)

    Decays are multiplied over up to 112 steps in the state's dtype; where they are
    larger than 1 and that product overflows, the result does too, unless the
    state before those steps is zero; where it underflows to zero, an infinite
    state before them becomes NaN.

    Returns ``h``, of the shape and dtype of ``a`` and ``x`` (promoted together);
    it is written to ``out`` if that is given (``out`` may be ``a`` or ``x``).
    """
    what = "linear_recurrence"
    a, x = _arr(a, what), _arr(x, what)
    if a._shape != x._shape:
        raise ValueError(f"{what}: a has shape {a._shape} and x {x._shape} (broadcast_to makes them alike)")
    shape = x._shape
    axis = _axis(axis, len(shape), what)
    dt = a._dtype
    if x._dtype != dt:
        dt = resolve_dtype(np.result_type(dt, x._dtype))
        a, x = _cast(a, dt), _cast(x, dt)
    _floating(dt, what)
    sdt = _F64 if dt == _F64 else _F32
    outer, steps, inner = _split(shape, axis)
    sshape = shape[:axis] + shape[axis + 1:]
    if h0 is not None:
        h0 = _state(h0, sshape, sdt, what, "h0")
    a, a_so, a_st = _view3(a, axis)
    x, x_so, x_st = _view3(x, axis)
    inputs = (a, x) if h0 is None else (a, x, h0)
    h, h_so, h_st = _out3(out, shape, dt, axis, what, "out", inputs, (True, True, False))
    state = None
    if state_out is not None:
        _check_out(state_out, sshape, sdt, what, "state_out")
        state = state_out
        buf = state._buffer
        if state._strides != _c_contiguous_strides(sshape) or (
                (buf is a._buffer or buf is x._buffer or buf is h._buffer)
                and any(_overlap(state, b) for b in (a, x, h))) or (
                h0 is not None and _overlap(state, h0) and not _same(state, h0)):
            state = ndarray._empty(sshape, sdt)
    _cb.check(_cb.lib.mmp_recurrence(MMP_CODES[dt], bool(gated), outer, steps, inner, a._ptr, a_so, a_st, x._ptr,
                                     x_so, x_st, _p(h0), h._ptr, h_so, h_st, _p(state)), what)
    if state is not state_out:
        state_out[...] = state
    if out is None or h is out:
        return h
    out[...] = h
    return out


def linear_recurrence_grad(a, x, h, grad, h0=None, *, axis=-2, gated=False, grad_state=None, out=None):
    """Gradients of :func:`linear_recurrence` with respect to ``a``, ``x`` and ``h0``.

    ``a``, ``x``, ``h0`` are the inputs and ``h`` the output of that call; ``grad``
    is the gradient with respect to ``h``, and ``grad_state`` (zeros if None) the
    one with respect to the state after the last step, for a sequence that went
    on in another call.  With ``gated=False``, ``x`` is not read and may be None.

    Returns ``(grad_a, grad_x, grad_h0)``: the first two in the arrays' shape and
    dtype (for a broadcast view, sum them over its broadcast axes), the last in
    the state's dtype, or None where ``h0`` is None.  ``out``, a
    tuple of two or three arrays, receives them (the first two may be ``a``,
    ``x`` or ``grad`` themselves, not one another).
    """
    what = "linear_recurrence_grad"
    gated = bool(gated)
    a, h, grad = _arr(a, what), _arr(h, what), _arr(grad, what)
    if x is None:
        if gated:
            raise ValueError(f"{what}: x is needed with gated=True")
    else:
        x = _arr(x, what)
    ops = [a, h, grad] if x is None else [a, h, grad, x]
    shape = a._shape
    for o in ops:
        if o._shape != shape:
            raise ValueError(f"{what}: shapes {', '.join(str(q._shape) for q in ops)} of a, h, grad"
                             f"{'' if x is None else ', x'} differ")
    axis = _axis(axis, len(shape), what)
    if not gated:  # nor has it a part in the dtype
        x, ops = None, ops[:3]
    dt = a._dtype
    if any(o._dtype != dt for o in ops):
        dt = resolve_dtype(np.result_type(*[o._dtype for o in ops]))
    _floating(dt, what)
    sdt = _F64 if dt == _F64 else _F32
    outer, steps, inner = _split(shape, axis)
    sshape = shape[:axis] + shape[axis + 1:]
    if h0 is not None:
        h0 = _state(h0, sshape, sdt, what, "h0")
    if grad_state is not None:
        grad_state = _state(grad_state, sshape, sdt, what, "grad_state")
    a, a_so, a_st = _view3(_cast(a, dt), axis)
    h, h_so, h_st = _view3(_cast(h, dt), axis)
    grad, g_so, g_st = _view3(_cast(grad, dt), axis)
    x_so = x_st = 0
    if gated:
        x, x_so, x_st = _view3(_cast(x, dt), axis)
    want = 3 if h0 is not None else 2
    if out is None:
        out = (None,) * want
    elif not isinstance(out, (tuple, list)) or len(out) != want:
        raise ValueError(f"{what}: out must be a tuple of {want} arrays")
    inputs = [a, grad] + ([x] if gated else []) + [h] + [s for s in (h0, grad_state) if s is not None]
    same_ok = [True, True] + ([True] if gated else []) + [False] * 3
    ga, ga_so, ga_st = _out3(out[0], shape, dt, axis, what, "out[0]", inputs, same_ok)
    gx, gx_so, gx_st = _out3(out[1], shape, dt, axis, what, "out[1]", inputs + [ga], same_ok[:len(inputs)] + [False])
    gh0 = None
    if want == 3:
        gh0 = out[2]
        if gh0 is not None:
            _check_out(gh0, sshape, sdt, what, "out[2]")
            if not gh0._is_c_contiguous() or any(_overlap(gh0, b) and not (b is grad_state and _same(gh0, b))
                                                 for b in inputs + [ga, gx]):
                gh0 = None
        if gh0 is None:
            gh0 = ndarray._empty(sshape, sdt)
    _cb.check(_cb.lib.mmp_recurrence_grad(MMP_CODES[dt], gated, outer, steps, inner, a._ptr, a_so, a_st, _p(x), x_so,
                                          x_st, h._ptr, h_so, h_st, grad._ptr, g_so, g_st, _p(h0), _p(grad_state),
                                          ga._ptr, ga_so, ga_st, gx._ptr, gx_so, gx_st, _p(gh0)), what)
    res = []
    for o, r in zip(out, (ga, gx, gh0)):
        if o is not None and o is not r:
            o[...] = r
            r = o
        res.append(r)
    return res[0], res[1], res[2] if want == 3 else None


# ------------------------------------------------------------------ embedding

def _token_ids(ids, what) -> ndarray:
    ids = _arr(ids, what)
    if ids._dtype.kind not in "iu":
        raise TypeError(f"{what}: ids must be integers, got {ids._dtype}")
    if ids._dtype != _I32 and ids._dtype != _I64:
        ids = ids.astype(_I64)
    return ids._ensure_contiguous()


def _rows2(a: ndarray, width: int):
    """(array, row stride) of an array seen as rows of ``width`` contiguous
    elements an even stride apart, of a contiguous copy where needed."""
    a._materialize_if_lazy()
    r = _strides3(a, a.ndim - 1) if a.ndim > 1 else (0, 1)
    if r is None or (width > 1 and a._strides[-1] != 1):
        a = a._contiguous_copy()
        return a, width
    return a, r[0]


def embedding(weight, ids, scale=1.0, *, out=None):
    """Rows of a table by token id, times ``scale``: ``weight[ids] * scale``.

    ``weight`` is ``(rows, width)`` (a slice of a larger table is read in place),
    ``ids`` integers of any shape; the result has the shape ``ids.shape +
    (width,)`` and the table's dtype, the product rounded once.  Ids are in
    ``[0, rows)``: they are not checked on the host (``take`` does, and waits for
    the device).  One outside gives a row of zeros, and the next
    ``synchronize()`` raises.
    """
    what = "embedding"
    weight, ids = _arr(weight, what), _token_ids(ids, what)
    if weight.ndim != 2:
        raise ValueError(f"{what}: weight must be 2-D (rows, width), got shape {weight._shape}")
    dt = _floating(weight._dtype, what)
    rows, width = weight._shape
    scale = float(scale)
    weight, stride = _rows2(weight, width)
    shape = ids._shape + (width,)
    res = out
    if out is not None:
        _check_out(out, shape, dt, what)
        if not out._is_c_contiguous() or _overlap(out, weight) or _overlap(out, ids):
            res = None
    if res is None:
        res = ndarray._empty(shape, dt)
    _cb.check(_cb.lib.mmp_embedding(MMP_CODES[dt], weight._ptr, rows, width, stride, MMP_CODES[ids._dtype], ids._ptr,
                                    ids.size, scale, res._ptr), what)
    if out is None or res is out:
        return res
    out[...] = res
    return out


def embedding_grad(ids, grad, num_rows, scale=1.0, *, padding_idx=None, out=None):
    """Gradient of :func:`embedding` with respect to its table.

    ``grad`` is the gradient of the result, ``ids.shape + (width,)``.  Returns the
    whole ``(num_rows, width)`` gradient in ``grad``'s dtype: row ``v`` is ``scale``
    times the sum of ``grad`` over the tokens whose id is ``v``, zeros where there
    is none and for ``padding_idx``.  The sums are float32 (float64 for float64),
    in an order that the ids alone decide: equal calls give equal bits.  An id
    outside ``[0, num_rows)`` adds nothing, and the next ``synchronize()`` raises.
    """
    what = "embedding_grad"
    ids, grad = _token_ids(ids, what), _arr(grad, what)
    dt = _floating(grad._dtype, what)
    if grad._shape[:-1] != ids._shape or grad.ndim != ids.ndim + 1:
        raise ValueError(f"{what}: grad has shape {grad._shape}, needs {ids._shape + ('width',)}")
    rows, width = int(num_rows), grad._shape[-1]
    if rows < 0:
        raise ValueError(f"{what}: num_rows must not be negative, got {rows}")
    pad = -1
    if padding_idx is not None:
        pad = int(padding_idx)
        if not -rows <= pad < rows:
            raise IndexError(f"{what}: padding_idx {pad} is out of bounds for {rows} rows")
        pad %= rows
    scale = float(scale)
    grad, stride = _rows2(grad, width)
    res = out
    if out is not None:
        _check_out(out, (rows, width), dt, what)
        if not out._is_c_contiguous() or _overlap(out, grad) or _overlap(out, ids):
            res = None
    if res is None:
        res = ndarray._empty((rows, width), dt)
    _cb.check(_cb.lib.mmp_embedding_grad(MMP_CODES[dt], MMP_CODES[ids._dtype], ids._ptr, ids.size, grad._ptr, stride,
                                         rows, width, scale, pad, res._ptr), what)
    if out is None or res is out:
        return res
    out[...] = res
    return out


# ------------------------------------------------------------------ global norm

_LAYOUT = operator.attrgetter("_buffer", "_offset", "_shape", "_strides", "_dtype")
_PTR = operator.attrgetter("ptr")
_KIND = {np.dtype(t): (MMP_CODES[np.dtype(t)], np.dtype(t).itemsize) for t in (np.float16, np.float32, np.float64)}


class _Shapes(dict):
    """shape -> (C-contiguous strides, size)."""

    def __missing__(self, shape):
        r = (_c_contiguous_strides(shape), math.prod(shape))
        if len(self) < 4096:
            self[shape] = r
        return r


_SHAPES = _Shapes()


class _Listed:
    """A list of C-contiguous floating arrays as the library takes it: addresses,
    sizes and dtype codes.  Gradients come by the hundred, and a few attribute
    reads an array are what the host may spend on each (some 0.3 us; checks one
    by one took 2.5); so whatever does not fit at once is left to `of_any`."""

    __slots__ = ("arrays", "shapes", "dtypes", "codes", "sizes", "ptrs", "ends")

    @classmethod
    def of(cls, arrays):
        """None if one of the arrays is lazy, strided or not an array of floats."""
        if not arrays or set(map(type, arrays)) != {ndarray}:
            return None
        bufs, offs, shapes, strides, dts = zip(*map(_LAYOUT, arrays))
        kinds = list(map(_KIND.get, dts))
        if None in bufs or None in kinds:  # lazy, not floating
            return None
        want, sizes = zip(*map(_SHAPES.__getitem__, shapes))
        if strides != want:
            return None
        codes, items = zip(*kinds)
        r = cls()
        r.arrays, r.shapes, r.dtypes = arrays, shapes, dts
        r.codes, r.sizes = array.array("i", codes), array.array("q", sizes)
        r.ptrs = list(map(_PTR, bufs))
        if any(offs):
            r.ptrs = list(map(operator.add, r.ptrs, map(operator.mul, offs, items)))
        r.ends = list(map(operator.add, r.ptrs, map(operator.mul, sizes, items)))
        return r

    @classmethod
    def of_any(cls, arrays, what):
        arrays = [_arr(a, what) for a in arrays]
        for a in arrays:
            _floating(a._dtype, what)
        arrays = [a._ensure_contiguous() for a in arrays]
        for i, a in enumerate(arrays):
            if a._strides != _c_contiguous_strides(a._shape):  # axes of one entry: the same memory
                arrays[i] = a._view(a._shape, _c_contiguous_strides(a._shape), a._offset)
        r = cls.of(arrays)
        if r is None:
            r = cls()
            r.arrays, r.shapes, r.dtypes, r.ptrs, r.ends = [], (), (), [], []
            r.codes, r.sizes = array.array("i"), array.array("q")
        return r


def _apart(lists, norm_out):
    """Whether no two arrays of the lists, and the norm's, share memory: then, and
    only then, the sorted ends each lie before the next of the sorted starts."""
    starts, ends = [], []
    for r in lists:
        starts += r.ptrs
        ends += r.ends
    if norm_out is not None:
        p = norm_out._ptr
        starts.append(p)
        ends.append(p + norm_out._dtype.itemsize)
    starts.sort()
    ends.sort()
    return all(map(operator.le, ends, itertools.islice(starts, 1, None)))


def _norm_call(src, dst, max_norm, norm_out, what, name, apart=False):
    """The norm of the arrays of `src`, and with `dst` the clipped arrays
    (`apart`: the norm's array is known to overlap none)."""
    ndt = _F64 if _F64 in src.dtypes else _F32
    if norm_out is not None:
        _check_out(norm_out, (), ndt, what, name)
        p = norm_out._ptr
        for r in () if apart else (src, dst) if dst is not None else (src,):
            if any(a < p + ndt.itemsize and p < b for a, b in zip(r.ptrs, r.ends)):
                raise ValueError(f"{what}: {name} overlaps one of the arrays")
        norm = norm_out
    else:
        norm = ndarray._empty0(ndt)
    x = array.array("q", src.ptrs)
    y = None if dst is None else array.array("q", dst.ptrs)
    _cb.check(_cb.lib.mmp_global_norm(len(src.codes), src.codes.buffer_info()[0], x.buffer_info()[0],
                                      None if y is None else y.buffer_info()[0], src.sizes.buffer_info()[0], max_norm,
                                      MMP_CODES[ndt], norm._ptr), what)
    return norm


def _norm_list(arrays, what):
    if not isinstance(arrays, (list, tuple)):
        raise TypeError(f"{what} takes a list of arrays, got {type(arrays).__name__}")
    return _Listed.of(arrays) or _Listed.of_any(arrays, what)


def global_norm(arrays, *, out=None):
    """Euclidean norm over all elements of a list of arrays, as one 0-d array.

    ``sqrt(sum(sum(x * x) for x in arrays))`` for arrays of any shapes and
    floating dtypes, summed in float64 (where squares of float64 elements
    beyond 1e154 are infinite); float32, or float64 if one of the arrays is.
    An empty list has norm 0.
    """
    what = "global_norm"
    return _norm_call(_norm_list(arrays, what), None, 0.0, out, what, "out")


def clip_by_global_norm(arrays, max_norm, *, out=None, norm_out=None):
    """Scale a list of arrays so that their :func:`global_norm` is at most ``max_norm``.

    Every array is multiplied by ``1`` if the norm is at most ``max_norm``, else by
    ``max_norm / norm``.  An infinite norm therefore gives zeros, and NaN where an
    element is infinite; a NaN norm gives NaN everywhere.

    Returns ``(clipped, norm)``: a list of arrays of the same shapes and dtypes, and
    the norm before clipping, as :func:`global_norm` returns it (nothing waits for
    the device).  ``out``, a list of arrays, receives the clipped ones; pass the
    list itself to clip in place, where nothing is written if nothing is to be
    scaled.  ``norm_out`` receives the norm.
    """
    what = "clip_by_global_norm"
    src = _norm_list(arrays, what)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"{what}: max_norm must be >= 0, got {max_norm}")
    if out is None:
        res = [ndarray._empty(s, d) for s, d in zip(src.shapes, src.dtypes)]
        dst = _Listed.of(res) or _Listed.of_any(res, what)
        return res, _norm_call(src, dst, max_norm, norm_out, what, "norm_out")
    if not isinstance(out, (list, tuple)) or len(out) != len(src.codes):
        raise ValueError(f"{what}: out must be a list of {len(src.codes)} arrays")
    res = list(out)
    # the usual cases: the arrays themselves, or others that are all apart
    if out is arrays and src.arrays is arrays:
        if _apart((src,), norm_out if norm_out.__class__ is ndarray else None):
            return res, _norm_call(src, src, max_norm, norm_out, what, "norm_out", True)
    else:
        dst = _Listed.of(res)
        if dst is not None and dst.shapes == src.shapes and dst.dtypes == src.dtypes:
            same = dst.ptrs == src.ptrs
            if _apart((src,) if same else (src, dst), norm_out if norm_out.__class__ is ndarray else None):
                return res, _norm_call(src, dst, max_norm, norm_out, what, "norm_out", True)
    for o, s, d in zip(res, src.shapes, src.dtypes):
        _check_out(o, s, d, what)
    outs = list(res)
    _norm_outs(outs, src.arrays)
    norm = _norm_call(src, _Listed.of_any(outs, what), max_norm, norm_out, what, "norm_out")
    for o, r in zip(outs, res):
        if o is not r:
            r[...] = o
    return res, norm


def _norm_outs(outs, srcs):
    """Replace by temporaries the outputs that the kernel cannot write directly:
    not contiguous, overlapping an input other than by being it (an array that
    is listed twice among them), or overlapping an output before them."""
    spans = sorted((_span(a) + (i,) for i, a in enumerate(srcs) if a.size), key=lambda s: s[0])
    starts = [s[0] for s in spans]
    reach, top = [], 0  # furthest end of the inputs up to each
    for s in spans:
        top = max(top, s[1])
        reach.append(top)
    mine = []
    for i, o in enumerate(outs):
        if o.size == 0:
            continue
        lo, hi = _span(o)
        ok = o._is_c_contiguous()
        if ok:
            k = bisect.bisect_left(starts, hi)  # inputs that start before this output ends
            if k and reach[k - 1] > lo:
                ok = [s[2] for s in spans[:k] if s[1] > lo] == [i] and _same(o, srcs[i])
        if ok:
            mine.append((lo, hi, i))
        else:
            outs[i] = ndarray._empty(o._shape, o._dtype)
    end = 0
    for lo, hi, i in sorted(mine):
        if lo < end:
            outs[i] = ndarray._empty(outs[i]._shape, outs[i]._dtype)
        else:
            end = hi
