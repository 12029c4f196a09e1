"""Calls of the hand-written kernels: replay of recorded launches, overlap of
outputs with inputs, arrays seen as rows.

An operator's function collects the arrays of a call (those that were given,
inputs before outputs) and first asks :func:`replay` for an earlier call with
the same signature (``_launch_plan``: types, shapes, strides, alignment,
device; never an address).  Otherwise a :class:`Call` checks and converts the
arrays, launches, and records what it launched.
"""
import functools
import struct

import numpy

from cupy_amd import _dryrun
from cupy_amd import _rt
from cupy_amd._core import _launch_plan
from cupy_amd._core import _tuning
from cupy_amd._core import internal
from cupy_amd._core._kernel import _check_peer_access
from cupy_amd._core._scalar import get_typename
from cupy_amd._core.core import ndarray, array as _array, ascontiguousarray, _byte_extent
from cupy_amd.cuda import compiler
from cupy_amd.cuda import device as _device
from cupy_amd.cuda import memory as _memory
from cupy_amd.cuda import stream as _stream

FLOATS = 'efd'

_float64 = numpy.dtype('float64')
_float32 = numpy.dtype('float32')


def acc_dtype(dtype):
    """Type sums over ``dtype`` are held in."""
    return _float64 if dtype == _float64 else _float32


# -- argument checks ------------------------------------------------------------------

def check_array(a, name):
    if not isinstance(a, ndarray):
        raise TypeError('%s must be a cupy.ndarray, got %s' % (name, type(a).__name__))


def check_float(a, name):
    check_array(a, name)
    if a.dtype.char not in FLOATS or not a.dtype.isnative:
        raise TypeError('%s must be of type float16, float32 or float64, got %s' % (name, a.dtype))


def check_out(out, shape, dtype, name='out'):
    """An output handed in has to be what the call would allocate."""
    check_array(out, name)
    if out._shape != tuple(shape):
        raise ValueError('%s has the wrong shape: %r, expected %r'
                         % (name, out._shape, tuple(shape)))
    if out.dtype != dtype:
        raise TypeError('%s has the wrong type: %s, expected %s' % (name, out.dtype, dtype))


def index_array(ids, name):
    """``ids`` as a device array of integers (host integers and lists are uploaded)."""
    if not isinstance(ids, ndarray):
        if not hasattr(ids, '__cuda_array_interface__'):
            ids = numpy.asarray(ids)
            if ids.size == 0 and ids.dtype.kind == 'f':
                ids = ids.astype(numpy.int64)
            if ids.dtype.kind not in 'iu':
                raise IndexError('%s must be of integer type, got %s' % (name, ids.dtype))
        ids = _array(ids, copy=False)
    if ids.dtype.kind not in 'iu':
        raise IndexError('%s must be of integer type, got %s' % (name, ids.dtype))
    return ids


def as_index(ids):
    """Integers the kernels read as they are: int32 or int64, stored in one piece."""
    if ids.dtype.char not in 'ilq':
        if ids.dtype.itemsize == 8:
            # uint64: what exceeds int64 is out of every range; its image as a
            # negative number is as well
            ids = ids.view(numpy.int64) if ids._c_contiguous else ids.copy('C').view(numpy.int64)
        else:
            ids = ids.astype(numpy.int64)
    return ascontiguousarray(ids)


# -- rows -----------------------------------------------------------------------------

def row_form(a):
    """(rows, elements between rows) of an array whose last axis is stored in
    one piece and whose other axes step evenly; None for any other layout."""
    shape, strides, item = a._shape, a._strides, a.dtype.itemsize
    width = shape[-1]
    if width > 1 and strides[-1] != item:
        return None
    rows, pitch = 1, None
    for n, st in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if n == 1:
            continue
        if pitch is None:
            if st % item:
                return None
            pitch = st
        elif st != pitch * rows:
            return None
        rows *= n
    return rows, (width if pitch is None else pitch // item)


def writable_rows(a):
    """True if the kernels can write the rows of ``a`` where they are."""
    form = row_form(a)
    return form is not None and (form[0] <= 1 or abs(form[1]) >= a._shape[-1])


# -- kernels --------------------------------------------------------------------------

class Source:
    """Kernels of one source text, compiled per set of definitions and device."""

    def __init__(self, text):
        self._text = text
        self._memo = {}

    def function(self, name, **defines):
        key = (_device.get_device_id(), name, tuple(defines.items()))
        fn = self._memo.get(key)
        if fn is None:
            head = ''.join('#define %s %s\n' % (k, _define(v)) for k, v in defines.items())
            fn = compiler.compile_with_cache(head + self._text).get_function(name)
            self._memo[key] = fn
        return fn


def _define(v):
    if isinstance(v, numpy.dtype):
        return get_typename(v)
    if isinstance(v, bool):
        return 'true' if v else 'false'
    return str(v)


class Ref:
    """Stands for the address of one of a call's arrays or temporaries."""
    __slots__ = ('index',)

    def __init__(self, index):
        self.index = index


# -- replay ---------------------------------------------------------------------------

_NOTHING = object()
_call = _rt.hot.call


def replay(plans, arrays, extra):
    """``(result, key)``: the result of a recorded call replayed on ``arrays``
    (``_NOTHING`` if there is none, the call has to be made in full), and the
    key to record it under (None: not to be recorded).

    A plan is ``(spans, record, ret, fast)``: which arrays may not overlap, the
    launches if addresses are all that changes in them and no result is allocated
    (made again by the extension module without a way back here), the
    positions of the results, the recorded call, and the temporaries if there
    are any."""
    r = _call(plans, arrays, _device.get_device_id(), _tuning._version, extra,
              _stream.get_current_stream_ptr())
    if type(r) is list:
        if len(r) == 1:
            return _NOTHING, r[0]
        return r[1][3].run(arrays), r[0]
    if r is None:
        return _NOTHING, None
    if type(r) is int:
        _rt.check(r)
    return r, None


def _temporary(nbytes):
    """Memory for a call that is made again; None under ``static_scratch``, where
    the call is replayed by its record."""
    if _memory._static_scratch_open and _memory.static_scratch_active():
        return None
    return _memory.alloc(nbytes)


def _span(a):
    lo, hi = _byte_extent(a._shape, a._strides, a.dtype.itemsize)
    return (lo, hi) if a.size else (0, 0)


def _pack_spans(arrays, pairs):
    return (struct.pack('<II', len(arrays), len(pairs))
            + b''.join(struct.pack('<qq', *_span(a)) for a in arrays)
            + b''.join(struct.pack('<II', a, b | (1 << 31 if same else 0))
                       for a, b, same in pairs))


class _Geometry:
    """An array's place in memory, for NumPy to look at and nobody to read."""

    def __init__(self, address, shape, strides, itemsize):
        self.__array_interface__ = {'version': 3, 'data': (address, True), 'shape': shape,
                                    'strides': strides, 'typestr': '|V%d' % itemsize}


@functools.lru_cache(maxsize=4096)
def _share(offset, a, b):
    base = 1 << 60                        # (no address: ``offset`` may be negative)
    try:
        return numpy.shares_memory(numpy.asarray(_Geometry(base, *a)),
                                   numpy.asarray(_Geometry(base + offset, *b)), max_work=1 << 20)
    except numpy.exceptions.TooHardError:
        return True


def share_elements(a, b):
    """Whether any byte belongs to elements of both arrays.  Column blocks of one
    matrix, or its odd and even rows, overlap as ranges of addresses and share
    nothing.  (A question too hard to answer counts as yes.)"""
    if not _rt.hot.overlap([a, b], _pack_spans([a, b], [(0, 1, False)])):
        return False
    return _share(b.data.ptr - a.data.ptr, (a._shape, a._strides, a.dtype.itemsize),
                  (b._shape, b._strides, b.dtype.itemsize))


class Call:
    """One call made in full.

    Args:
        plans, key: where to record it (key None: not recorded).
        arrays: the arrays the caller handed in, inputs before outputs.
        n_in: how many of them are inputs.
        in_place: (input, output) positions that may be the very same memory.
    """

    def __init__(self, plans, key, arrays, n_in, in_place=()):
        dev = _device.get_device_id()
        for a in arrays:
            _check_peer_access(a, dev)
        self.plans, self.key = plans, key
        self.user = list(arrays)
        self.refs = list(arrays)          # as the kernels see them
        self.n_in = n_in
        self.made = []                    # outputs allocated here
        self.temps = []
        self.copies = []                  # (stand-in, output to copy it to)
        self.rec = None
        self._pairs = pairs = []
        outs = range(n_in, len(arrays))
        for o in outs:
            for i in range(o):
                a, b = arrays[i], arrays[o]
                same = ((i, o) in in_place and a._shape == b._shape
                        and a._strides == b._strides and a.dtype == b.dtype)
                pairs.append((i, o, same))
        self._spans = _pack_spans(arrays, pairs) if pairs else None
        if self._spans is not None and _rt.hot.overlap(self.user, self._spans):
            self._separate()

    def _separate(self):
        """Inputs that share elements with an output are copied; outputs have to be
        apart."""
        self.key = None
        for pair in self._pairs:
            i, o, _ = pair
            a, b = self.user[i], self.user[o]
            if _rt.hot.overlap(self.user, _pack_spans(self.user, [pair])) and share_elements(a, b):
                if i >= self.n_in:
                    raise ValueError('two outputs of one call overlap in memory')
                self.refs[i] = a.copy()

    def convert(self, i, a):
        """The kernels are given ``a`` in the place of array ``i``."""
        if a is not self.refs[i]:
            self.refs[i] = a
            self.key = None

    def rows(self, i):
        """Elements between the rows of array ``i``, which is copied into one
        piece if it is not stored as rows."""
        a = self.refs[i]
        if i < self.n_in:
            form = row_form(a)
            if form is None:
                self.convert(i, ascontiguousarray(a))
                return a._shape[-1]
            return form[1]
        if not writable_rows(a):
            stand_in = ndarray._new_contiguous(a._shape, a.dtype)
            self.copies.append((stand_in, a))
            self.convert(i, stand_in)
            return a._shape[-1]
        return row_form(a)[1]

    def dense(self, i):
        """Array ``i`` has to be stored in one piece for the kernels."""
        a = self.refs[i]
        if a._c_contiguous:
            return
        if i < self.n_in:
            self.convert(i, ascontiguousarray(a))
        else:
            stand_in = ndarray._new_contiguous(a._shape, a.dtype)
            self.copies.append((stand_in, a))
            self.convert(i, stand_in)

    def allocate(self, shape, dtype):
        """Position of an output that the call allocates."""
        a = ndarray._new_contiguous(tuple(shape), numpy.dtype(dtype))
        self.made.append(a)
        self.refs.append(a)
        return len(self.refs) - 1

    def begin(self):
        """All arrays are known: launches from here on are recorded."""
        if self.key is not None:
            self.rec = _launch_plan.Recorder(len(self.refs))
        self.stream = _stream.get_current_stream_ptr()

    def temp(self, nbytes):
        """Position of a temporary of ``nbytes``."""
        mem = _memory.alloc(nbytes)
        self.temps.append(mem)
        if self.rec is not None:
            self.rec.temp(nbytes)
        return len(self.refs) + len(self.temps) - 1

    def launch(self, fn, grid, block, fmt, *values):
        """Launches ``fn``; ``fmt`` is a ``struct`` format, values of type Ref
        are addresses."""
        args = _launch_plan.ArgBlock()
        n = len(self.refs)
        for v in values:
            if type(v) is Ref:
                k = v.index
                args.ptr(k, self.refs[k].data.ptr if k < n else self.temps[k - n].ptr)
            else:
                args.const(v)
        _launch_plan.launch(self.rec, fn, grid, (block, 1, 1), _packer(fmt), args, self.stream)

    def finish(self, ret):
        """Records the call; returns the arrays at the positions ``ret`` (one,
        or a tuple)."""
        if self.copies:
            from cupy_amd._core._ufuncs import elementwise_copy
            for src, dst in self.copies:
                elementwise_copy(src, dst)
        if self.rec is not None and self.rec.launches:
            fast = _launch_plan.FastCall(
                len(self.user), [(a._shape, a.dtype) for a in self.made], self.rec, ret)
            direct = (not self.made and fast.quick is not None
                      and ret is not None and not _dryrun.enabled())
            plan = self._spans, fast.quick[0] if direct else None, ret, fast
            if direct and self.rec.temps:
                plan += ((_temporary, *self.rec.temps),)
            _launch_plan.remember(self.plans, self.key, plan)
        held = self.user + self.made
        if isinstance(ret, tuple):
            return tuple(held[r] for r in ret)
        return None if ret is None else held[ret]


_packers = {}


def _packer(fmt):
    p = _packers.get(fmt)
    if p is None:
        p = _packers[fmt] = struct.Struct('@' + fmt)
    return p


# -- geometry -------------------------------------------------------------------------

def compute_units():
    return _device.get_compute_units(_device.get_device_id())


def clp2(n):
    return internal.clp2(n)


def stream_hints(nbytes_in, nbytes_out):
    return _tuning.stream_policy('auto', nbytes_in, nbytes_out)
