"""Norm of many arrays taken together, and scaling them down to a bound on it.

``global_norm`` is the square root of the sum of the squares of all elements of
all arrays; ``clip_by_global_norm`` multiplies every array by
``min(1, max_norm / (norm + eps))``.  The arrays are described by tables in the
argument block (up to 100 to a launch), so that a model's hundreds of gradients
take a few launches: the squares are summed per piece of 32 KiB, a single
workgroup joins the pieces' sums in order and derives the factor, and the
scaling reads it from device memory: nothing waits for the host.
"""
import struct

import numpy

from cupy_amd import _rt
from cupy_amd._core import _op_calls as _oc
from cupy_amd._core._kernel import _check_peer_access
from cupy_amd._core._ufuncs import elementwise_copy
from cupy_amd._core.core import ndarray, _byte_extent
from cupy_amd.cuda import device as _device
from cupy_amd.cuda import memory as _memory
from cupy_amd.cuda import stream as _stream

_MAX = 100                  # arrays to a launch: 3200 bytes of its 4 KiB of arguments
_BLOCK = 256
_UNROLL = 8                 # vectors of 16 bytes per thread
_ENTRY = numpy.dtype([('src', 'u8'), ('dst', 'u8'), ('n', 'u8'), ('first', 'u4'), ('pad', 'u4')])
_TYPES = [numpy.dtype(c) for c in _oc.FLOATS]
_SIZES = numpy.array([t.itemsize for t in _TYPES])
# what the extension module says of an array: address, elements, position of its
# type in _TYPES, 1 if stored in C order plus 2 if in Fortran order, device
_DESCRIPTION = numpy.dtype([('ptr', 'u8'), ('n', 'u8'), ('type', 'u4'), ('dense', 'u4'),
                            ('device', 'i8')])

_SOURCE = _oc.Source(r'''
#include <cupy/rows.cuh>
typedef cupy::acc_of<X_T>::type A;

struct Entry {
  const X_T* src;
  X_T* dst;
  unsigned long long n;
  unsigned int first;       // the array's first workgroup
  unsigned int pad;
};
struct Table { Entry e[MAX_ENTRIES]; };

// The array a workgroup works on: the last one that begins at or before it,
// found by every wave in one step, a lane per array (a search by halves is a
// chain of seven loads).
_CUPY_DEV int entry_of(const Table& t, int n, unsigned int block) {
  const int lane = threadIdx.x & 63;
  int found = 0;
#pragma unroll
  for (int base = 0; base < MAX_ENTRIES; base += 64) {
    const int at = base + lane < MAX_ENTRIES ? base + lane : MAX_ENTRIES - 1;
    found += __popcll(__ballot(base + lane < n && t.e[at].first <= block));
  }
  return __builtin_amdgcn_readfirstlane(found - 1);
}

// Vectors on 16-byte borders of the source, whatever the array starts on.  A
// piece that lies inside its array is loaded without a question between the
// requests.
struct Piece {
  long long c0;      // the thread's first element
  long long n;
  bool inside;
  cupy::Vec<X_T, VEC> v[UNROLL];
  _CUPY_DEV long long column(int k) const { return c0 + (long long)k * BLOCK * VEC; }
  _CUPY_DEV void load(const Entry& e, unsigned int block) {
    const int phase = (int)((reinterpret_cast<unsigned long long>(e.src) & 15) / sizeof(X_T));
    n = (long long)e.n;
    const long long first = (long long)block * UNROLL * BLOCK * VEC - phase;
    inside = first >= 0 && first + UNROLL * BLOCK * VEC <= n;
    c0 = first + threadIdx.x * VEC;
    if (inside) {
#pragma unroll
      for (int k = 0; k < UNROLL; ++k) v[k] = cupy::load_vec<X_T, VEC, NT_IN>(e.src + column(k));
    } else {
#pragma unroll
      for (int k = 0; k < UNROLL; ++k) {
        const long long c = column(k);
        if (c >= 0 && c + VEC <= n) {
          v[k] = cupy::load_vec<X_T, VEC, NT_IN>(e.src + c);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            v[k].v[i] = c + i >= 0 && c + i < n ? e.src[c + i] : static_cast<X_T>(0.0f);
        }
      }
    }
  }
  _CUPY_DEV void store(X_T* to, int k, const cupy::Vec<X_T, VEC>& r) const {
    const long long c = column(k);
    if (inside || (c >= 0 && c + VEC <= n)) {
      cupy::store_vec<X_T, VEC, NT_OUT>(to + c, r);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (c + i >= 0 && c + i < n) to[c + i] = r.v[i];
    }
  }
};

struct Add {
  template <typename T> _CUPY_DEV T operator()(T a, T b) const { return a + b; }
};

// float16: 64 squares, at most 2^32 each, are added in 32 bits, the rest in 64.
// float32: the squares are taken in 64 bits, where none over- or underflows.
// Bound by memory: 145 arrays, 604 MB of float16, 102 us in two launches, 5.9 TB/s.
extern "C" __global__ void __launch_bounds__(BLOCK)
cupy_square_sums(const Table t, const int entries, double* temp, const long long at) {
  __shared__ double lds[BLOCK / 64];
  const int k = entry_of(t, entries, blockIdx.x);
  const Entry e = t.e[k];
  Piece p;
  p.load(e, blockIdx.x - e.first);
  double total;
  if (sizeof(X_T) == 2) {
    float s = 0.0f;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float x = static_cast<float>(p.v[u].v[i]);
        s = __builtin_fmaf(x, x, s);
      }
    total = s;
  } else {
    total = 0.0;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const double x = static_cast<double>(static_cast<A>(p.v[u].v[i]));
        total = __builtin_fma(x, x, total);
      }
  }
  total = cupy::row_allreduce<BLOCK, BLOCK>(total, Add(), lds);
  if (threadIdx.x == 0) temp[at + blockIdx.x] = total;
}

// What elements are multiplied by.  float32: the product is taken in 64 bits, for a
// factor may lie below the range of float32 where its product with them does not (a
// norm of 1e40 scaled to 1), and is rounded once.  float16: any factor that a
// float32 cannot hold takes all of them to 0.
template <typename T> struct factor_of { typedef double type; };
template <> struct factor_of<float16> { typedef float type; };

// Bound by memory: the same arrays, 198 us in two launches, 6.1 TB/s.
extern "C" __global__ void __launch_bounds__(BLOCK)
cupy_scale_arrays(const Table t, const int entries, const int blocks, const double* temp) {
  // last pieces first: they are what the sums have left in the cache
  const unsigned int block = blocks - 1 - blockIdx.x;
  const Entry e = t.e[entry_of(t, entries, block)];
  typedef factor_of<X_T>::type F;
  const F factor = static_cast<F>(temp[0]);
  if (factor == F(1) && e.src == e.dst) return;       // what is there is the result
  Piece p;
  p.load(e, block - e.first);
#pragma unroll
  for (int k = 0; k < UNROLL; ++k) {
    cupy::Vec<X_T, VEC> r;
#pragma unroll
    for (int i = 0; i < VEC; ++i) r.v[i] = static_cast<X_T>(static_cast<F>(p.v[k].v[i]) * factor);
    p.store(e.dst, k, r);
  }
}
''')

_FINISH = _oc.Source(r'''
#include <cupy/rows.cuh>
struct Add {
  template <typename T> _CUPY_DEV T operator()(T a, T b) const { return a + b; }
};
// One workgroup: every thread a run of the sums, which follow the place of the
// factor, the threads by a tree.
extern "C" __global__ void __launch_bounds__(1024)
cupy_norm_of_sums(double* temp, const long long n, N_T* norm, const double max_norm,
                  const double eps) {
  __shared__ double lds[16];
  const double* sums = temp + 1;
  double t = 0.0;
  for (long long i = threadIdx.x; i < n; i += 8 * 1024) {
    double v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = sums[i + 1024 * k < n ? i + 1024 * k : i];
#pragma unroll
    for (int k = 0; k < 8; ++k) if (i + 1024 * k < n) t += v[k];
  }
  t = cupy::row_allreduce<1024, 1024>(t, Add(), lds);
  if (threadIdx.x == 0) {
    const double r = __builtin_sqrt(t);
    *norm = static_cast<N_T>(r);
    // (compared before the division: 0 / 0 and inf / inf leave the arrays as they
    // are; the factor of a NaN is one)
    temp[0] = max_norm >= r + eps ? 1.0 : max_norm / (r + eps);
  }
}
''')


def _describe(arrays, name):
    """Addresses, sizes, types and layouts of a list of arrays, checked."""
    d = numpy.frombuffer(_rt.hot.describe(arrays, _TYPES), _DESCRIPTION)
    if len(d):
        if d['type'].max() >= len(_TYPES):
            for a in arrays:
                _oc.check_float(a, name)
        dev = _device.get_device_id()
        if (d['device'] != dev).any():
            for a in arrays:
                _check_peer_access(a, dev)
    return d


def _ranges(arrays, d):
    """First and one-past-last address that each array touches (0 and 0 where it
    has no elements: such arrays overlap nothing)."""
    start = d['ptr'].astype(numpy.int64)
    end = start + d['n'].astype(numpy.int64) * _SIZES[d['type']]
    for i in numpy.flatnonzero(d['dense'] == 0):
        lo, hi = _byte_extent(arrays[i]._shape, arrays[i]._strides, arrays[i].dtype.itemsize)
        start[i], end[i] = start[i] + lo, start[i] + hi
    start[d['n'] == 0] = end[d['n'] == 0] = 0
    return start, end


def _check_apart(arrays, start, end):
    """The arrays to write may not share memory with each other."""
    order = numpy.argsort(start, kind='stable')
    reach = numpy.maximum.accumulate(end[order])
    for k in numpy.flatnonzero(start[order][1:] < reach[:-1]) + 1:
        # some array before it goes on behind its beginning
        for j in range(k):
            if end[order[j]] > start[order[k]] and _oc.share_elements(arrays[order[j]], arrays[order[k]]):
                raise ValueError('two of the arrays to write overlap in memory')


def _hit_by(src, dst):
    """Positions of the inputs whose range of addresses meets that of an output
    other than their own (which may be the very same memory)."""
    # (outputs may lie inside each other's ranges: those that begin before the end of
    # an input, less those that end before its beginning)
    first = numpy.searchsorted(numpy.sort(dst[1]), src[0], 'right')
    last = numpy.searchsorted(numpy.sort(dst[0]), src[1], 'left')
    own = (src[0] == dst[0]) & (src[1] == dst[1])
    return numpy.flatnonzero(last - first > own)


def _prepare(arrays, targets, write):
    """Arrays the kernels cannot take as they are: refused, or replaced by
    copies.  Returns (arrays to read, arrays to write, positions of those made
    beside their target)."""
    src = _describe(arrays, 'arrays')
    if not write:
        return [a if d else a.copy('C') for a, d in zip(arrays, src['dense'])], None, ()
    finals, dst = arrays, src
    if targets is not None:
        finals, dst = targets, _describe(targets, 'out')
        for i, (a, b) in enumerate(zip(arrays, targets)):
            if a._shape != b._shape or a.dtype != b.dtype:
                raise ValueError('out[%d] has the shape %r and type %s, expected %r %s'
                                 % (i, b._shape, b.dtype, a._shape, a.dtype))
    ranges = _ranges(finals, dst)
    _check_apart(finals, *ranges)
    reads, writes = list(arrays), list(finals)
    if targets is not None:
        for i in _hit_by(_ranges(arrays, src), ranges):
            reads[i] = arrays[i].copy('K')
    # an array and its result are walked in the order they are stored in: where
    # these differ, or are no order at all, the result is made aside
    aside = numpy.flatnonzero((src['dense'] & dst['dense']) == 0)
    for i in aside:
        reads[i] = arrays[i].copy('C')
        writes[i] = ndarray(arrays[i]._shape, arrays[i].dtype)
    return reads, writes, aside


def _tables(arrays, targets, write, beside=None):
    return _rt.hot.tables(arrays, targets, _TYPES, _MAX, _BLOCK * _UNROLL,
                          _device.get_device_id(), write, beside)


class _Temporary:
    """``words`` doubles for the launches of one call, or the runtime library's
    static array where nothing may be allocated."""

    def __init__(self, words):
        self.nbytes = 8 * words
        self.stream = _stream.get_current_stream_ptr()
        self.static = _memory.static_scratch_active()
        if not self.static:
            self.memory = _memory.alloc(self.nbytes)
        elif self.nbytes > _rt.RT_SCRATCH_MAX_BYTES:
            raise RuntimeError(
                'static_scratch: the call needs %d bytes of scratch memory, the runtime '
                'library holds %d' % (self.nbytes, _rt.RT_SCRATCH_MAX_BYTES))

    def launch(self, fn, blocks, block, before, after=b''):
        """``before`` and ``after`` are the arguments around the temporary's address."""
        if self.static:
            fn.launch_packed_scratch((blocks, 1, 1), (block, 1, 1), before + bytes(8) + after,
                                     len(before), self.nbytes, 0, self.stream)
        else:
            fn.launch_packed((blocks, 1, 1), (block, 1, 1),
                             before + struct.pack('<Q', self.memory.ptr) + after, 0, self.stream)


_functions = {}


def _function(name, dev, t, nbytes):
    """The kernel for arrays of the type ``_TYPES[t]``, ``nbytes`` in all."""
    key = name, dev, t, _oc.stream_hints(nbytes, nbytes)[1]
    fn = _functions.get(key)
    if fn is None:
        fn = _functions[key] = _SOURCE.function(
            name, X_T=_TYPES[t], MAX_ENTRIES=_MAX, BLOCK=_BLOCK, UNROLL=_UNROLL,
            VEC=16 // _TYPES[t].itemsize, NT_IN=False, NT_OUT=key[3])
    return fn


def _run(arrays, targets, norm_out, max_norm, eps):
    write = max_norm is not None
    dev = _device.get_device_id()
    if norm_out is not None:
        _oc.check_array(norm_out, 'norm_out')
        _check_peer_access(norm_out, dev)
    finals, aside = arrays if targets is None else targets, ()
    tables = _tables(arrays, targets, write, norm_out)
    if tables is None:
        if write and norm_out is not None:
            _check_beside(norm_out, finals)
            _check_beside(norm_out, arrays)
        arrays, targets, aside = _prepare(arrays, targets, write)
        tables = _tables(arrays, targets, write)
    dtype = _TYPES[2 if tables and tables[-1][0] == 2 else 1]
    if norm_out is None:
        norm_out = ndarray((), dtype)
    else:
        _oc.check_out(norm_out, (), dtype, 'norm_out')
    total = sum(blocks for _, launches, _ in tables for _, _, blocks in launches)
    temp = _Temporary(total + 1)              # the factor, then the sums
    at = 1
    for t, launches, nbytes in tables:
        if not launches:
            continue
        fn = _function('cupy_square_sums', dev, t, nbytes)
        for table, n, blocks in launches:
            temp.launch(fn, blocks, _BLOCK, table + struct.pack('<ii', n, 0), struct.pack('<q', at))
            at += blocks
    fn = _FINISH.function('cupy_norm_of_sums', N_T=dtype)
    temp.launch(fn, 1, 1024, b'', struct.pack('<qQdd', total, norm_out.data.ptr,
                                              max_norm if write else 0.0, eps))
    if write:
        for t, launches, nbytes in reversed(tables):
            if not launches:
                continue
            fn = _function('cupy_scale_arrays', dev, t, nbytes)
            for table, n, blocks in reversed(launches):
                temp.launch(fn, blocks, _BLOCK, table + struct.pack('<ii', n, blocks))
        for i in aside:
            elementwise_copy(targets[i], finals[i])
    return norm_out


def _check_beside(norm_out, arrays):
    _oc.check_array(norm_out, 'norm_out')
    for a in arrays:
        _oc.check_array(a, 'arrays')
        if _oc.share_elements(a, norm_out):
            raise ValueError('norm_out overlaps an array to scale or to write')


def global_norm(arrays, *, norm_out=None):
    """Square root of the sum of the squares of all elements of ``arrays``.

    Args:
        arrays: sequence of float16, float32 and float64 arrays of any shapes;
            of no arrays the norm is 0.
        norm_out (cupy.ndarray): receives the result, of shape ``()``.

    Elements are added up as they are stored, by 16-byte vectors: arrays stored in
    another order, or that start elsewhere modulo 16 bytes, may give other last bits.

    Returns:
        cupy.ndarray: of shape ``()``; float32, or float64 if any array is.
        Nothing waits for it: it is on the device.
    """
    return _run(_as_list(arrays, 'arrays'), None, norm_out, None, 0.0)


def clip_by_global_norm(arrays, max_norm, *, eps=1e-6, out=None, norm_out=None):
    """Scales arrays down so that their :func:`global_norm` is ``max_norm`` at most.

    Every array is multiplied by ``min(1, max_norm / (norm + eps))``, a factor of 64
    bits (rounded to 32 for float16 arrays), and rounded once.  Where the norm is
    infinite the factor is 0, where it is NaN the factor is NaN.  Arrays whose norm plus ``eps`` does not exceed ``max_norm``,
    which may be infinite, keep their bits.

    Args:
        arrays: sequence of float16, float32 and float64 arrays; scaled in
            place without ``out``.
        max_norm (float): bound on the norm.
        eps (float): added to the norm in the quotient.
        out: sequence of arrays that receive the results, of the same shapes
            and types; each may be the array it belongs to.
        norm_out (cupy.ndarray): receives the norm, of shape ``()``; it may not
            lie in any of the arrays.

    Returns:
        cupy.ndarray: the norm before scaling, as :func:`global_norm` returns it.
    """
    max_norm, eps = float(max_norm), float(eps)
    if not (max_norm >= 0 and eps >= 0):
        raise ValueError('max_norm and eps must not be negative, got %r and %r' % (max_norm, eps))
    arrays = _as_list(arrays, 'arrays')
    if out is not None:
        out = _as_list(out, 'out')
        if len(out) != len(arrays):
            raise ValueError('out holds %d arrays, expected %d' % (len(out), len(arrays)))
    return _run(arrays, out, norm_out, max_norm, eps)


def _as_list(arrays, name):
    if isinstance(arrays, ndarray):
        raise TypeError('%s is a sequence of arrays, not one array' % name)
    return list(arrays)
