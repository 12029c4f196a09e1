"""Host side of the hand-written operators, without a GPU: what they refuse, how
arrays are seen as rows, overlap checks, records of calls."""
import struct

import numpy as np
import pytest

import cupy_amd as cp
from cupy_amd import _dryrun, _rt
from cupy_amd._core import _global_norm, _op_calls

dry = pytest.mark.skipif(not _dryrun.enabled(), reason='looks at launches that are only recorded')


def arr(shape, dtype='float32'):
    return cp.empty(shape, dtype)


# -- refusals -------------------------------------------------------------------------

def test_rms_norm_refuses():
    x, w = arr((4, 8)), arr((8,))
    for bad in (np.zeros((4, 8), 'f'), [1.0], 3.0, None):
        with pytest.raises(TypeError):
            cp.rms_norm(bad, w)
    for kind in ('int32', 'complex64', 'bool'):
        with pytest.raises(TypeError):
            cp.rms_norm(arr((4, 8), kind))
    with pytest.raises(TypeError):
        cp.rms_norm(x, np.zeros(8, 'f'))
    with pytest.raises(ValueError):
        cp.rms_norm(arr(()))
    with pytest.raises(ValueError):
        cp.rms_norm(x, arr((7,)))
    with pytest.raises(ValueError):
        cp.rms_norm(x, arr((4, 8)))
    with pytest.raises(TypeError):
        cp.rms_norm(x, arr((8,), 'float64'))
    with pytest.raises(TypeError):
        cp.rms_norm(x, arr((8,), 'float16'))
    with pytest.raises(ValueError):
        cp.rms_norm(x, w, arr((8,)))
    with pytest.raises(TypeError):
        cp.rms_norm(x, w, arr((4, 8), 'float16'))
    with pytest.raises(ValueError):
        cp.rms_norm(x, w, out=arr((8, 4)))
    with pytest.raises(TypeError):
        cp.rms_norm(x, w, out=arr((4, 8), 'float16'))
    with pytest.raises(ValueError):
        cp.rms_norm(x, w, residual_out=arr((4, 8)))
    with pytest.raises(TypeError):
        cp.rms_norm_int8(x, w, out=arr((4, 8)))
    with pytest.raises(ValueError):
        cp.rms_norm_int8(x, w, scale_out=arr((4, 1)))
    with pytest.raises(TypeError):
        cp.rms_norm(x, w, eps=None)
    both = arr((4, 8))
    with pytest.raises(ValueError):
        cp.rms_norm(x, w, arr((4, 8)), out=both, residual_out=both)


def test_rms_norm_grad_refuses():
    x, w = arr((4, 8)), arr((8,))
    with pytest.raises(ValueError):
        cp.rms_norm_grad(arr((8, 4)), x, w)
    with pytest.raises(ValueError):
        cp.rms_norm_grad(arr((4, 8), 'float16'), x, w)
    with pytest.raises(ValueError):
        cp.rms_norm_grad(x, x, weight_out=w)
    with pytest.raises(TypeError):
        cp.rms_norm_grad(x, x, w, weight_out=arr((8,), 'float16'))
    with pytest.raises(ValueError):
        cp.rms_norm_grad(x, x, w, residual_grad=arr((4, 7)))
    with pytest.raises(TypeError):
        cp.rms_norm_grad(np.zeros((4, 8), 'f'), x)


def test_embedding_refuses():
    table, ids = arr((10, 4)), arr((3,), 'int64')
    with pytest.raises(TypeError):
        cp.embedding(np.zeros((10, 4), 'f'), ids)
    with pytest.raises(TypeError):
        cp.embedding(arr((10, 4), 'int32'), ids)
    with pytest.raises(ValueError):
        cp.embedding(arr((10,)), ids)
    for bad in (arr((3,), 'float32'), arr((3,), 'bool'), [0.5], np.array([True])):
        with pytest.raises(IndexError):
            cp.embedding(table, bad)
    with pytest.raises(ValueError):
        cp.embedding(table, ids, out=arr((3, 5)))
    with pytest.raises(TypeError):
        cp.embedding(table, ids, out=arr((3, 4), 'float16'))
    with pytest.raises((TypeError, ValueError)):
        cp.embedding(table, ids, 'x')
    grad = arr((3, 4))
    with pytest.raises(ValueError):
        cp.embedding_grad(arr((4, 4)), ids, 10)
    with pytest.raises(ValueError):
        cp.embedding_grad(arr((3,)), ids, 10)
    with pytest.raises(ValueError):
        cp.embedding_grad(grad, ids, -1)
    with pytest.raises(ValueError):
        cp.embedding_grad(grad, ids, 1 << 31)
    with pytest.raises(TypeError):
        cp.embedding_grad(grad, ids, 10.0)
    with pytest.raises(TypeError):
        cp.embedding_grad(grad, ids, 10, dtype='float16')
    with pytest.raises(TypeError):
        cp.embedding_grad(grad, ids, 10, dtype='float32', out=arr((10, 4)))
    with pytest.raises(ValueError):
        cp.embedding_grad(grad, ids, 10, out=arr((11, 4)))


def test_token_log_prob_refuses():
    x, t = arr((4, 50)), arr((4,), 'int64')
    with pytest.raises(TypeError):
        cp.token_log_prob(np.zeros((4, 50), 'f'), t)
    with pytest.raises(TypeError):
        cp.token_log_prob(arr((4, 50), 'int32'), t)
    with pytest.raises(ValueError):
        cp.token_log_prob(x, arr((5,), 'int64'))
    with pytest.raises(ValueError):
        cp.token_log_prob(x, arr((4, 1), 'int64'))
    with pytest.raises(IndexError):
        cp.token_log_prob(x, arr((4,)))
    with pytest.raises(ValueError):
        cp.token_log_prob(arr((4, 0)), t)
    for top in (-1, 33, 51):
        with pytest.raises(ValueError):
            cp.token_log_prob(x, t, top=top)
    with pytest.raises(ValueError):
        cp.token_log_prob(arr((4, 5)), t, top=6)
    for top in (1.0, '1', None):
        with pytest.raises(TypeError):
            cp.token_log_prob(x, t, top=top)
    out = cp.TokenLogProb(arr(4), arr(4), None, None, None)
    with pytest.raises(TypeError):
        cp.token_log_prob(x, t, out=arr((4,)))
    with pytest.raises(ValueError):
        cp.token_log_prob(x, t, entropy=True, out=out)
    with pytest.raises(ValueError):
        cp.token_log_prob(x, t, out=out._replace(entropy=arr(4)))
    with pytest.raises(TypeError):
        cp.token_log_prob(x, t, out=out._replace(lse=arr(4, 'float64')))
    with pytest.raises(ValueError):
        cp.token_log_prob(x, t, out=out._replace(lse=out.log_prob))
    with pytest.raises(ValueError):
        cp.token_log_prob_grad(arr(4), x, t, arr(4), entropy=arr(4))
    with pytest.raises(ValueError):
        cp.token_log_prob_grad(arr(4), x, t, arr(4), entropy_grad=arr(4))
    with pytest.raises(ValueError):
        cp.token_log_prob_grad(arr(5), x, t, arr(4))
    with pytest.raises(TypeError):
        cp.token_log_prob_grad(1.0, x, t, arr(4))
    with pytest.raises(TypeError):
        cp.token_log_prob_grad(arr(4), x, t, arr(4), out=arr((4, 50), 'float16'))


def test_global_norm_refuses():
    x = arr((4, 50))
    with pytest.raises(TypeError):
        cp.global_norm(x)
    with pytest.raises(TypeError):
        cp.global_norm([x, np.zeros(3, 'f')])
    with pytest.raises(TypeError):
        cp.global_norm([x, arr(3, 'int32')])
    with pytest.raises(TypeError):
        cp.global_norm([x], norm_out=arr((), 'float64'))
    with pytest.raises(ValueError):
        cp.global_norm([x], norm_out=arr((1,)))
    for bad in (-1.0, float('nan')):
        with pytest.raises(ValueError):
            cp.clip_by_global_norm([x], bad)
    with pytest.raises(ValueError):
        cp.clip_by_global_norm([x], 1.0, out=[])
    with pytest.raises(ValueError):
        cp.clip_by_global_norm([x], 1.0, out=[arr((50, 4))])
    with pytest.raises(ValueError):
        cp.clip_by_global_norm([x], 1.0, out=[arr((4, 50), 'float16')])
    # written twice: by name, and by views that share elements
    with pytest.raises(ValueError):
        cp.clip_by_global_norm([x, x], 1.0)
    with pytest.raises(ValueError):
        cp.clip_by_global_norm([x[:3], x[2:]], 1.0)
    with pytest.raises(ValueError):
        cp.clip_by_global_norm([x, arr((4, 50))], 1.0, out=[x, x])
    flat = arr(10)
    with pytest.raises(ValueError):
        cp.clip_by_global_norm([flat], 1.0, norm_out=flat[3:4].reshape(()))
    cp.global_norm([x, x])       # read twice is no harm
    with pytest.raises(TypeError):
        cp.clip_by_global_norm([x], 1.0, norm_out=3)
    with pytest.raises(TypeError):
        cp.clip_by_global_norm([x], 1.0, norm_out=arr((), 'int32'))
    assert cp.global_norm([x, arr(0, 'float64')]).dtype == 'float64'


def test_the_norm_is_written_beside_what_is_scaled():
    # (the norm is written between the two readings of an array)
    flat, into = arr(10), arr(10)
    for a, b in ((flat, into), (flat[::2], into[::2])):
        with pytest.raises(ValueError):
            cp.clip_by_global_norm([a], 1.0, out=[b], norm_out=flat[4:5].reshape(()))
        with pytest.raises(ValueError):
            cp.clip_by_global_norm([a], 1.0, out=[b], norm_out=into[4:5].reshape(()))
    cp.clip_by_global_norm([flat], 1.0, out=[into], norm_out=arr(()))
    cp.global_norm([flat], norm_out=flat[4:5].reshape(()))        # (read once, before)


def elsewhere(a):
    """An array like ``a`` on another device (never read)."""
    memory = cp.cuda.memory.UnownedMemory(a.data.ptr, max(a.nbytes, 1), a, a.data.device_id + 1)
    return cp.ndarray(a.shape, a.dtype, cp.cuda.memory.MemoryPointer(memory, 0))


def test_arrays_of_another_device_are_refused():
    x, w, r, y, h = arr((4, 8)), arr(8), arr((4, 8)), arr((4, 8)), arr((4, 8))
    q, s, ids, table, n = arr((4, 8), 'int8'), arr(4), arr(4, 'int64'), arr((9, 8)), arr(())
    stats = [arr(4) for _ in range(5)]
    top = [arr((4, 2)), arr((4, 2), 'int64')]
    calls = [
        (lambda x, w, r, y, h: cp.rms_norm(x, w, r, out=y, residual_out=h), [x, w, r, y, h]),
        (lambda x, w, r, q, s, h: cp.rms_norm_int8(x, w, r, out=q, scale_out=s, residual_out=h),
         [x, w, r, q, s, h]),
        (lambda g, x, w, r, y, d: cp.rms_norm_grad(g, x, w, residual_grad=r, out=y, weight_out=d),
         [x, r, w, h, y, arr(8)]),
        (lambda t, i, y: cp.embedding(t, i, out=y), [table, ids, y]),
        (lambda g, i, t: cp.embedding_grad(g, i, 9, out=t), [y, ids, table]),
        (lambda x, i, *o: cp.token_log_prob(x, i, entropy=True, top=2, out=cp.TokenLogProb(*o)),
         [x, ids] + stats[:3] + top),
        (lambda g, x, i, l, e, d, y: cp.token_log_prob_grad(g, x, i, l, entropy=e, entropy_grad=d, out=y),
         [stats[0], x, ids, stats[1], stats[2], stats[3], y]),
        (lambda x, r, n: cp.global_norm([x, r], norm_out=n), [x, r, n]),
        (lambda x, r, n: cp.clip_by_global_norm([x, r], 1.0, norm_out=n), [x, r, n]),
        (lambda x, r, y, h, n: cp.clip_by_global_norm([x, r], 1.0, out=[y, h], norm_out=n), [x, r, y, h, n]),
    ]
    for call, arrays in calls:
        for _ in range(2):                        # (the second time beside a record)
            for k in range(len(arrays)):
                given = list(arrays)
                given[k] = elsewhere(given[k])
                with pytest.raises(ValueError, match='device'):
                    call(*given)
            call(*arrays)


# -- rows, overlap, descriptions ----------------------------------------------------------

def test_row_form():
    a = arr((6, 10, 40))
    assert _op_calls.row_form(a) == (60, 40)
    assert _op_calls.row_form(a[:, :, 3:20]) == (60, 40)
    assert _op_calls.row_form(a[::2]) is None
    assert _op_calls.row_form(a[:, ::2]) == (30, 80)
    assert _op_calls.row_form(a[:, 3]) == (6, 400)
    assert _op_calls.row_form(a[2, 3]) == (1, 40)
    assert _op_calls.row_form(a[..., ::2]) is None
    assert _op_calls.row_form(a[..., :1]) == (60, 40)
    assert _op_calls.row_form(a[::-1]) is None
    assert _op_calls.row_form(a[0, ::-1]) == (10, -40)
    assert _op_calls.row_form(a.transpose(1, 0, 2)) is None
    assert _op_calls.row_form(cp.broadcast_to(a[0, 0], (5, 40))) == (5, 0)
    assert not _op_calls.writable_rows(cp.broadcast_to(a[0, 0], (5, 40)))
    assert _op_calls.writable_rows(a[0, ::-1])


def test_overlap_of_listed_pairs():
    a = arr((10, 8))
    views = [a, a[:5], a[5:], arr((3,)), a[::2], a[0:0]]

    def hit(i, j, same=False):
        return _rt.hot.overlap(views, _op_calls._pack_spans(views, [(i, j, same)]))
    assert hit(0, 1) and hit(1, 0) and hit(0, 0) and hit(1, 4)
    assert not hit(1, 2) and not hit(0, 3) and not hit(0, 5) and not hit(5, 5)
    assert not hit(0, 0, True) and not hit(0, 1, True) and hit(2, 4, True)
    rev = a[::-1]
    views.append(rev)
    assert hit(6, 1) and hit(6, 2) and not hit(6, 3)
    with pytest.raises(ValueError):
        _rt.hot.overlap(views, b'1234')
    with pytest.raises(ValueError):
        _rt.hot.overlap([], _op_calls._pack_spans(views, [(0, 1, False)]))
    bad = bytearray(_op_calls._pack_spans(views, [(0, 1, False)]))
    bad[-8:] = struct.pack('<II', 99, 1)
    with pytest.raises(ValueError):
        _rt.hot.overlap(views, bytes(bad))
    with pytest.raises(AttributeError):
        _rt.hot.overlap([1], _op_calls._pack_spans([a], []))


def test_sharing_elements_is_decided_exactly():
    """Views of one piece of memory, against the sets of bytes they touch."""
    rng = np.random.default_rng(1)
    flat = arr(4000, 'float16')
    host = np.arange(8000, dtype=np.int64)

    def view(base, shape, start, steps):
        return np.lib.stride_tricks.as_strided(base[2 * start:], shape, [16 * t for t in steps])
    cases = []
    for _ in range(400):
        shape = tuple(int(n) for n in rng.integers(1, 7, 2))
        steps = [int(t) for t in rng.choice([1, 2, 3, 7, 10, 40, -1, -3], 2)]
        start = 1000 + int(rng.integers(0, 60))
        first = view(host, shape, start, steps)
        touched = set(first.ravel()) | set(first.ravel() + 1)
        a = cp.ndarray(shape, 'float16', flat.data + 2 * start, strides=[2 * t for t in steps])
        cases.append((a, touched))
    met = [0, 0]
    for (a, p), (b, q) in zip(cases[:200], cases[200:]):
        want = bool(p & q)
        met[want] += 1
        assert _op_calls.share_elements(a, b) == _op_calls.share_elements(b, a) == want
    assert min(met) > 20
    # of different types: the bytes count
    assert _op_calls.share_elements(flat[1:2], flat[:4].view('float32')[:1])
    assert not _op_calls.share_elements(flat[2:3], flat[:4].view('float32')[:1])
    assert not _op_calls.share_elements(flat[:0], flat)


def test_outputs_beside_each_other_are_no_overlap():
    """Column blocks, odd and even rows, every second element of one array."""
    a, w = arr((8, 128)), arr(64)
    x, ids = arr((4, 128)), arr(4, 'int64')
    for views in ((a[:, :64], a[:, 64:]), (a[:4].reshape(8, 64)[::2], a[:4].reshape(8, 64)[1::2]),
                  (a[:, ::2], a[:, 1::2])):
        x1, x2 = arr(views[0].shape), arr(views[0].shape)
        assert cp.rms_norm(x1, w, x2, out=views[0], residual_out=views[1])[0] is views[0]
        assert cp.rms_norm(views[0], w, out=views[1]) is views[1]
        cp.clip_by_global_norm(list(views), 1.0)
        cp.clip_by_global_norm([x1, x2], 1.0, out=list(views), norm_out=arr(()))
    r = arr((4, 3))
    out = cp.TokenLogProb(r[:, 0], r[:, 1], r[:, 2], None, None)
    assert cp.token_log_prob(x, ids, entropy=True, out=out).lse is out.lse
    flat = arr(20)
    cp.clip_by_global_norm([flat[::2]], 1.0, norm_out=flat[5:6].reshape(()))
    cp.clip_by_global_norm([flat[::9], flat[1:9]], 1.0)
    # those that do share elements are refused still
    for views in ((a[:, :65], a[:, 64:]), (a[::2], a[::3]), (a[:, ::2], a[:, 2::2])):
        with pytest.raises(ValueError):
            cp.clip_by_global_norm(list(views), 1.0)
    with pytest.raises(ValueError):
        cp.rms_norm(arr((8, 64)), w, arr((8, 64)), out=a[:, :64], residual_out=a[:, 63:127])
    with pytest.raises(ValueError):
        cp.token_log_prob(x, ids, out=cp.TokenLogProb(r[:, 0], r[:, :2].T[0], None, None, None))


@dry
def test_inputs_beside_an_output_are_not_copied():
    a, w = arr((8, 128)), arr(64)
    _dryrun.launches.clear()
    cp.rms_norm(a[:, :64], w, out=a[:, 64:])
    assert [l[0] for l in _dryrun.launches] == ['cupy_rms_norm']
    _dryrun.launches.clear()
    cp.rms_norm(a[:, :64], w, out=a[:, 63:127])
    assert len(_dryrun.launches) == 2


def test_inputs_inside_the_ranges_of_several_outputs():
    """Each input of the one is looked for among outputs that lie inside each other's
    ranges of addresses."""
    flat = arr(100)
    src = [flat[90:95], flat[40:50], arr(4)]
    dst = [flat[0:100:20], flat[1:81:8], flat[60:64]]
    arrays, targets = [a.ravel() for a in src], dst
    ranges = [_global_norm._ranges(v, _global_norm._describe(v, 'v')) for v in (arrays, targets)]
    assert list(_global_norm._hit_by(*ranges)) == [1]
    assert list(_global_norm._hit_by(ranges[1], ranges[1])) == [0, 1, 2]


def test_descriptions():
    a = arr((6, 4), 'float16')
    arrays = [a, a.T, a[:, ::2], arr((), 'float64'), arr((0, 3)), arr(3, 'int32')]
    d = np.frombuffer(_rt.hot.describe(arrays, _global_norm._TYPES), _global_norm._DESCRIPTION)
    assert list(d['type']) == [0, 0, 0, 2, 1, 3]
    assert list(d['n']) == [24, 24, 12, 1, 0, 3]
    assert list(d['dense']) == [1, 2, 0, 3, 3, 3]
    assert [int(p) for p in d['ptr']] == [x.data.ptr for x in arrays]
    with pytest.raises(TypeError):
        _rt.hot.describe([None], _global_norm._TYPES)
    with pytest.raises(TypeError):
        _rt.hot.describe(arrays, 3)


@pytest.mark.parametrize('item,dtype', [(2, 'float16'), (4, 'float32'), (8, 'float64')])
def test_tables_cover_every_array(item, dtype):
    """Replays the kernels' search: every element of every array is met once, by
    a workgroup of the array it belongs to."""
    rng = np.random.default_rng(1)
    flat = arr(1 << 20, dtype)
    cuts = np.sort(rng.integers(0, 1 << 20, 500))
    arrays = [flat[a:b] for a, b in zip(cuts[:-1], cuts[1:])]
    (found, launches, nbytes), = _global_norm._tables(arrays, None, True)
    assert _global_norm._TYPES[found] == np.dtype(dtype) and nbytes == (cuts[-1] - cuts[0]) * item
    per = 16 // item * 256 * 8
    seen = 0
    for table, n, blocks in launches:
        entries = np.frombuffer(table, _global_norm._ENTRY)
        assert len(entries) == 100 and n <= 100 and len(table) == 3200
        firsts = entries['first'][:n].astype(int)
        for k in range(n):
            e = entries[k]
            phase = (int(e['src']) & 15) // item
            count = (firsts[k + 1] if k + 1 < n else blocks) - firsts[k]
            assert (count - 1) * per < phase + int(e['n']) <= count * per
            seen += int(e['n'])
    assert seen == cuts[-1] - cuts[0]


# -- records --------------------------------------------------------------------------

def calls():
    x, w, r = arr((40, 96), 'float16'), arr((96,), 'float16'), arr((40, 96), 'float16')
    y, h, q, s = arr((40, 96), 'float16'), arr((40, 96), 'float16'), arr((40, 96), 'int8'), arr(40)
    dw = arr(96, 'float16')
    ids = arr((40,), 'int32')
    table = arr((300, 96), 'float16')
    stats = [arr(40) for _ in range(5)]
    result = cp.TokenLogProb(arr(40), arr(40), arr(40), arr((40, 3)), arr((40, 3), 'int64'))
    return [
        lambda: cp.rms_norm(x, w, r, out=y, residual_out=h),
        lambda: cp.rms_norm_int8(x, w, r, out=q, scale_out=s, residual_out=h),
        lambda: cp.rms_norm_grad(y, x, w, residual_grad=r, out=h, weight_out=dw),
        lambda: cp.embedding(table, ids, 2.0, out=y),
        lambda: cp.embedding_grad(y, ids, 300, 2.0, out=table),
        lambda: cp.token_log_prob(table[:40], ids, entropy=True, top=3, out=result),
        lambda: cp.token_log_prob_grad(stats[0], x, ids, stats[1], entropy=stats[2],
                                       entropy_grad=stats[3], out=y),
        lambda: cp.rms_norm(x, w, r, out=x, residual_out=r),
        lambda: cp.clip_by_global_norm([x, w], 1.0, out=[y, dw]),
    ]


@dry
@pytest.mark.parametrize('which', range(9))
def test_a_replayed_call_launches_the_same(which):
    call = calls()[which]
    seen = []
    for _ in range(3):
        _dryrun.launches.clear()
        call()
        seen.append([(l[0], l[1], l[2], l[3], len(l[4])) for l in _dryrun.launches])
    assert seen[0] and seen[0] == seen[1] == seen[2]


@dry
def test_records_are_found_by_layout_not_by_address():
    a, b = arr((4, 8)), arr((4, 8))
    keys = set()
    for x in (a, b):
        result, key = _op_calls.replay({}, [x], (1,))
        assert result is _op_calls._NOTHING and key is not None
        keys.add(key)
    assert len(keys) == 1
    assert _op_calls.replay({}, [np.zeros(3)], ())[1] is None
    # another layout, type or option: another key
    keys = {_op_calls.replay({}, [x], e)[1] for x, e in
            ((a, (1,)), (a, (2,)), (a[:, ::2], (1,)), (arr((4, 8), 'float16'), (1,)))}
    assert len(keys) == 4


@dry
def test_no_kernel_reads_a_table_of_no_rows():
    _dryrun.launches.clear()
    out = cp.embedding(arr((0, 4)), arr(3, 'int64'))
    cp.embedding(arr((0, 4)), arr(3, 'int64'), out=out)
    cp.embedding_grad(out, arr(3, 'int64'), 0)
    assert out.shape == (3, 4)
    assert not [l for l in _dryrun.launches if l[0].startswith('cupy_embedding')]


@dry
@pytest.mark.parametrize('which', range(8))
def test_calls_on_arrays_as_they_are_are_recorded(which):
    from cupy_amd._core import _embedding, _rms_norm, _token_log_prob
    tables = [_rms_norm._plans, _rms_norm._plans_int8, _rms_norm._plans_grad, _embedding._plans,
              _embedding._plans_grad, _token_log_prob._plans, _token_log_prob._plans_grad]
    for t in tables:
        t.clear()
    call = calls()[which]
    call(), call()
    assert sum(len(t) for t in tables) == 1


@dry
def test_options_that_compare_equal_are_not_mixed_up():
    table, ids = arr((10, 4)), arr((3,), 'int64')
    scales = []
    for scale in (0.0, -0.0, 0.0):
        _dryrun.launches.clear()
        cp.embedding(table, ids, scale)
        scales.append(struct.unpack_from('<d', _dryrun.launches[-1][4], 64)[0])
    assert [str(s) for s in scales] == ['0.0', '-0.0', '0.0']
    cp.embedding_grad(arr((3, 4)), ids, 10)
    with pytest.raises(TypeError):
        cp.embedding_grad(arr((3, 4)), ids, 10.0)
    x, t = arr((4, 50)), arr((4,), 'int64')
    cp.token_log_prob(x, t, top=1)
    with pytest.raises(TypeError):
        cp.token_log_prob(x, t, top=1.0)
    # an array in the place of another result of the same shape and type
    out = cp.TokenLogProb(arr(4), arr(4), arr(4), None, None)
    cp.token_log_prob(x, t, entropy=True, out=out)
    with pytest.raises(ValueError):
        cp.token_log_prob(x, t, entropy=True,
                          out=cp.TokenLogProb(arr(4), arr(4), None, arr(4), None))
    with pytest.raises(TypeError):
        cp.token_log_prob(x, t, out=(arr(4), arr(4), None, None, None))


def test_recorded_calls_made_by_the_extension():
    """hot.call without a launch: records of no launches."""
    a, b, c = arr((4, 8)), arr((4, 8)), arr(3)
    nothing = struct.pack('<II', 0, 0)
    plans = {}

    def call(arrays, extra=(1,), table=None):
        return _rt.hot.call(plans if table is None else table, arrays, 0, 0, extra, 0)
    miss = call([a, b])
    assert type(miss) is list and len(miss) == 1
    key = miss[0]
    plans[key] = (None, nothing, 1, None)
    assert call([a, b]) is b and call([b, a]) is a
    plans[key] = (None, nothing, (1, 0), None)
    assert call([a, b])[0] is b
    assert call([a, b])[1] is a
    assert type(call([a, b], (2,))) is list and type(call([a, c])) is list
    plans[key] = (None, None, 0, 'recorded')
    found = call([a, b])
    assert found[0] == key and found[1][3] == 'recorded'
    plans[key] = (_op_calls._pack_spans([a, b], [(0, 1, False)]), nothing, 0, None)
    assert call([a, b]) is a
    assert call([a, a]) is None                 # the pair overlaps
    assert call([a, 'x']) is None               # of no signature
    plans[key] = (_op_calls._pack_spans([a, b], [(0, 1, True)]), nothing, 0, None)
    assert call([a, a]) is a
    for bad in (3, (None, nothing, 0), (3, nothing, 0, None), (None, nothing, 2, None),
                (None, nothing, -1, None), (None, nothing, (0, 5), None), (None, b'1', 0, None),
                (b'1234', nothing, 0, None)):
        plans[key] = bad
        with pytest.raises(ValueError):
            call([a, b])
    with pytest.raises(TypeError):
        _rt.hot.call([], [a], 0, 0, (), 0)
    with pytest.raises(TypeError):
        _rt.hot.call({}, [a], 0, 0, ([],), 0)       # a key that cannot be looked up
    with pytest.raises(TypeError):
        _rt.hot.call({}, [a], 0, 0, ())


def test_recorded_calls_with_temporaries():
    """The extension asks for their memory, hands it to the launches behind the
    arrays, and leaves the call to its record where there is none to be had."""
    a, b = arr((4, 8)), arr((4, 8))
    nothing, asked = struct.pack('<II', 0, 0), []

    def allocate(nbytes):
        asked.append(nbytes)
        return cp.cuda.alloc(nbytes)
    plans = {}
    key = _rt.hot.call(plans, [a, b], 0, 0, (), 0)[0]
    plans[key] = (None, nothing, 1, None, (allocate, 512, 64))
    assert _rt.hot.call(plans, [a, b], 0, 0, (), 0) is b and asked == [512, 64]
    plans[key] = (None, nothing, 1, 'recorded', (lambda nbytes: None, 512, 64))
    assert _rt.hot.call(plans, [a, b], 0, 0, (), 0)[1][3] == 'recorded'
    plans[key] = (None, None, 1, 'recorded', (allocate, 512))
    assert _rt.hot.call(plans, [a, b], 0, 0, (), 0)[1][3] == 'recorded' and len(asked) == 2

    def fail(nbytes):
        raise MemoryError
    plans[key] = (None, nothing, 1, None, (fail, 512))
    with pytest.raises(MemoryError):
        _rt.hot.call(plans, [a, b], 0, 0, (), 0)
    for bad in ((None, nothing, 1, None, ()), (None, nothing, 1, None, 512),
                (None, nothing, 1, None, (allocate, 512), 3)):
        plans[key] = bad
        with pytest.raises(ValueError):
            _rt.hot.call(plans, [a, b], 0, 0, (), 0)
    # under static_scratch the record's own path is taken
    assert _op_calls._temporary(100).ptr is not None
    with cp.cuda.memory.static_scratch():
        assert _op_calls._temporary(100) is None


@dry
def test_training_sizes_run_under_static_scratch():
    """The temporaries of a step's calls fit the runtime library's static array, up to
    32768 columns of a norm and millions of tokens; what does not fit says so."""
    def twice(call):
        counts = []
        call()
        for _ in range(2):
            _dryrun.launches.clear()
            with cp.cuda.memory.static_scratch():
                call()
            counts.append(len(_dryrun.launches))
        assert counts[0] == counts[1] > 0
    for rows, width, kind in ((16384, 4096, 'float16'), (8192, 2048, 'float16'), (4096, 1024, 'float16'),
                              (100000, 32768, 'float16'), (20000, 16384, 'float32'), (9000, 4096, 'float64'),
                              (5000, 40001, 'float16'), (3, 1000000, 'float32'), (300, 12000, 'float16')):
        g, x, w = arr((rows, width), kind), arr((rows, width), kind), arr(width, kind)
        dx, dw = arr((rows, width), kind), arr(width, kind)
        twice(lambda: cp.rms_norm_grad(g, x, w, out=dx, weight_out=dw))
    for n, width, rows, kind in ((16384, 2048, 131072, 'float16'), (8192, 4096, 131072, 'float16'),
                                 (262144, 4096, 131072, 'float16'), (1 << 20, 2048, 50257, 'float32'),
                                 (65536, 8192, 32768, 'float32'), (3000000, 512, 50257, 'float32'),
                                 (4001, 509, 8191, 'float32'), (1000, 178, 9846, 'float32')):
        g, ids, t = arr((n, width), kind), arr(n, 'int64'), arr((rows, width), kind)
        twice(lambda: cp.embedding_grad(g, ids, rows, out=t))
    g, ids, t = arr((10000000, 8), 'float16'), arr(10000000, 'int64'), arr((100, 8), 'float16')
    cp.embedding_grad(g, ids, 100, out=t)
    with cp.cuda.memory.static_scratch(), pytest.raises(RuntimeError, match='bytes of scratch'):
        cp.embedding_grad(g, ids, 100, out=t)


def test_tables_of_what_needs_preparation():
    def tables(arrays, targets=None, write=True):
        return _global_norm._tables(arrays, targets, write)
    a, b = arr((6, 4)), arr((6, 4))
    assert tables([a, b]) and tables([a], [b]) and tables([a, b], [a, b]) and tables([a, a], None, False)
    assert tables([]) == []
    assert tables([arr((0, 3)), arr(0, 'float64')]) == [(1, [], 0), (2, [], 0)]
    assert _global_norm._tables([a], None, True, b[2, 2]) and not _global_norm._tables([a], None, True, a[2, 2])
    assert _global_norm._tables([a], None, False, a[2, 2])
    assert tables([a.T], [arr((6, 4)).T]) and tables([arr((0, 3)), a], [arr((0, 3)), b])
    for case in (([a, a],), ([a, b], [b, a]), ([a], [a.T]), ([a], [b.T.reshape(6, 4)[::1, ::-1]]),
                 ([a[:, ::2]],), ([a], [arr((4, 6))]), ([a], [arr((6, 4), 'float16')]),
                 ([arr(3, 'int32')],), ([a[:4], a[2:]],), ([a[:3], b[:3]], [a[2:5], b[3:]]),
                 ([a[:3], b[:3]], [b[:3], a[:3]])):
        assert tables(*case) is None
    # the same pieces shifted by one: each input is another array's output
    flat = arr(100)
    assert tables([flat[10:20], flat[20:30]], [flat[20:30], flat[10:20]]) is None
    assert tables([flat[10:20], flat[20:30]], [flat[30:40], flat[40:50]])
    mixed = tables([arr(5, 'float64'), arr(70000, 'float16'), a, arr(3, 'float16')])
    assert [t for t, _, _ in mixed] == [0, 1, 2] and [n for _, l, _ in mixed for _, n, _ in l] == [2, 1, 1]
    with pytest.raises(TypeError):
        tables([3])
    with pytest.raises(ValueError):
        tables([a], [])
    for bad in ((0, 5), (5, 0), (5000, 5)):
        with pytest.raises(ValueError):
            _rt.hot.tables([a], None, _global_norm._TYPES, *bad, 0, True, None)
