"""embedding and embedding_grad against NumPy in float64.

A looked up element is a product in the type sums are held in, rounded to the
table's type: u_out + 2 u (the scale itself is rounded).  A gradient row of n
terms is off by at most (n + 2) u times the sum of their sizes, and u_out."""
import numpy as np
import pytest

import cupy_amd as cp

pytestmark = pytest.mark.gpu

TYPES = ['float16', 'float32', 'float64']


def half_step(dtype):
    return np.finfo(dtype).eps / 2


def acc_step(dtype):
    return half_step('float64' if np.dtype(dtype) == np.float64 else 'float32')


def tiny(dtype):
    return float(np.finfo(dtype).smallest_subnormal) / 2


def make(shape, dtype, seed):
    return np.random.default_rng(seed).standard_normal(shape).astype(dtype)


def lookup64(table, ids, scale):
    met = (ids >= 0) & (ids < len(table))
    rows = np.zeros(ids.shape + table.shape[1:])
    rows[met] = table[ids[met].astype(np.int64)].astype(np.float64) * scale
    return rows


def check_lookup(got, table, ids, scale):
    want = lookup64(table, ids, scale)
    dtype = table.dtype
    assert got.dtype == dtype and got.shape == want.shape
    bound = (half_step(dtype) + 2 * acc_step(dtype)) * np.abs(want) + tiny(dtype)
    assert np.all(np.abs(got.get().astype(np.float64) - want) <= bound)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,width,n', [(1, 1, 1), (7, 5, 3), (100, 64, 1000), (1000, 777, 33),
                                          (50, 9000, 4), (4, 2048, 3000)])
def test_lookup(rows, width, n, dtype):
    table = make((rows, width), dtype, 1)
    rng = np.random.default_rng(2)
    ids = rng.integers(-2, rows + 2, n)
    for scale in (1.0, 0.37, -45.25):
        check_lookup(cp.embedding(cp.asarray(table), cp.asarray(ids), scale), table, ids, scale)
    got = cp.embedding(cp.asarray(table), cp.asarray(ids)).get()
    assert np.array_equal(got, lookup64(table, ids, 1).astype(dtype))


@pytest.mark.parametrize('kind', ['int8', 'uint8', 'int16', 'int32', 'uint32', 'int64', 'uint64'])
def test_types_of_ids(kind):
    table = make((90, 33), 'float32', 1)
    ids = np.random.default_rng(3).integers(0, 90, (4, 5)).astype(kind)
    top = np.iinfo(kind).max
    if top > 90:
        ids[1, 2] = top
    if kind.startswith('i'):
        ids[2, 3] = np.iinfo(kind).min
    check_lookup(cp.embedding(cp.asarray(table), cp.asarray(ids), 2.0), table, ids, 2.0)
    check_lookup(cp.embedding(cp.asarray(table), ids, 2.0), table, ids, 2.0)
    check_lookup(cp.embedding(cp.asarray(table), cp.asarray(ids)[::2, ::-1], 2.0), table,
                 ids[::2, ::-1], 2.0)
    grad = make((4, 5, 33), 'float32', 4)
    check_grad(cp.embedding_grad(cp.asarray(grad), cp.asarray(ids), 90), grad, ids, 90, 1.0)


def test_lookup_layouts():
    base = make((60, 200), 'float16', 1)
    d = cp.asarray(base)
    ids = np.array([[3, 0, 19], [7, 7, -1]])
    for view in ((lambda a: a[::3, 1:100]), (lambda a: a[::-1]), (lambda a: a[:, ::2]),
                 (lambda a: a.T)):
        table = np.ascontiguousarray(view(base))
        check_lookup(cp.embedding(view(d), cp.asarray(ids), 3.0), table, ids, 3.0)
        frame = cp.zeros((2, 4, table.shape[1] + 5), 'float16')
        into = frame[:, 1:, 2:-3]
        assert cp.embedding(view(d), cp.asarray(ids), 3.0, out=into) is into
        check_lookup(into, table, ids, 3.0)
        assert not frame.get()[:, 0].any() and not frame.get()[..., -3:].any()
    # the result over the table it is read from
    check_lookup(cp.embedding(d, cp.arange(60)[::-1], 1.0, out=d), base, np.arange(60)[::-1], 1.0)
    assert cp.embedding(cp.zeros((0, 4), 'float32'), cp.asarray([0, 1])).get().shape == (2, 4)
    assert cp.embedding(cp.ones((3, 4), 'float32'), 2).shape == (4,)
    assert cp.embedding(cp.ones((3, 4), 'float32'), []).shape == (0, 4)


def check_grad(got, grad, ids, rows, scale, dtype=None):
    dtype = np.dtype(dtype or grad.dtype)
    flat, g = ids.reshape(-1), grad.reshape(-1, grad.shape[-1]).astype(np.float64)
    met = (flat >= 0) & (flat < rows)
    flat, g = flat[met].astype(np.int64), g[met]
    want, size = np.zeros((rows, grad.shape[-1])), np.zeros((rows, grad.shape[-1]))
    np.add.at(want, flat, g)
    np.add.at(size, flat, np.abs(g))
    n = np.bincount(flat, minlength=rows)[:, None]
    want, size = want * scale, size * abs(scale)
    assert got.dtype == dtype and got.shape == want.shape
    bound = half_step(dtype) * np.abs(want) + (n + 2) * acc_step(grad.dtype) * size + tiny(dtype)
    assert np.all(np.abs(got.get().astype(np.float64) - want) <= bound)


# ids: how many, drawn how: spread out, few values, all the same, sorted, descending
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n,rows,width', [(1, 1, 1), (1, 9, 3), (65, 40, 17), (1000, 8191, 64),
                                          (1024, 511, 8), (1025, 512, 100), (5000, 100, 509),
                                          (16384, 3000, 24), (16385, 70000, 20), (50000, 262150, 4)])
@pytest.mark.parametrize('kind', ['spread', 'few', 'same', 'sorted', 'falling'])
def test_gradient(n, rows, width, kind, dtype):
    rng = np.random.default_rng(n)
    if kind == 'few':
        ids = rng.choice([0, rows - 1, rows // 2, -1], n)
    elif kind == 'same':
        ids = np.full(n, rows - 1)
    else:
        ids = rng.integers(-1, rows + 1, n)
        if kind == 'sorted':
            ids = np.sort(ids)
        elif kind == 'falling':
            ids = np.sort(ids)[::-1].copy()
    grad = make((n, width), dtype, 5)
    gd, idd = cp.asarray(grad), cp.asarray(ids)
    got = cp.embedding_grad(gd, idd, rows, 0.5)
    check_grad(got, grad, ids, rows, 0.5)
    # the same bits again, into memory that held something else
    out = cp.full((rows, width), 7, dtype)
    assert cp.embedding_grad(gd, idd, rows, 0.5, out=out) is out
    assert np.array_equal(out.get(), got.get())


# the counting of up to 4096, 8192 and 12288 pairs, the first sort behind it; 4, 8 and
# 16 pairs to a thread of the sort, and more than 64 tiles of the largest kind
@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('n,rows,width', [(4096, 300, 24), (4097, 300, 24), (8192, 200, 24), (8193, 200, 24),
                                          (12288, 70000, 20), (12289, 70000, 20), (131073, 700, 8),
                                          (300000, 262150, 4), (600000, 513, 5), (1100000, 70000, 4)])
@pytest.mark.parametrize('kind', ['spread', 'same', 'falling'])
def test_gradient_of_many_tokens(n, rows, width, kind, dtype):
    test_gradient(n, rows, width, kind, dtype)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,width', [(1, 1), (1, 40000), (70000, 1), (33333, 2), (9000, 7), (4097, 33),
                                        (2500, 509), (700, 4100), (90, 40001)])
def test_gradient_of_few_tokens(rows, width, dtype):
    """Every element of the table is written once, whatever the table starts on,
    and nothing beside it."""
    rng = np.random.default_rng(rows)
    for n, start in ((1, 0), (2, 1), (300, 3), (1024, 5)):
        n = min(n, max(1, 2000000 // width))
        ids = rng.integers(-1, rows + 1, n)
        ids[:n // 4] = rng.integers(0, rows)
        some = ids[n // 2:][:20]                       # the first rows, and the last
        some[:] = np.arange(len(some)) - 3
        ids[-1] = rows - 1
        grad = make((n, width), dtype, n)
        frame = cp.full(rows * width + 16, 7, dtype)
        out = frame[start:start + rows * width].reshape(rows, width)
        cp.embedding_grad(cp.asarray(grad), cp.asarray(ids), rows, 2.0, out=out)
        check_grad(out, grad, ids, rows, 2.0)
        rest = frame.get()
        rest[start:start + rows * width] = 7
        assert np.all(rest == 7)


def test_gradient_types_and_layouts():
    ids = np.random.default_rng(1).integers(0, 50, (6, 40))
    grad = make((6, 40, 100), 'float16', 2)
    got = cp.embedding_grad(cp.asarray(grad), cp.asarray(ids, dtype='int32'), 50, dtype='float32')
    check_grad(got, grad, ids, 50, 1.0, 'float32')
    wide = cp.asarray(make((6, 40, 230), 'float16', 3))
    for view in ((lambda a: a[..., 3:103]), (lambda a: a[..., ::2]), (lambda a: a[:, ::-1, :64])):
        part = view(wide)
        check_grad(cp.embedding_grad(part, cp.asarray(ids), 50), part.get(), ids, 50, 1.0)
    frame = cp.full((54, 109), 3, 'float16')
    into = frame[2:52, 5:105]
    assert cp.embedding_grad(cp.asarray(grad), cp.asarray(ids), 50, out=into) is into
    check_grad(into, grad, ids, 50, 1.0)
    rest = frame.get()
    rest[2:52, 5:105] = 3
    assert np.all(rest == 3)
    one = cp.broadcast_to(cp.asarray(grad[0, 0]), (6, 40, 100))
    check_grad(cp.embedding_grad(one, cp.asarray(ids), 50), np.broadcast_to(grad[0, 0], (6, 40, 100)),
               ids, 50, 1.0)
    assert not cp.embedding_grad(cp.zeros((0, 4), 'float32'), cp.zeros(0, 'int64'), 5).get().any()
    assert cp.embedding_grad(cp.zeros((3, 4), 'float32'), cp.zeros(3, 'int64'), 0).shape == (0, 4)
    assert not cp.embedding_grad(cp.ones((3, 4), 'float32'), cp.full(3, -1, 'int64'), 5).get().any()


def test_gradient_of_the_lookup_against_differences():
    """The lookup is linear: differences are exact up to rounding (1e-16 / 1e-3)."""
    table, ids = make((11, 6), 'float64', 1), np.array([3, 3, 10, -1, 0, 3])
    c = make((6, 6), 'float64', 2)
    grad = cp.embedding_grad(cp.asarray(c), cp.asarray(ids), 11, 1.7).get()
    for at in ((3, 2), (10, 5), (0, 0), (1, 1)):
        e = np.zeros_like(table)
        e[at] = 1e-3
        f = [float((cp.embedding(cp.asarray(table + s * e), cp.asarray(ids), 1.7).get() * c).sum())
             for s in (1, -1)]
        assert abs((f[0] - f[1]) / 2e-3 - grad[at]) <= 1e-10


def test_streams_and_replays():
    ids = np.random.default_rng(1).integers(0, 500, 20000)
    grad = cp.asarray(make((20000, 40), 'float32', 2))
    idd = cp.asarray(ids)
    want = cp.embedding_grad(grad, idd, 500).get()
    streams = [cp.cuda.Stream(non_blocking=True) for _ in range(2)]
    results = []
    for k in range(6):
        with streams[k % 2]:
            results.append(cp.embedding_grad(grad, idd, 500))
    for s in streams:
        s.synchronize()
    for r in results:
        assert np.array_equal(r.get(), want)


def test_table_past_32_bits():
    """Rows behind 2**31 elements are read and written where they are."""
    rows, width = (1 << 20) + 5, 2056
    table = cp.empty((rows, width), 'float16')
    table.fill(0)
    table[rows - 1] = cp.asarray((np.arange(width) % 100).astype('float16'))
    got = cp.embedding(table, cp.asarray([rows - 1, rows, 0])).get()
    assert np.array_equal(got[0], np.arange(width) % 100) and not got[1:].any()
    grad = cp.asarray(make((3, width), 'float16', 1))
    cp.embedding_grad(grad, cp.asarray([rows - 1, 2, rows - 1]), rows, out=table)
    check_grad(table[rows - 4:], grad.get(), np.array([3, -1, 3]), 4, 1.0)
    check_grad(table[:4], grad.get(), np.array([-1, 2, -1]), 4, 1.0)
