"""global_norm and clip_by_global_norm against NumPy in float64.

float16: 64 squares are added in 32 bits (64 * 2^-24, half of it in the root),
the rest in 64; the result is rounded to its type, the scaled elements once."""
import numpy as np
import pytest

import cupy_amd as cp

pytestmark = pytest.mark.gpu

TYPES = ['float16', 'float32', 'float64']


def half_step(dtype):
    return np.finfo(dtype).eps / 2


def off(dtypes):
    return 34 * 2.0 ** -24 if 'float16' in dtypes else 2.0 ** -40 if 'float64' not in dtypes else 2.0 ** -48


def make(shapes, dtype, seed=0, spread=1.0):
    rng = np.random.default_rng(seed)
    types = dtype if isinstance(dtype, list) else [dtype] * len(shapes)
    return [(rng.standard_normal(s) * spread).astype(t) for s, t in zip(shapes, types)]


def norm64(arrays):
    return float(np.sqrt(sum((a.astype(np.float64) ** 2).sum() for a in arrays)))


SHAPES = [(), (1,), (7, 3), (0,), (4096, 9), (16384,), (16385,), (3, 5, 7), (100, 1001), (2, 0, 3)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('copies', [1, 15, 31])
def test_norm_and_clipping(dtype, copies):
    arrays = make(SHAPES * copies, dtype, copies)
    dev = [cp.asarray(a) for a in arrays]
    want = norm64(arrays)
    got = cp.global_norm(dev)
    kind = 'float64' if dtype == 'float64' else 'float32'
    assert got.dtype == kind and got.shape == ()
    assert abs(float(got.get()) - want) <= (half_step(kind) + off([dtype])) * want
    for share in (0.25, 0.999, 1.5):
        outs = [cp.empty_like(a) for a in dev]
        norm = cp.clip_by_global_norm(dev, want * share, out=outs)
        assert np.array_equal(norm.get(), got.get())
        factor = min(1.0, want * share / (want + 1e-6))
        for a, o, d in zip(arrays, outs, dev):
            exact = a.astype(np.float64) * factor
            bound = (half_step(dtype) + off([dtype]) + 2 * half_step(kind)) * np.abs(exact)
            assert np.all(np.abs(o.get() - exact) <= bound + float(np.finfo(dtype).smallest_subnormal) / 2)
            assert np.array_equal(d.get(), a)
    inside = [a.copy() for a in dev]
    cp.clip_by_global_norm(inside, want * 0.25)
    again = [cp.empty_like(a) for a in dev]
    cp.clip_by_global_norm(dev, want * 0.25, out=again)
    for a, b in zip(inside, again):
        assert np.array_equal(a.get(), b.get())
    cp.clip_by_global_norm(inside, want * 2)          # nothing to do
    for a, b in zip(inside, again):
        assert np.array_equal(a.get(), b.get())


def test_mixed_types_and_layouts():
    shapes = [(50, 60), (33,), (20, 30), (7, 8, 9), (64, 64)]
    arrays = make(shapes, ['float16', 'float32', 'float32', 'float64', 'float16'], 3)
    base = [cp.asarray(a) for a in arrays]
    dev = [base[0].T, base[1][::2], base[2][:, 1::3], base[3].transpose(2, 0, 1), base[4][5:40]]
    host = [arrays[0].T, arrays[1][::2], arrays[2][:, 1::3], arrays[3].transpose(2, 0, 1), arrays[4][5:40]]
    want = norm64(host)
    got = cp.global_norm(dev)
    assert got.dtype == 'float64'
    assert abs(float(got.get()) - want) <= off(['float16']) * want
    factor = 3.0 / (want + 1e-6)
    outs = [cp.empty(a.shape, a.dtype) for a in dev]
    cp.clip_by_global_norm(dev, 3.0, out=outs)
    cp.clip_by_global_norm(dev, 3.0)
    for a, o, d in zip(host, outs, dev):
        exact = a.astype(np.float64) * factor
        bound = (half_step(a.dtype) + off(['float16']) + 2 * half_step('float32')) * np.abs(exact) + 2.0 ** -25
        assert np.all(np.abs(o.get() - exact) <= bound)
        # (in place: the arrays are walked in another order where they are copied
        # first, which regroups the 64 squares added in 32 bits: the same bound,
        # not the same bits)
        assert np.all(np.abs(d.get() - exact) <= bound)
    # what lies between the elements of the views is left as it was
    assert np.array_equal(base[1].get()[1::2], arrays[1][1::2])
    assert np.array_equal(base[2].get()[:, ::3], arrays[2][:, ::3])


def test_large_small_and_missing_values():
    big = [cp.full(1000, 3e30, 'float32'), cp.full(10, -3e30, 'float32')]
    assert abs(float(cp.global_norm(big).get()) / (3e30 * np.sqrt(1010.0)) - 1) < 1e-6
    small = [cp.full(1000, 3e-30, 'float32')]
    assert abs(float(cp.global_norm(small).get()) / (3e-30 * np.sqrt(1000.0)) - 1) < 1e-6
    top = [cp.full(100000, 65504, 'float16')]
    assert abs(float(cp.global_norm(top).get()) / (65504 * np.sqrt(1e5)) - 1) < 1e-5
    x = [cp.ones(5, 'float32'), cp.asarray(np.array([1, np.inf, 2], 'float32'))]
    n = cp.clip_by_global_norm(x, 1.0)
    assert np.isinf(n.get()) and not x[0].get().any() and np.isnan(x[1].get()[1])
    x = [cp.ones(5, 'float32'), cp.asarray(np.array([1, np.nan, 2], 'float32'))]
    n = cp.clip_by_global_norm(x, 1.0)
    assert np.isnan(n.get()) and np.all(np.isnan(x[0].get()))
    zero = [cp.zeros(5, 'float32')]
    assert cp.clip_by_global_norm(zero, 1.0).get() == 0 and not zero[0].get().any()
    assert cp.global_norm([]).get() == 0 and cp.global_norm([cp.zeros((0, 3))]).get() == 0
    x = [cp.full(4, 2.0, 'float32')]
    cp.clip_by_global_norm(x, 0.0)
    assert not x[0].get().any()


def test_factors_below_the_range_of_float32():
    """What float32 arrays are multiplied by need not be a float32: a norm of 9.5e39
    scaled to 1e-3, a norm of 1e60 (of a float64 array beside them) to 1e20.  The
    factor is off by 2^-40, the product is rounded once."""
    values = np.linspace(-3e38, 3e38, 1001).astype('float32')
    for beside, bound in (([], 1e-3), ([np.full(3, 1e60)], 1e20)):
        host = [values] + beside
        want = norm64(host)
        dev = [cp.asarray(a) for a in host]
        outs = [cp.empty_like(a) for a in dev]
        cp.clip_by_global_norm(dev, bound, out=outs)
        cp.clip_by_global_norm(dev, bound)
        for a, o, d in zip(host, outs, dev):
            exact = a.astype(np.float64) * (bound / (want + 1e-6))
            assert np.all(np.abs(o.get() - exact) <= (half_step(a.dtype) + 2.0 ** -40) * np.abs(exact))
            assert np.array_equal(o.get(), d.get())


def test_bounds_that_are_met_exactly():
    for values, bound in (([0.0, 0.0], 0.0), ([3.0, 4.0], 5.0), ([3.0, 4.0], np.inf), ([np.inf, 1.0], np.inf)):
        x = cp.asarray(np.array(values, 'float32'))
        n = cp.clip_by_global_norm([x], bound, eps=0.0)
        assert n.get() == np.sqrt(np.sum(np.square(values)))
        assert np.array_equal(x.get(), np.array(values, 'float32'))


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
def test_arrays_that_start_anywhere(dtype):
    flat = np.random.default_rng(1).standard_normal(200000).astype(dtype)
    src, dst = cp.asarray(flat), cp.zeros(200000, dtype)
    cuts = [(0, 1), (1, 3), (5, 40), (40, 16451), (16461, 60000), (60001, 60001), (60003, 199999)]
    xs, ys = [src[a:b] for a, b in cuts], [dst[a:b] for a, b in cuts]
    want = norm64([flat[a:b] for a, b in cuts])
    n = cp.empty((), 'float32')
    assert cp.clip_by_global_norm(xs, 1.0, out=ys, norm_out=n) is n
    assert abs(float(n.get()) - want) <= (2 ** -24 + off([dtype])) * want
    got = dst.get().astype(np.float64)
    held = np.zeros(200000, bool)
    for a, b in cuts:
        held[a:b] = True
    assert not got[~held].any()
    exact = flat[held].astype(np.float64) / (want + 1e-6)
    bound = (half_step(dtype) + off([dtype]) + 2.0 ** -23) * np.abs(exact) + 2.0 ** -25
    assert np.all(np.abs(got[held] - exact) <= bound)


def test_results_that_overlap_inputs():
    flat = np.random.default_rng(1).standard_normal(40000).astype('float32')
    want = [flat[:30000] / (norm64([flat[:30000], flat[30000:]]) + 1e-6),
            flat[30000:] / (norm64([flat[:30000], flat[30000:]]) + 1e-6)]
    d = cp.asarray(flat)
    # each result where the other array is
    cp.clip_by_global_norm([d[:30000], d[30000:]], 1.0, out=[d[10000:], d[:10000]])
    assert np.allclose(d.get()[10000:], want[0], rtol=1e-6) and np.allclose(d.get()[:10000], want[1], rtol=1e-6)
    d = cp.asarray(flat)
    cp.clip_by_global_norm([d[:30000], d[30000:]], 1.0, out=[d[:30000], cp.empty(10000, 'float32')])
    assert np.allclose(d.get()[:30000], want[0], rtol=1e-6)


@pytest.mark.parametrize('dtype', TYPES)
def test_views_beside_each_other(dtype):
    """Column blocks of one matrix, odd and even rows, every second element, and an
    array between the elements of another: scaled in place and into views, with the
    rest left as it was."""
    host = np.random.default_rng(3).standard_normal((40, 130)).astype(dtype)
    for cut in ((lambda a: [a[:, :64], a[:, 64:100], a[:, 101:]]), (lambda a: [a[::2], a[1::2, :50]]),
                (lambda a: [a[:, ::2], a[:, 1::2]]), (lambda a: [a[3::9, 5], a[4, 6:90], a[5:11].T])):
        parts = cut(host)
        want = norm64(parts)
        exact = host.astype(np.float64)
        for part in cut(exact):
            part *= 1.0 / (want + 1e-6)
        bound = ((half_step(dtype) + off([dtype]) + 2.0 ** -24 * (dtype == 'float16')) * np.abs(exact)
                 + float(np.finfo(dtype).smallest_subnormal) / 2)
        for place in range(2):
            d = cp.asarray(host)
            n = cp.clip_by_global_norm(cut(d) if place else [cp.asarray(p) for p in parts], 1.0, out=cut(d))
            assert abs(float(n.get()) - want) <= (2.0 ** -24 + off([dtype])) * want
            assert np.all(np.abs(d.get() - exact) <= bound)
        d = cp.asarray(host)
        cp.clip_by_global_norm(cut(d), 1.0)
        assert np.all(np.abs(d.get() - exact) <= bound)


def test_streams():
    arrays = [cp.asarray(a) for a in make([(1000, 300), (17,)] * 5, 'float32', 1)]
    want = cp.global_norm(arrays).get()
    streams = [cp.cuda.Stream(non_blocking=True) for _ in range(2)]
    results = []
    for k in range(6):
        with streams[k % 2]:
            outs = [cp.empty_like(a) for a in arrays]
            results.append((cp.clip_by_global_norm(arrays, 1.0, out=outs), outs))
    for s in streams:
        s.synchronize()
    first = [o.get() for o in results[0][1]]
    for n, outs in results:
        assert np.array_equal(n.get(), want)
        assert all(np.array_equal(o.get(), f) for o, f in zip(outs, first))


def test_static_scratch():
    arrays = [cp.asarray(a) for a in make([(300, 70), (17,), (5, 9)], 'float16', 1)]
    outs, n = [cp.empty_like(a) for a in arrays], cp.empty((), 'float32')
    cp.clip_by_global_norm(arrays, 1.0, out=outs, norm_out=n)
    want, want_n = [o.get() for o in outs], n.get()
    for o in outs:
        o.fill(0)
    n.fill(0)
    with cp.cuda.memory.static_scratch():
        cp.clip_by_global_norm(arrays, 1.0, out=outs, norm_out=n)
    assert np.array_equal(n.get(), want_n)
    assert all(np.array_equal(o.get(), w) for o, w in zip(outs, want))
    with cp.cuda.memory.static_scratch():
        with pytest.raises(RuntimeError):
            cp.clip_by_global_norm(arrays, 1.0, out=outs)
        with pytest.raises(RuntimeError):
            cp.clip_by_global_norm([a.T[::2] for a in arrays[:1]], 1.0, norm_out=n)
