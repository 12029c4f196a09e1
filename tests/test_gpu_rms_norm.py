"""rms_norm, rms_norm_int8 and rms_norm_grad against the formula in float64.

Bounds, with u = eps / 2 of the type sums are held in and ``terms`` the longest
chain of additions one lane makes: a sum of squares is off by at most
``terms * u`` relative to itself, its root by half of that, and each further
operation adds u; the result is rounded once more, to its own type."""
import numpy as np
import pytest

import cupy_amd as cp

pytestmark = pytest.mark.gpu

TYPES = ['float16', 'float32', 'float64']
SHAPES = [(1, 1), (3, 5), (7, 8), (300, 64), (65, 127), (1030, 513), (9, 2047), (2, 8192),
          (600, 4100), (3, 16385), (2, 40001), (1500, 1000), (2, 3, 48), (96,)]


def half_step(dtype):
    return np.finfo(dtype).eps / 2


def acc_step(dtype):
    return half_step('float64' if np.dtype(dtype) == np.float64 else 'float32')


def tiny(dtype):
    # half of the smallest subnormal: what rounding below the normal range costs
    return float(np.finfo(dtype).smallest_subnormal) / 2


def terms(width):
    # a lane adds at most 32 elements of a row in registers, width / 1024 + 8 of a
    # longer one; the lanes are joined in at most 10 steps
    return 42 + width / 1024 + 8


def inputs(shape, dtype, seed=0, spread=1.0):
    rng = np.random.default_rng(seed)
    return (rng.standard_normal(shape) * spread).astype(dtype)


def norm64(h, w, eps):
    h = h.astype(np.float64)
    r = 1 / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    y = h * r
    return y if w is None else y * w.astype(np.float64)


def check_norm(y, want, width, dtype):
    bound = (half_step(dtype) + (terms(width) / 2 + 8) * acc_step(dtype)) * np.abs(want) + tiny(dtype)
    assert y.dtype == dtype
    assert np.all(np.abs(y.astype(np.float64) - want) <= bound)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', SHAPES)
def test_norm(shape, dtype):
    x, w, r = inputs(shape, dtype, 1), inputs(shape[-1:], dtype, 2), inputs(shape, dtype, 3, 3.0)
    for weight in (None, w):
        got = cp.rms_norm(cp.asarray(x), None if weight is None else cp.asarray(weight), eps=1e-5)
        check_norm(got.get(), norm64(x, weight, 1e-5), shape[-1], dtype)
    y, h = cp.rms_norm(cp.asarray(x), cp.asarray(w), cp.asarray(r), 1e-5)
    h64 = x.astype(np.float64) + r.astype(np.float64)
    check_norm(y.get(), norm64(h64, w, 1e-5), shape[-1], dtype)
    assert h.dtype == dtype
    assert np.all(np.abs(h.get().astype(np.float64) - h64) <= half_step(dtype) * np.abs(h64) * 1.001)


@pytest.mark.parametrize('shape', [(5, 96), (700, 1001), (2, 33000)])
def test_float32_weight_and_residual_with_float16(shape):
    x, w, r = inputs(shape, 'float16', 1), inputs(shape[-1:], 'float32', 2), inputs(shape, 'float32', 3)
    y, h = cp.rms_norm(cp.asarray(x), cp.asarray(w), cp.asarray(r))
    h64 = x.astype(np.float64) + r.astype(np.float64)
    check_norm(y.get(), norm64(h64, w, 1e-6), shape[-1], 'float16')
    assert h.dtype == np.float32
    assert np.all(np.abs(h.get() - h64) <= half_step('float32') * np.abs(h64) * 1.001)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', SHAPES)
def test_norm_to_int8(shape, dtype):
    x, w, r = inputs(shape, dtype, 4), inputs(shape[-1:], dtype, 5), inputs(shape, dtype, 6)
    q, s, h = cp.rms_norm_int8(cp.asarray(x), cp.asarray(w), cp.asarray(r))
    want = norm64(x.astype(np.float64) + r.astype(np.float64), w, 1e-6)
    step = np.abs(want).max(-1) / 127
    assert q.dtype == np.int8 and s.dtype == np.float32 and s.shape == shape[:-1]
    off = (terms(shape[-1]) / 2 + 10) * acc_step(dtype)
    s_, q_ = s.get().astype(np.float64), q.get().astype(np.float64)
    assert np.all(np.abs(s_ - step) <= (off + half_step('float32')) * step)
    # half a step, and what the quotient (at most 127) is off by
    assert np.all(np.abs(q_ - want / np.where(step > 0, step, 1)[..., None]) <= 0.5 + 127 * off)
    assert np.all(np.abs(q_).max(-1) == 127)
    h64 = x.astype(np.float64) + r.astype(np.float64)
    assert np.all(np.abs(h.get().astype(np.float64) - h64) <= half_step(dtype) * np.abs(h64) * 1.001)


def test_int8_rows_of_zeros_of_tiny_and_of_huge_values():
    x = np.zeros((6, 40), np.float32)
    x[1] = 1e-37 * np.linspace(-1, 1, 40)
    x[2] = 1e15 * np.linspace(-1, 1, 40)
    x[3, 7] = np.inf
    x[4, 9] = np.nan
    x[5, 3] = -2.5
    q, s = cp.rms_norm_int8(cp.asarray(x))
    q, s = q.get(), s.get()
    assert np.all(q[0] == 0) and s[0] == 0
    for row in (1, 2):
        assert np.all(np.abs(q[row] - 127 * np.linspace(-1, 1, 40)) <= 0.5 + 1e-3)
    assert np.isnan(s[3]) and np.isnan(s[4])
    assert q[5, 3] == -127 and np.all(np.delete(q[5], 3) == 0)
    y = cp.rms_norm(cp.asarray(x)).get()
    assert np.all(y[0] == 0) and np.isnan(y[3, 7]) and np.all(np.delete(y[3], 7) == 0)
    assert np.all(np.isnan(y[4]))


def grad64(g, x, w, eps):
    g, x = g.astype(np.float64), x.astype(np.float64)
    a = g if w is None else g * w.astype(np.float64)
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    n = x * r
    dx = r * (a - n * (a * n).mean(-1, keepdims=True))
    lead = tuple(range(x.ndim - 1))
    # and the sizes of what is added up, for the bounds
    size = np.abs(r * a) + np.abs(n) * r * np.abs(a * n).mean(-1, keepdims=True)
    return dx, (g * n).sum(lead), size, np.abs(g * n).sum(lead)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', SHAPES)
def test_gradient(shape, dtype):
    g, x = inputs(shape, dtype, 7), inputs(shape, dtype, 8, 2.0)
    w, d = inputs(shape[-1:], dtype, 9), inputs(shape, dtype, 10)
    u, out = acc_step(dtype), half_step(dtype)
    rows = x.size // shape[-1]
    off = 1.5 * terms(shape[-1]) + 10
    for weight, extra in ((None, None), (w, None), (w, d), (None, d)):
        got = cp.rms_norm_grad(cp.asarray(g), cp.asarray(x),
                               None if weight is None else cp.asarray(weight), 1e-5,
                               residual_grad=None if extra is None else cp.asarray(extra))
        dx, dw, size, dw_size = grad64(g, x, weight, 1e-5)
        if extra is not None:
            dx = dx + extra.astype(np.float64)
            size = size + np.abs(extra.astype(np.float64))
        if weight is not None:
            got, got_w = got
            assert got_w.dtype == dtype
            bound = out * np.abs(dw) + (rows + off) * u * dw_size + tiny(dtype)
            assert np.all(np.abs(got_w.get().astype(np.float64) - dw) <= bound)
        bound = out * np.abs(dx) + off * u * size + tiny(dtype)
        assert np.all(np.abs(got.get().astype(np.float64) - dx) <= bound)


# a row shorter than a vector, rows that share a wave, dw from the inputs, partial rows
# of dw, rows walked twice
FORMS = [(4, 1), (4, 3), (3, 5), (300, 64), (7, 1000), (600, 4100), (2, 40001)]


def check_scaled_gradient(shape, dtype, power, eps):
    """Rows of the size 2**power against the formula at the size 1, where nothing
    leaves the range of float64: dx(s x, eps) = dx(x, eps / s^2) / s, and dw is the
    same.  dx is compared times s, for where it is subnormal it is off by half of the
    smallest subnormal more (and the bound has room for as much again): in float64
    2^-1075, which float64 itself holds only times s."""
    s = 2.0 ** power
    g, x, w = inputs(shape, dtype, 1), inputs(shape, dtype, 2, 2.0), inputs(shape[-1:], dtype, 3)
    rows = x.size // shape[-1]
    u, out, off = acc_step(dtype), half_step(dtype), 1.5 * terms(shape[-1]) + 10
    scaled = np.ldexp(x, power)
    x = np.ldexp(scaled.astype(np.float64), -power)          # (subnormals have lost bits)
    for weight in (None, w):
        dx, dw, size, dw_size = grad64(g, x, weight, eps / s / s)
        got = cp.rms_norm_grad(cp.asarray(g), cp.asarray(scaled),
                               None if weight is None else cp.asarray(weight), eps)
        if weight is not None:
            got, got_w = got
            bound = out * np.abs(dw) + (rows + off) * u * dw_size + tiny(dtype)
            assert np.all(np.abs(got_w.get().astype(np.float64) - dw) <= bound)
        bound = out * np.abs(dx) + off * u * size + float(np.finfo(dtype).smallest_subnormal) * s
        assert np.all(np.abs(np.ldexp(got.get().astype(np.float64), power) - dx) <= bound)


@pytest.mark.parametrize('shape', FORMS)
@pytest.mark.parametrize('dtype,power,eps', [
    ('float32', 50, 1e-6), ('float32', 54, 1e-6), ('float32', -46, 0.0),
    ('float64', 430, 1e-6), ('float64', -365, 0.0)])
def test_gradient_of_large_and_small_rows(shape, dtype, power, eps):
    """Powers of the inverse root of the mean square (the third enters dx) leave the
    type's range long before that root, its square and dx do."""
    check_scaled_gradient(shape, dtype, power, eps)


@pytest.mark.parametrize('shape', FORMS)
@pytest.mark.parametrize('dtype,power,eps', [
    ('float32', 40, 1e-6), ('float32', 70, 1e-6), ('float32', 124, 1e-6), ('float32', -35, 0.0),
    ('float32', -80, 0.0), ('float32', -80, 1e-40), ('float32', -80, 1e-60), ('float32', -120, 0.0)])
def test_gradient_of_rows_of_any_size(shape, dtype, power, eps):
    """The squares themselves leave the type's range."""
    check_scaled_gradient(shape, dtype, power, eps)


@pytest.mark.parametrize('shape', FORMS + [(9, 2047)])
@pytest.mark.parametrize('dtype,power,eps', [
    ('float32', 70, 1e-6), ('float32', 124, 1e-6), ('float32', -80, 0.0), ('float32', -80, 1e-40),
    ('float32', -80, 1e-60), ('float32', -130, 0.0), ('float32', -30, 0.0)])
def test_rows_of_any_size(shape, dtype, power, eps):
    """y of rows times s and eps times s^2 is y of the rows; the scale of the 8 bits as
    well.  Rows of every size side by side, zeros and an infinity among them."""
    s = 2.0 ** power
    x, w, r = inputs(shape, dtype, 1), inputs(shape[-1:], dtype, 2), inputs(shape, dtype, 3)
    plain = np.arange(shape[0]) % 5 == 3                    # rows of the ordinary size
    powers = np.where(plain, 0, power)[:, None]
    xs, rs = np.ldexp(x, powers), np.ldexp(r, powers)
    one = np.ldexp(1.0, -powers)
    h64 = xs.astype(np.float64) * one + rs.astype(np.float64) * one
    eps64 = np.where(plain, eps, eps / s / s)[:, None]
    want = norm64(h64, w, eps64)
    xd, rd, wd = cp.asarray(xs), cp.asarray(rs), cp.asarray(w)
    y, h = cp.rms_norm(xd, wd, rd, eps)
    check_norm(y.get(), want, shape[-1], dtype)
    assert np.all(np.abs(h.get().astype(np.float64) * one - h64)
                  <= half_step(dtype) * np.abs(h64) * 1.001 + tiny(dtype) * one)
    h64 = xs.astype(np.float64) * one
    check_norm(cp.rms_norm(xd, wd, eps=eps).get(), norm64(h64, w, eps64), shape[-1], dtype)
    q, s_, _ = (a.get().astype(np.float64) for a in cp.rms_norm_int8(xd, wd, rd, eps))
    step = np.abs(want).max(-1) / 127
    off = (terms(shape[-1]) / 2 + 10) * acc_step(dtype)
    assert np.all(np.abs(s_ - step) <= (off + half_step('float32')) * step)
    assert np.all(np.abs(q - want / step[:, None]) <= 0.5 + 127 * off)
    assert np.all(np.abs(q).max(-1) == 127)


@pytest.mark.parametrize('shape', [(1030, 3), (5000, 64), (3000, 127), (2000, 250), (3000, 1003), (1536, 4096), (300, 12000), (700, 33000)])
def test_rows_of_all_sizes_side_by_side(shape):
    """Few rows in between that leave the range, where workgroups take several: the
    others have the bits that they have among themselves, and dw holds all of them."""
    rng = np.random.default_rng(5)
    powers = np.where(rng.random(shape[0]) < 0.02, rng.choice([-80, 40, 70, 120], shape[0]), 0)
    powers[[0, -1]] = 70, -80
    plain, s = powers == 0, np.ldexp(1.0, powers)[:, None]
    x, g, d = (inputs(shape, 'float32', k) for k in range(3))
    w = inputs(shape[-1:], 'float32', 3)
    xs, ds = np.ldexp(x, powers[:, None]), np.ldexp(d, powers[:, None])
    wd, eps = cp.asarray(w), 1e-60
    # in the place of the inputs
    for q8 in (False, True):
        want = cp.rms_norm(cp.asarray(x), wd, cp.asarray(d), eps)[0].get()
        xd, dd = cp.asarray(xs), cp.asarray(ds)
        if q8:
            want = [a.get() for a in cp.rms_norm_int8(cp.asarray(x), wd, cp.asarray(d), eps)]
            q, sc, h = cp.rms_norm_int8(xd, wd, dd, eps, residual_out=dd)
            assert np.array_equal(q.get()[plain], want[0][plain])
            assert np.array_equal(sc.get()[plain], want[1][plain])
            # (every step is exact but the sum's own rounding: the same 8 bits)
            assert np.array_equal(q.get(), want[0])
        else:
            y, h = cp.rms_norm(xd, wd, dd, eps, out=xd, residual_out=dd)
            assert y is xd and h is dd
            assert np.array_equal(y.get()[plain], want[plain])
            h64 = (xs.astype(np.float64) + ds.astype(np.float64)) / s
            check_norm(y.get(), norm64(h64, w, eps / s / s), shape[-1], 'float32')
    u, off = acc_step('float32'), 1.5 * terms(shape[-1]) + 10
    dx, dw, size, dw_size = grad64(g, x, w, eps / s / s)
    want, _ = (a.get() for a in cp.rms_norm_grad(cp.asarray(g), cp.asarray(x), wd, eps))
    for place in range(3):
        gd, xd = cp.asarray(g), cp.asarray(xs)
        got, got_w = cp.rms_norm_grad(gd, xd, wd, eps, out=(None, gd, xd)[place])
        if not place:
            assert np.array_equal(got.get()[plain], want[plain])
        bound = u * np.abs(dx) + off * u * size + s * 2.0 ** -149
        assert np.all(np.abs(got.get() * s - dx) <= bound)
        bound = u * np.abs(dw) + (shape[0] + off) * u * dw_size + tiny('float32')
        assert np.all(np.abs(got_w.get() - dw) <= bound)


@pytest.mark.parametrize('shape', [(600, 100), (2000, 1003), (200, 8192), (50, 33000)])
def test_gradients_without_a_value_stay_in_their_row(shape):
    """An infinity and a NaN among the gradients, products too large for float32: the
    other rows have their bits, the other columns of dw their value."""
    g, x, w = inputs(shape, 'float32', 1), inputs(shape, 'float32', 2), inputs(shape[-1:], 'float32', 3)
    want, _ = (a.get() for a in cp.rms_norm_grad(cp.asarray(g), cp.asarray(x), cp.asarray(w)))
    rows = [3, shape[0] // 2, shape[0] - 1]
    g[rows[0], 7], g[rows[1], 8], g[rows[2], 9:12] = np.inf, np.nan, 3e38
    x[rows[2], 9:12] = 9.0
    with np.errstate(invalid='ignore'):
        _, dw, _, dw_size = grad64(g, x, w, 1e-6)
    for into in (False, True):
        gd = cp.asarray(g)
        got, got_w = (a.get() for a in cp.rms_norm_grad(gd, cp.asarray(x), cp.asarray(w),
                                                        out=gd if into else None))
        if not into:
            assert np.array_equal(np.delete(got, rows, 0), np.delete(want, rows, 0))
        assert np.isnan(got[rows[1]]).all() and not np.isfinite(got[rows[0]]).any()
        columns = np.arange(shape[1])
        columns = columns[(columns < 7) | (columns > 11)]
        off = (shape[0] + 1.5 * terms(shape[-1]) + 10) * acc_step('float32')
        assert np.all(np.abs(got_w[columns] - dw[columns])
                      <= 2.0 ** -24 * np.abs(dw[columns]) + off * dw_size[columns])


@pytest.mark.parametrize('shape', [(4, 5), (4, 64), (4, 1000), (4, 40001)])
def test_rows_of_zeros_infinities_and_nan_without_eps(shape):
    """As with one: what has no value is NaN, and the rows beside it keep theirs."""
    x, g, w = inputs(shape, 'float32', 1), inputs(shape, 'float32', 2), inputs(shape[-1:], 'float32', 3)
    x[0], x[1, 2], x[2, 3] = 0, np.inf, np.nan
    x[3] *= np.float32(1e30)
    y = cp.rms_norm(cp.asarray(x), cp.asarray(w), eps=0.0).get()
    assert np.all(np.isnan(y[0])) and np.isnan(y[1, 2]) and not np.delete(y[1], 2).any()
    assert np.all(np.isnan(y[2]))
    check_norm(y[3], norm64(x[3], w, 0.0), shape[-1], 'float32')
    q, s = (a.get() for a in cp.rms_norm_int8(cp.asarray(x), cp.asarray(w), eps=0.0))
    assert np.all(np.isnan(s[:3])) and np.isfinite(s[3]) and np.abs(q[3]).max() == 127
    dx = cp.rms_norm_grad(cp.asarray(g), cp.asarray(x), eps=0.0).get()
    assert np.isnan(dx[0]).all() and np.isnan(dx[1, 2]) and np.isnan(dx[2]).all()
    # (rows of zeros with an eps, however small)
    for dtype, eps in (('float32', 1e-40), ('float32', 1e-70), ('float16', 1e-70), ('float64', 1e-300)):
        z, wd = cp.zeros(shape, dtype), cp.asarray(w.astype(dtype))
        assert not cp.rms_norm(z, wd, eps=eps).get().any()
        q, s = cp.rms_norm_int8(z, wd, eps=eps)
        assert not q.get().any() and not s.get().any()
        _, dw = cp.rms_norm_grad(cp.asarray(g.astype(dtype)), z, wd, eps)
        assert not dw.get().any()


def test_float32_residual_of_any_size_with_float16():
    for power in (100, -100):
        x, w = inputs((6, 300), 'float16', 1), inputs((300,), 'float16', 2)
        r = np.ldexp(inputs((6, 300), 'float32', 3), power)
        if power < 0:
            x[:] = 0
        y, h = cp.rms_norm(cp.asarray(x), cp.asarray(w), cp.asarray(r), 0.0)
        h64 = np.ldexp(x.astype(np.float64), -power) + np.ldexp(r.astype(np.float64), -power)
        check_norm(y.get(), norm64(h64, w, 0.0), 300, 'float16')


@pytest.mark.parametrize('shape', [(4, 7), (3, 300), (2, 9000)])
def test_gradient_against_differences(shape):
    """f = sum(c * y) in float64: (f(x + h e) - f(x - h e)) / 2h, h = 1e-5, is off
    by h^2 times a third derivative of order one and by 1e-16 |f| / h."""
    x, w, c = inputs(shape, 'float64', 1), inputs(shape[-1:], 'float64', 2), inputs(shape, 'float64', 3)
    r = inputs(shape, 'float64', 4)
    dh = inputs(shape, 'float64', 5)

    def loss(x, w):
        y, h = cp.rms_norm(cp.asarray(x), cp.asarray(w), cp.asarray(r))
        return float((y.get() * c).sum() + (h.get() * dh).sum())
    _, h = cp.rms_norm(cp.asarray(x), cp.asarray(w), cp.asarray(r))
    dx, dw = cp.rms_norm_grad(cp.asarray(c), h, cp.asarray(w), residual_grad=cp.asarray(dh))
    dx, dw = dx.get(), dw.get()
    step = 1e-5
    rng = np.random.default_rng(0)
    for _ in range(6):
        at = tuple(rng.integers(0, n) for n in shape)
        e = np.zeros(shape)
        e[at] = step
        diff = (loss(x + e, w) - loss(x - e, w)) / (2 * step)
        assert abs(diff - dx[at]) <= 1e-6 * (1 + abs(dx[at]))
        e = np.zeros(shape[-1:])
        e[at[-1]] = step
        diff = (loss(x, w + e) - loss(x, w - e)) / (2 * step)
        assert abs(diff - dw[at[-1]]) <= 1e-6 * (1 + abs(dw[at[-1]]))


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
def test_layouts(dtype):
    """Windows, every second row, reversed and broadcast rows, transposed storage."""
    big = inputs((40, 200), dtype, 1)
    d = cp.asarray(big)
    views = [(lambda a: a[3:30, 1:100]), (lambda a: a[::2, 5:69]), (lambda a: a[::-1, :64]),
             (lambda a: a[:, ::3]), (lambda a: a.T), (lambda a: a.reshape(4, 10, 200)[:, ::2, 7:90]),
             (lambda a: a.reshape(4, 10, 200).transpose(1, 0, 2))]
    for view in views:
        x, dx = np.ascontiguousarray(view(big)), view(d)
        w, r = inputs(x.shape[-1:], dtype, 2), inputs(x.shape, dtype, 3)
        y, h = cp.rms_norm(dx, cp.asarray(w), cp.asarray(r))
        h64 = x.astype(np.float64) + r
        check_norm(y.get(), norm64(h64, w, 1e-6), x.shape[-1], dtype)
        # the results into windows of other arrays, which keep the rest
        frame = cp.zeros(tuple(n + 3 for n in x.shape), dtype)
        into = frame[tuple(slice(1, n + 1) for n in x.shape)]
        again = cp.rms_norm(dx, cp.asarray(w), cp.asarray(r), out=into)
        assert again[0] is into
        assert np.array_equal(into.get(), y.get())
        assert np.count_nonzero(frame.get()) == np.count_nonzero(y.get())
        g = cp.rms_norm_grad(dx, dx, cp.asarray(w))
        g2 = cp.rms_norm_grad(cp.asarray(x), cp.asarray(x), cp.asarray(w))
        assert np.array_equal(g[0].get(), g2[0].get()) and np.array_equal(g[1].get(), g2[1].get())
    row = cp.broadcast_to(d[0], (6, 200))
    got = cp.rms_norm(row).get()
    assert np.array_equal(got, np.broadcast_to(cp.rms_norm(d[:1]).get(), (6, 200)))


@pytest.mark.parametrize('shape', [(50, 512), (4, 40000)])
def test_outputs_on_inputs(shape):
    x, w, r = inputs(shape, 'float16', 1), inputs(shape[-1:], 'float16', 2), inputs(shape, 'float16', 3)
    want, want_h = (a.get() for a in cp.rms_norm(cp.asarray(x), cp.asarray(w), cp.asarray(r)))
    wd = cp.asarray(w)
    for _ in range(2):                # the second time from the record
        xd, rd = cp.asarray(x), cp.asarray(r)
        y, h = cp.rms_norm(xd, wd, rd, out=xd, residual_out=rd)
        assert y is xd and h is rd
        assert np.array_equal(xd.get(), want) and np.array_equal(rd.get(), want_h)
    # overlapping by half: as if the inputs had been copied
    store = cp.zeros((shape[0] + 1, shape[1]), 'float16')
    store[:-1][...] = cp.asarray(x)
    y, h = cp.rms_norm(store[:-1], wd, cp.asarray(r), out=store[1:])
    assert np.array_equal(y.get(), want) and np.array_equal(h.get(), want_h)
    for k in range(3):
        args = [cp.asarray(x), cp.asarray(r), cp.asarray(x)]
        plain = cp.rms_norm_grad(args[0], args[1], wd, residual_grad=args[2])
        got = cp.rms_norm_grad(args[0], args[1], wd, residual_grad=args[2], out=args[k])
        assert np.array_equal(got[0].get(), plain[0].get())
        assert np.array_equal(got[1].get(), plain[1].get())


@pytest.mark.parametrize('width', [48, 1000, 40000])
def test_outputs_beside_inputs_and_each_other(width):
    """Column blocks and odd and even rows of one array: nothing is shared."""
    x, w, r = inputs((6, width), 'float16', 1), inputs((width,), 'float16', 2), inputs((6, width), 'float16', 3)
    wd = cp.asarray(w)
    want, want_h = (a.get() for a in cp.rms_norm(cp.asarray(x), wd, cp.asarray(r)))
    for place in ((lambda a, k: a[:, 3 + k * (width + 1):][:, :width]),
                  (lambda a, k: a[:].reshape(-1)[:24 * width].reshape(24, width)[k::4])):
        for _ in range(2):
            a = cp.full((6, 4 * (width + 1) + 3), 9, 'float16')
            xd, rd, y, h = (place(a, k) for k in range(4))
            xd[...], rd[...] = cp.asarray(x), cp.asarray(r)
            before = a.get()
            got = cp.rms_norm(xd, wd, rd, out=y, residual_out=h)
            assert got[0] is y and got[1] is h
            assert np.array_equal(y.get(), want) and np.array_equal(h.get(), want_h)
            y[...], h[...] = 9, 9
            assert np.array_equal(a.get(), before)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', [(1, 600), (7, 1000), (50, 4099), (130, 8192)])
def test_gradient_of_few_long_rows(shape, dtype):
    """dw from the inputs where dx is written elsewhere, and in the place of each
    of them, by name and by another view of the same memory; rows apart."""
    g, x, d = inputs(shape, dtype, 1), inputs(shape, dtype, 2, 2.0), inputs(shape, dtype, 3)
    w = inputs(shape[-1:], dtype, 4)
    dx, dw, size, dw_size = grad64(g, x, w, 1e-5)
    dx, size = dx + d.astype(np.float64), size + np.abs(d.astype(np.float64))
    u, out = acc_step(dtype), half_step(dtype)
    off = 1.5 * terms(shape[-1]) + 10
    wide = cp.zeros((shape[0], shape[1] + 5), dtype)
    for where in range(8):
        args = [cp.asarray(a) for a in (g, x, d)]
        into = (None, args[0], args[1], args[2], args[0][:], args[1].reshape(shape), args[2][:],
                wide[:, 2:-3])[where]
        for _ in range(2):
            for a, b in zip(args, (g, x, d)):
                a[...] = cp.asarray(b)
            got, got_w = cp.rms_norm_grad(args[0], args[1], cp.asarray(w), 1e-5, residual_grad=args[2],
                                          out=into)
            bound = out * np.abs(dx) + off * u * size + tiny(dtype)
            assert np.all(np.abs(got.get().astype(np.float64) - dx) <= bound)
            bound = out * np.abs(dw) + (shape[0] + off) * u * dw_size + tiny(dtype)
            assert np.all(np.abs(got_w.get().astype(np.float64) - dw) <= bound)


def test_streams_and_repeated_calls():
    x, w = inputs((2000, 768), 'float16', 1), inputs((768,), 'float16', 2)
    g = inputs((2000, 768), 'float16', 3)
    xd, wd, gd = cp.asarray(x), cp.asarray(w), cp.asarray(g)
    first = [a.get() for a in cp.rms_norm_grad(gd, xd, wd)]
    streams = [cp.cuda.Stream(non_blocking=True) for _ in range(2)]
    results = []
    for k in range(6):
        with streams[k % 2]:
            results.append(cp.rms_norm_grad(gd, xd, wd))
    for s in streams:
        s.synchronize()
    for dx, dw in results:
        assert np.array_equal(dx.get(), first[0]) and np.array_equal(dw.get(), first[1])


def test_static_scratch():
    x, w, g = (cp.asarray(inputs(s, 'float32', k)) for k, s in enumerate([(64, 300), (300,), (64, 300)]))
    out, wout = cp.empty((64, 300), 'float32'), cp.empty((300,), 'float32')
    want = [a.get() for a in cp.rms_norm_grad(g, x, w, out=out, weight_out=wout)]
    out.fill(0), wout.fill(0)
    with cp.cuda.memory.static_scratch():
        cp.rms_norm_grad(g, x, w, out=out, weight_out=wout)
    assert np.array_equal(out.get(), want[0]) and np.array_equal(wout.get(), want[1])
    with cp.cuda.memory.static_scratch():
        with pytest.raises(RuntimeError):
            cp.rms_norm(x, w)


def test_empty():
    for shape in ((0, 5), (5, 0), (0,)):
        x, w = cp.zeros(shape, 'float16'), cp.ones(shape[-1:], 'float16')
        y, h = cp.rms_norm(x, w, x)
        assert y.shape == shape and h.shape == shape
        q, s = cp.rms_norm_int8(x, w)
        assert q.shape == shape and s.shape == shape[:-1] and not s.get().any()
        dx, dw = cp.rms_norm_grad(x, x, w)
        assert dx.shape == shape and dw.shape == shape[-1:] and not dw.get().any()


def test_rows_far_apart():
    """Rows whose offsets pass 32 bits: a stride of 2**31 elements of float16."""
    pitch = (1 << 31) + 8
    buf = cp.empty(pitch + 512, 'float16')
    rows = cp.ndarray((2, 512), 'float16', buf.data, strides=(pitch * 2, 2))
    x = inputs((2, 512), 'float16', 1)
    rows[...] = cp.asarray(x)
    check_norm(cp.rms_norm(rows, out=rows).get(), norm64(x, None, 1e-6), 512, 'float16')
