"""token_log_prob and token_log_prob_grad against the formulas in float64.

Bounds, u = eps / 2 of the results' type, d = m - x >= 0, E = sum(p d),
E2 = sum(p d^2): an exponential is off by 2u and by its argument's rounding
(d u), a sum of n by n u.  lse: (n + 4 + 2 E) u and its own rounding; the
constant log2(e) is rounded (to at most u / 2 relative), which counts as
another H u.  entropy = log s - u / s: the same, and each term of u again."""
import numpy as np
import pytest

import cupy_amd as cp

pytestmark = pytest.mark.gpu

TYPES = ['float16', 'float32', 'float64']


def half_step(dtype):
    return np.finfo(dtype).eps / 2


def acc(dtype):
    return np.dtype('float64' if np.dtype(dtype) == np.float64 else 'float32')


def logits_of(shape, dtype, seed=0, spread=3.0):
    return (np.random.default_rng(seed).standard_normal(shape) * spread).astype(dtype)


def tokens_of(shape, seed=1):
    return np.random.default_rng(seed).integers(0, shape[-1], shape[:-1])


class Exact:
    def __init__(self, x):
        x = x.astype(np.float64)
        self.u = None
        with np.errstate(all='ignore'):
            m = x.max(-1, keepdims=True)
            d = np.where(np.isneginf(x), 0.0, m - x)
            e = np.where(np.isneginf(x), 0.0, np.exp(x - m))
            s = e.sum(-1, keepdims=True)
            self.lse = (m + np.log(s))[..., 0]
            self.p = e / s
            # (not x - lse: rows of the lowest value swallow log s)
            self.log_p = np.where(np.isneginf(x), x, x - m - np.log(s))
            self.entropy = (np.log(s) + (self.p * d).sum(-1, keepdims=True))[..., 0]
            self.e1 = (self.p * d).sum(-1)
            self.e2 = (self.p * d * d).sum(-1)

    def off(self, n):
        return n + 6 + 2 * self.e1 + np.abs(self.entropy)


def chain(width):
    # additions a lane makes (64 lanes at least to rows of up to 1024 vectors of 8
    # elements and a few single ones, 128 to twice as long ones, 256 to longer ones),
    # and joins
    return width / (64 if width <= 8208 else 128 if width <= 16400 else 256) + 40


def check(x, tokens, got, top=0):
    kind = acc(x.dtype)
    u, n = half_step(kind), chain(x.shape[-1])
    ex = Exact(x)
    off = ex.off(n) * u
    assert got.lse.dtype == kind and got.log_prob.dtype == kind
    assert np.all(np.abs(got.lse.get() - ex.lse) <= off + 2 * u * np.abs(ex.lse))
    met = (tokens >= 0) & (tokens < x.shape[-1])
    want = np.take_along_axis(ex.log_p, np.where(met, tokens, 0)[..., None], -1)[..., 0]
    want = np.where(met, want, 0.0)
    lp = got.log_prob.get().astype(np.float64)
    # (for float32 the token's own logit is exact, lse is not: it is used unrounded)
    ruled_out = np.isneginf(want)
    assert np.array_equal(np.isneginf(lp), ruled_out)
    ok = ~ruled_out
    assert np.all((np.abs(lp - want) <= off + u * (np.abs(want) + np.abs(ex.lse) * (kind == np.float64)))[ok])
    if got.entropy is not None:
        bound = u * np.abs(ex.entropy) + off * (1 + ex.e1) + 4 * u * ex.e2
        assert np.all(np.abs(got.entropy.get() - ex.entropy) <= bound)
    if top:
        order = np.argsort(-x.astype(np.float64), axis=-1, kind='stable')[..., :top]
        assert got.top_token.dtype == np.int64
        assert np.array_equal(got.top_token.get(), order)
        want = np.take_along_axis(ex.log_p, order, -1)
        have = got.top_log_prob.get().astype(np.float64)
        ruled_out = np.isneginf(want)
        assert np.array_equal(np.isneginf(have), ruled_out)
        off = off[..., None] + u * (np.abs(want) + np.abs(ex.lse[..., None]) * (kind == np.float64))
        assert np.all((np.abs(have - want) <= off)[~ruled_out])


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', [(1, 1), (3, 2), (5, 33), (40, 64), (700, 1001), (4, 3, 257),
                                   (2, 50257), (600, 8193), (1, 200003), (130, 5000), (17,),
                                   (1100, 1), (1030, 40), (2000, 1001), (1200, 4095), (1024, 9000)])
def test_log_prob(shape, dtype):
    x, t = logits_of(shape, dtype), tokens_of(shape)
    xd, td = cp.asarray(x), cp.asarray(t)
    got = cp.token_log_prob(xd, td)
    assert got.entropy is None and got.top_token is None
    check(x, t, got)
    top = min(5, shape[-1])
    check(x, t, cp.token_log_prob(xd, td, entropy=True, top=top), top)
    check(x, t, cp.token_log_prob(xd, td, entropy=True, top=top), top)      # the record
    top = min(32, shape[-1])
    check(x, t, cp.token_log_prob(xd, td, top=top), top)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('width', [40, 3001, 20000, 70001, 140001])
def test_ties_masks_and_bands(dtype, width):
    """Equal values, values in one place, ruled out elements: the likeliest tokens
    in every order of storage."""
    rng = np.random.default_rng(3)
    low = float(np.finfo(dtype).min)
    rows = []
    rows.append(np.zeros(width))                                   # all the same
    rows.append(np.round(rng.standard_normal(width)))              # few values
    rows.append(np.arange(width) * (1000.0 / width))               # rising
    rows.append(-np.arange(width) * (1000.0 / width))              # falling
    r = rng.standard_normal(width)
    r[:width // 3] = -np.inf
    rows.append(r)
    r = np.full(width, -np.inf)                                    # one left
    r[width // 2] = 3.5
    rows.append(r)
    rows.append(np.full(width, low))                               # the type's lowest
    r = np.full(width, low)
    r[-3:] = [0.5, 1.5, 0.5]
    rows.append(r)
    r = rng.standard_normal(width)
    r[width // 5:][:30] += 50                                      # a band of neighbours
    rows.append(r)
    r = np.full(width, -5.0)                                       # what few threads hold
    r[::256 * (16 // np.dtype(dtype).itemsize)] = 5.0
    rows.append(r)
    x = np.stack(rows).astype(dtype)
    t = rng.integers(0, width, len(rows))
    t[5] = width // 2
    xd, td = cp.asarray(x), cp.asarray(t)
    for top in (1, 7, 32):
        check(x, t, cp.token_log_prob(xd, td, entropy=True, top=top), top)
    # many rows: a workgroup each
    for n in (60, 104 if width < 20000 else 0):
        big = np.tile(x, (n, 1))
        if n:
            check(big, np.tile(t, n), cp.token_log_prob(cp.asarray(big), cp.asarray(np.tile(t, n)),
                                                        entropy=True, top=9), 9)


@pytest.mark.parametrize('dtype', TYPES)
def test_the_best_in_the_vectors_of_one_thread(dtype):
    """More candidates than are ranked at once: every 1024th (256th) vector high."""
    vec = 16 // np.dtype(dtype).itemsize
    for rows, lanes in ((600, 1024), (2, 256)):
        width = lanes * vec * 300
        if rows == 600:
            rows, width = 520, 1024 * vec * 40
        x = np.full((rows, width), -3.0, dtype)
        cols = np.arange(width)
        high = (cols // vec) % lanes < (16 if lanes == 1024 else 4) * 3
        x[:, high] = (np.arange(high.sum()) % 1000 / 100).astype(dtype)
        t = np.zeros(rows, np.int64)
        got = cp.token_log_prob(cp.asarray(x), cp.asarray(t), top=20)
        order = np.argsort(-x[0].astype(np.float64), kind='stable')[:20]
        assert np.array_equal(got.top_token.get(), np.broadcast_to(order, (rows, 20)))
    # a wave to each row: all of the best in 16 of its lanes
    rows, width = 1100, 64 * vec * 8 + 3
    x = np.full((rows, width), -3.0, dtype)
    cols = np.arange(width)
    high = (cols // vec) % 64 < 16
    x[:, high] = (np.arange(high.sum()) % 500 / 100).astype(dtype)
    got = cp.token_log_prob(cp.asarray(x), cp.zeros(rows, 'int64'), top=20)
    order = np.argsort(-x[0].astype(np.float64), kind='stable')[:20]
    assert np.array_equal(got.top_token.get(), np.broadcast_to(order, (rows, 20)))


def test_rows_with_nothing_left_and_with_nan():
    for dtype in TYPES:
        for width in (10, 30000):
            x = logits_of((5, width), dtype)
            x[0] = -np.inf
            x[1, 3] = np.nan
            x[2, 4] = np.inf
            t = np.array([2, 3, 4, -1, width])
            got = cp.token_log_prob(cp.asarray(x), cp.asarray(t), entropy=True, top=3)
            lp, lse, h, tops, best = (a.get() for a in got)
            assert lse[0] == -np.inf and lp[0] == -np.inf and h[0] == 0
            assert np.all(tops[0] == -np.inf) and list(best[0]) == [0, 1, 2]
            for row in (1, 2):
                assert np.isnan(lse[row]) and np.isnan(lp[row]) and np.isnan(h[row])
                assert np.all(np.isnan(tops[row])) and np.all(best[row] == -1)
            assert lp[3] == 0 and lp[4] == 0 and np.all(np.isfinite(lse[3:]))
            g = cp.token_log_prob_grad(cp.ones(5, acc(dtype)), cp.asarray(x), cp.asarray(t), got.lse,
                                       entropy=got.entropy, entropy_grad=cp.ones(5, acc(dtype))).get()
            assert not g[0].any() and np.all(np.isnan(g[1:3]).any(-1)) and np.all(np.isfinite(g[3:]))
            g = cp.token_log_prob_grad(cp.ones(5, acc(dtype)), cp.asarray(x), cp.asarray(t), got.lse).get()
            assert not g[0].any() and not g[3:].any()


def check_grad(got, x, t, lse, g, h=None, gh=None):
    kind = acc(x.dtype)
    u, out = half_step(kind), half_step(x.dtype)
    x64, lse64 = x.astype(np.float64), lse.astype(np.float64)[..., None]
    with np.errstate(all='ignore'):
        d = x64 - lse64
        p = np.exp(d)
    met = (t >= 0) & (t < x.shape[-1])
    gain = np.where(met, g, 0.0).astype(np.float64)[..., None]
    hit = (np.arange(x.shape[-1]) == np.where(met, t, -1)[..., None])
    d = np.where(np.isneginf(d), 0.0, d)
    factor, size = gain, np.abs(gain)
    if h is not None:
        h64, gh64 = h.astype(np.float64)[..., None], gh.astype(np.float64)[..., None]
        factor = factor + gh64 * (d + h64)
        size = size + np.abs(gh64) * (np.abs(d) + np.abs(h64))
    want = gain * hit - p * factor
    # the argument of the exponential is rounded twice, the factor three times
    bound = (out * np.abs(want) + p * size * (2 * np.abs(d) + 8) * u + 2 * u * np.abs(gain) * hit
             + float(np.finfo(x.dtype).smallest_subnormal) / 2
             + size * float(np.finfo(kind).tiny))          # exponentials below it are 0
    assert got.dtype == x.dtype
    assert np.all(np.abs(got.get().astype(np.float64) - want) <= bound)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', [(1, 1), (3, 2), (5, 33), (600, 1001), (4, 3, 257), (2, 50257),
                                   (33, 5000), (17,), (50, 130), (40, 600), (30, 2300)])
def test_gradient(shape, dtype):
    x, t = logits_of(shape, dtype, 4), tokens_of(shape, 5)
    if t.ndim == 1 and len(t) > 2:
        t[1], t[2] = -100, shape[-1]
    if shape[-1] > 30:
        x[..., 5::7] = -np.inf
    kind = acc(dtype)
    rng = np.random.default_rng(6)
    g, gh = ((50 * rng.standard_normal(shape[:-1])).astype(kind) for _ in range(2))
    xd, td, gd, ghd = (cp.asarray(a) for a in (x, t, g, gh))
    fwd = cp.token_log_prob(xd, td, entropy=True)
    lse, h = fwd.lse.get(), fwd.entropy.get()
    check_grad(cp.token_log_prob_grad(gd, xd, td, fwd.lse), x, t, lse, g)
    got = cp.token_log_prob_grad(gd, xd, td, fwd.lse, entropy=fwd.entropy, entropy_grad=ghd)
    check_grad(got, x, t, lse, g, h, gh)
    into = xd.copy()
    assert cp.token_log_prob_grad(gd, into, td, fwd.lse, entropy=fwd.entropy, entropy_grad=ghd,
                                  out=into) is into
    assert np.array_equal(into.get(), got.get())


def test_gradient_against_differences():
    """h = 1e-5 in float64: off by h^2 and by 1e-15 / h, times values of order ten."""
    x, t = logits_of((3, 40), 'float64', 7), np.array([3, -1, 39])
    g, gh = np.array([1.5, 2.0, -0.5]), np.array([0.3, -1.0, 2.0])

    def loss(x):
        r = cp.token_log_prob(cp.asarray(x), cp.asarray(t), entropy=True)
        return float((r.log_prob.get() * g).sum() + (r.entropy.get() * gh).sum())
    r = cp.token_log_prob(cp.asarray(x), cp.asarray(t), entropy=True)
    grad = cp.token_log_prob_grad(cp.asarray(g), cp.asarray(x), cp.asarray(t), r.lse,
                                  entropy=r.entropy, entropy_grad=cp.asarray(gh)).get()
    for at in ((0, 3), (0, 7), (1, 0), (1, 11), (2, 39), (2, 20)):
        e = np.zeros_like(x)
        e[at] = 1e-5
        assert abs((loss(x + e) - loss(x - e)) / 2e-5 - grad[at]) <= 1e-7


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('width', [7, 3000, 140001])
def test_rows_of_the_lowest_value(width, dtype):
    """All of n equal elements have the log probability -log(n), however large."""
    low = np.finfo(dtype).min
    x = np.full((3, width), low, dtype)
    x[1, 2:] = -np.inf
    x[2] = -low
    t = np.array([width - 1, 1, 0])
    for top in (0, 1, 5):
        r = cp.token_log_prob(cp.asarray(x), cp.asarray(t), entropy=True, top=top)
        want = np.log([width, 2, width])
        # (float16: of 65504, rounded to 32 bits on the way out of 64)
        assert np.allclose(r.log_prob.get(), -want, rtol=0, atol=1e-4 * (dtype != 'float64') + 1e-9)
        assert np.allclose(r.entropy.get(), want, rtol=0, atol=1e-4 * (dtype != 'float64') + 1e-9)
        if top:
            assert list(r.top_token.get()[0]) == list(range(top))
            assert np.allclose(r.top_log_prob.get()[0], -want[0], rtol=0, atol=1e-4)
    g = cp.asarray(np.full(3, 2.0, acc(dtype)))
    d = cp.token_log_prob_grad(g, cp.asarray(x), cp.asarray(t), r.lse, entropy=r.entropy, entropy_grad=g).get()
    if dtype == 'float16':
        # (each p to half a step of lse near 65504, 2^-9, and of the result, 2^-11)
        want = -2.0 / np.array([width, 2, width])
        assert np.allclose(d[0, :2], want[0], rtol=5e-3, atol=1e-7) and np.allclose(d[1, 0], want[1], rtol=5e-3)
        assert np.allclose(d[1, 1], 2 + want[1], rtol=5e-3) and not d[1, 2:].any()
    else:
        assert not d[:2].any()


@pytest.mark.parametrize('dtype', TYPES)
def test_large_gradients_of_the_entropy(dtype):
    # what is ruled out has the gradient 0, however large the row's is: the second
    # row's only token has p = 1, log p = 0 and the entropy 0
    x = np.full((2, 40), -np.inf, dtype)
    x[0, 3], x[0, 30], x[1, 7] = 1, 1, 2
    x[1, 20] = np.finfo(dtype).min
    xd, td = cp.asarray(x), cp.asarray([3, 7])
    r = cp.token_log_prob(xd, td, entropy=True)
    gh = cp.asarray(np.full(2, 1e12, acc(dtype)))
    got = cp.token_log_prob_grad(cp.zeros(2, acc(dtype)), xd, td, r.lse, entropy=r.entropy,
                                 entropy_grad=gh, out=cp.empty_like(xd)).get()
    assert not np.isnan(got).any()
    got[0, [3, 30]] = got[1, 7] = 0            # (rounding errors, times the gradient)
    assert not got.any()


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
def test_layouts(dtype):
    base = logits_of((30, 4100), dtype, 8)
    d = cp.asarray(base)
    for view in ((lambda a: a[:, 1:4000]), (lambda a: a[::2, 3:1000]), (lambda a: a[::-1]),
                 (lambda a: a[:, ::3]), (lambda a: a.T), (lambda a: a.reshape(5, 6, 4100)[:, ::2])):
        x = np.ascontiguousarray(view(base))
        t = tokens_of(x.shape, 9)
        r = cp.token_log_prob(view(d), cp.asarray(t), entropy=True, top=4)
        check(x, t, r, 4)
        g = cp.ones(t.shape, 'float32')
        frame = cp.full(tuple(n + 2 for n in x.shape), 9, dtype)
        into = frame[tuple(slice(1, n + 1) for n in x.shape)]
        cp.token_log_prob_grad(g, view(d), cp.asarray(t), r.lse, out=into)
        check_grad(into, x, t, r.lse.get(), np.ones(t.shape))
        edge = frame.get()
        edge[tuple(slice(1, n + 1) for n in x.shape)] = 9
        assert np.all(edge == 9)
    # results into every second place of other arrays
    t = tokens_of(base.shape, 9)
    frames = [cp.zeros(60, 'float32'), cp.zeros(60, 'float32'), cp.zeros((30, 8), 'float32'),
              cp.zeros((30, 8), 'int64')]
    out = cp.TokenLogProb(frames[0][::2], frames[1][1::2], None, frames[2][:, ::2], frames[3][:, 4:])
    r = cp.token_log_prob(d, cp.asarray(t), top=4, out=out)
    check(base, t, r, 4)
    check(base, t, out, 4)
    assert not frames[0].get()[1::2].any() and not frames[3].get()[:, :4].any()
    one = cp.broadcast_to(d[0], (4, 4100))
    check(np.tile(base[0], (4, 1)), t[:4], cp.token_log_prob(one, cp.asarray(t[:4]), top=2), 2)


@pytest.mark.parametrize('shape', [(1000, 300), (5, 100001)])
def test_results_in_columns_of_one_array(shape):
    x, t = logits_of(shape, 'float32', 1), tokens_of(shape)
    r = cp.full((shape[0], 5), 9, 'float32')
    out = cp.TokenLogProb(r[:, 0], r[:, 2], r[:, 1], None, None)
    for _ in range(2):
        r[...] = 9
        assert cp.token_log_prob(cp.asarray(x), cp.asarray(t), entropy=True, out=out).lse is out.lse
        check(x, t, out)
        assert np.all(r[:, 3:].get() == 9)


@pytest.mark.parametrize('width', [60000, 120000])
def test_streams_and_replays(width):
    x, t = logits_of((6, width), 'float16', 1), tokens_of((6, width))
    xd, td = cp.asarray(x), cp.asarray(t)
    want = [a.get() for a in cp.token_log_prob(xd, td, entropy=True, top=8)]
    streams = [cp.cuda.Stream(non_blocking=True) for _ in range(2)]
    results = []
    for k in range(6):
        with streams[k % 2]:
            results.append(cp.token_log_prob(xd, td, entropy=True, top=8))
    for s in streams:
        s.synchronize()
    for r in results:
        assert all(np.array_equal(a.get(), w) for a, w in zip(r, want))


def test_no_rows():
    r = cp.token_log_prob(cp.zeros((0, 7), 'float16'), cp.zeros(0, 'int64'), entropy=True, top=2)
    assert r.log_prob.shape == (0,) and r.top_token.shape == (0, 2)
    g = cp.token_log_prob_grad(r.lse, cp.zeros((0, 7), 'float16'), cp.zeros(0, 'int64'), r.lse)
    assert g.shape == (0, 7)


def test_logits_past_32_bits():
    rows, width = 3, (1 << 30) + 24
    x = cp.empty((rows, width), 'float16')
    x.fill(-np.inf)
    x[2, width - 3:] = cp.asarray([1.0, 2.0, 0.5], dtype='float16')
    x[0, 5] = 1.0
    x[1, :8] = cp.asarray(np.arange(8), dtype='float16')
    t = cp.asarray([5, 7, width - 1])
    r = cp.token_log_prob(x, t, entropy=True, top=3)
    tail = np.array([1.0, 2.0, 0.5])
    lse = np.log(np.exp(tail).sum())
    assert list(r.top_token.get()[2]) == [width - 2, width - 3, width - 1]
    assert abs(r.lse.get()[2] - lse) < 1e-6 and abs(r.log_prob.get()[2] - (0.5 - lse)) < 1e-6
    assert r.log_prob.get()[0] == 0 and list(r.top_token.get()[1]) == [7, 6, 5]
    cp.token_log_prob_grad(cp.ones(3, 'float32'), x, t, r.lse, out=x)
    p = np.exp(tail - lse)
    assert np.allclose(x[2, width - 3:].get(), np.array([0, 0, 1]) - p, atol=1e-3)
    assert not x[2, :1000].get().any() and not x[0, 6:2000].get().any()
