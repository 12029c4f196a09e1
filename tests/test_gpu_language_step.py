"""The operators together, as a program uses them: a bigram language model (the
logits of the next token are the normalised row of a table, so that no matrix
product is needed) with its backward pass and a clipped step, against NumPy in
float64; scoring with alternatives; a step captured into a graph."""
import numpy as np
import pytest

import cupy_amd as cp

pytestmark = pytest.mark.gpu

V, N, EPS, SCALE = 257, 600, 1e-5, 1.5


def start(dtype):
    rng = np.random.default_rng(1)
    table = rng.standard_normal((V, V)).astype(dtype)
    bias = (0.1 * rng.standard_normal((V, V))).astype(dtype)
    weight = (1 + 0.1 * rng.standard_normal(V)).astype(dtype)
    ids = rng.integers(0, V, N)
    ids[::50] = -1
    target = rng.integers(0, V, N)
    target[::37] = -1
    return table, bias, weight, ids, target


def step64(table, bias, weight, ids, target, max_norm):
    """Loss, entropies and the clipped gradients of both tables and the weight."""
    t, b, w = (a.astype(np.float64) for a in (table, bias, weight))
    met = ids >= 0
    safe = np.where(met, ids, 0)
    x = np.where(met[:, None], t[safe] * SCALE, 0.0)
    h = x + np.where(met[:, None], b[safe], 0.0)
    r = 1 / np.sqrt((h * h).mean(-1, keepdims=True) + EPS)
    y = h * r * w
    lse = np.log(np.exp(y - y.max(-1, keepdims=True)).sum(-1)) + y.max(-1)
    p = np.exp(y - lse[:, None])
    has = target >= 0
    tt = np.where(has, target, 0)
    lp = np.where(has, y[np.arange(N), tt] - lse, 0.0)
    g = np.where(has, -1.0 / N, 0.0)
    dy = -g[:, None] * p
    dy[np.arange(N), tt] += g
    n, a = h * r, dy * w
    dh = r * (a - n * (a * n).mean(-1, keepdims=True))
    dw = (dy * n).sum(0)
    dt, db = np.zeros_like(t), np.zeros_like(b)
    np.add.at(dt, ids[met], dh[met] * SCALE)
    np.add.at(db, ids[met], dh[met])
    norm = np.sqrt((dt ** 2).sum() + (db ** 2).sum() + (dw ** 2).sum())
    c = min(1.0, max_norm / (norm + 1e-6))
    return lp, norm, dt * c, db * c, dw * c


def step(table, bias, weight, ids, target, g, max_norm, grads):
    x = cp.embedding(table, ids, SCALE)
    b = cp.embedding(bias, ids)
    y, h = cp.rms_norm(x, weight, b, EPS)
    r = cp.token_log_prob(y, target)
    dy = cp.token_log_prob_grad(g, y, target, r.lse)
    dh, _ = cp.rms_norm_grad(dy, h, weight, EPS, weight_out=grads[2])
    cp.embedding_grad(dh, ids, V, SCALE, out=grads[0])
    cp.embedding_grad(dh, ids, V, out=grads[1])
    return r, cp.clip_by_global_norm(grads, max_norm)


@pytest.mark.parametrize('max_norm', [0.01, 1e3])
def test_training_step(max_norm):
    host = start('float64')
    lp, norm, *want = step64(*host, max_norm)
    dev = [cp.asarray(a) for a in host]
    g = cp.full(N, -1.0 / N)
    for dtype, rtol in (('float64', 1e-10), ('float32', 2e-4)):
        # (float32: a handful of roundings of 2^-24 along the way, through sums of
        # hundreds of terms of both signs: compared by the size of the whole)
        params = [a.astype(dtype) for a in dev[:3]]
        grads = [cp.empty(a.shape, dtype) for a in params]
        r, n = step(*params, *dev[3:], g.astype(dtype), max_norm, grads)
        assert np.abs(r.log_prob.get() - lp).max() <= rtol * 10
        assert abs(float(n.get()) / norm - 1) <= rtol
        for a, b in zip(grads, want):
            assert np.linalg.norm(a.get() - b) <= rtol * np.linalg.norm(b)
        first = [a.get() for a in grads]
        step(*params, *dev[3:], g.astype(dtype), max_norm, grads)
        for a, b in zip(grads, first):
            assert np.array_equal(a.get(), b)


def test_scoring_from_int8():
    """Rows handed on in 8 bits are scored like the rows themselves, to half a
    step of the scale per logit."""
    table, bias, weight, ids, target = start('float16')
    x = cp.embedding(cp.asarray(table), cp.asarray(ids))
    y = cp.rms_norm(x, cp.asarray(weight))
    q, s = cp.rms_norm_int8(x, cp.asarray(weight))
    z = (q.astype('float32') * s[:, None]).astype('float16')
    half = (s.get() / 2 + 8 * 2.0 ** -11)[:, None]
    assert np.all(np.abs(z.get().astype(np.float64) - y.get()) <= half * 1.01)
    a = cp.token_log_prob(y, cp.asarray(target), entropy=True, top=5)
    b = cp.token_log_prob(z, cp.asarray(target), entropy=True, top=5)
    # a log probability moves by at most twice what any logit moves
    assert np.all(np.abs(a.log_prob.get() - b.log_prob.get()) <= 2.1 * half[:, 0])
    assert np.all(np.abs(a.top_log_prob.get() - b.top_log_prob.get()) <= 2.1 * half)


def test_captured_into_a_graph():
    """Calls with every output given, captured and replayed; replays give what the
    calls themselves give, with eager work of the program between them."""
    torch = pytest.importorskip('torch')
    table, bias, weight, ids, target = start('float32')
    dev = [cp.asarray(a) for a in (table, bias, weight, ids, target)]
    x, y, h = (cp.empty((N, V), 'float32') for _ in range(3))
    g = cp.full(N, -1.0 / N, dtype='float32')
    r = cp.TokenLogProb(cp.empty(N, 'float32'), cp.empty(N, 'float32'), cp.empty(N, 'float32'),
                        cp.empty((N, 4), 'float32'), cp.empty((N, 4), 'int64'))
    dy, dh, dw = cp.empty((N, V), 'float32'), cp.empty((N, V), 'float32'), cp.empty(V, 'float32')
    b, table_grad, norm = cp.empty((N, V), 'float32'), cp.empty((V, V), 'float32'), cp.empty((), 'float32')
    clipped = [cp.empty((V, V), 'float32'), cp.empty(V, 'float32')]

    def work():
        cp.embedding(dev[0], dev[3], SCALE, out=x)
        cp.embedding(dev[1], dev[3], out=b)
        cp.rms_norm(x, dev[2], b, EPS, out=y, residual_out=h)
        cp.token_log_prob(y, dev[4], entropy=True, top=4, out=r)
        cp.token_log_prob_grad(g, y, dev[4], r.lse, out=dy)
        cp.rms_norm_grad(dy, h, dev[2], EPS, out=dh, weight_out=dw)
        cp.embedding_grad(dh, dev[3], V, SCALE, out=table_grad)
        cp.clip_by_global_norm([table_grad, dw], 1e-3, out=clipped, norm_out=norm)

    stream = cp.cuda.Stream(non_blocking=True)
    with stream:
        work()
    stream.synchronize()
    outs = [x, b, y, h, dy, dh, dw, table_grad, norm] + clipped + list(r)
    want = [a.get() for a in outs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(torch.cuda.ExternalStream(stream.ptr)):
        graph.capture_begin()
        try:
            with stream, cp.cuda.memory.static_scratch():
                work()
        finally:
            graph.capture_end()
    for k in range(4):
        for a in outs:
            a.fill(0)
        cp.cuda.Stream.null.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, wanted in zip(outs, want):
            assert np.array_equal(a.get(), wanted)
        # other inputs, and the program's own calls in between
        scale = np.float32(1 + k)
        dev[0][...] = cp.asarray(table * scale)
        with stream:
            work()
        stream.synchronize()
        want = [a.get() for a in outs]


def test_captured_at_training_sizes():
    """The gradients of a norm and of a table, whose partial sums take 12.6 and 17.4 MB
    (34 where a weight has 32768 columns), captured together: every replay, with eager work
    of the program between them, gives the bits of the calls themselves."""
    torch = pytest.importorskip('torch')
    rng = np.random.default_rng(2)
    cases = []
    for rows, width, table in ((16384, 1024, 5000), (8192, 4096, 5000), (600, 32768, 300)):
        g, x = (cp.asarray(rng.standard_normal((rows, width), dtype=np.float32).astype('float16')) for _ in range(2))
        w = cp.asarray((1 + rng.random(width)).astype('float16'))
        ids = cp.asarray(rng.integers(-1, table, rows))
        cases.append((g, x, w, ids, cp.empty_like(x), cp.empty_like(w), cp.empty((table, width), 'float16')))

    def work():
        for g, x, w, ids, dx, dw, dt in cases:
            cp.rms_norm_grad(g, x, w, out=dx, weight_out=dw)
            cp.embedding_grad(dx, ids, len(dt), out=dt)

    stream = cp.cuda.Stream(non_blocking=True)
    outs = [a for case in cases for a in case[4:]]
    with stream:
        work()
    stream.synchronize()
    want = [a.get() for a in outs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(torch.cuda.ExternalStream(stream.ptr)):
        graph.capture_begin()
        try:
            with stream, cp.cuda.memory.static_scratch():
                work()
        finally:
            graph.capture_end()
    for k in range(3):
        for a in outs:
            a.fill(0)
        cp.cuda.Stream.null.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, wanted in zip(outs, want):
            assert np.array_equal(a.get(), wanted)
        for case in cases:
            case[0][...] = case[0] * np.float16(-1.5)
        with stream:
            work()
        stream.synchronize()
        want = [a.get() for a in outs]


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
def test_the_same_bits_from_arrays_laid_out_alike(dtype):
    """What fixes the order of a sum: sizes, strides, storage order and the address
    modulo 16, and nothing else.  Where only the address differs modulo 16, results
    are compared to the bound that holds for either: both are off by at most n
    roundings of 2^-24 relative to the sum of the sizes, n the elements a lane adds up."""
    rng = np.random.default_rng(7)
    item = np.dtype(dtype).itemsize
    n, width = 70, 1003
    x, g = (rng.standard_normal((n, width)).astype(dtype) for _ in range(2))
    w = (1 + rng.random(width)).astype(dtype)
    ids, tokens = cp.asarray(rng.integers(-1, 900, n)), cp.asarray(rng.integers(0, width, n))
    grad = cp.asarray(rng.standard_normal(n).astype('float32'))

    def at(a, start):
        """``a`` at ``start`` elements behind a 256-byte border, other things around it."""
        store = cp.full(a.size + 64, 3, dtype)
        assert store.data.ptr % 256 == 0
        view = store[start:start + a.size].reshape(a.shape)
        view[...] = cp.asarray(a)
        return view

    def everything(start):
        xd, gd, wd = at(x, start), at(g, start), at(w, start)
        r = cp.token_log_prob(xd, tokens, entropy=True, top=3)
        out = [r.log_prob, r.lse, r.entropy, r.top_log_prob,
               cp.token_log_prob_grad(grad, xd, tokens, r.lse), cp.global_norm([xd, gd, wd])]
        out += [*cp.rms_norm_grad(gd, xd, wd), *cp.rms_norm(xd, wd, gd), *cp.rms_norm_int8(xd, wd)]
        out += [cp.embedding_grad(gd, ids, 900), cp.embedding(xd, ids, 1.5)]
        return r.top_token.get(), [a.get().astype(np.float64) for a in out]
    best, first = everything(0)
    for start in (0, 16 // item, 48 // item):                # the same modulo 16
        again, same = everything(start)
        assert np.array_equal(again, best)
        for a, b in zip(same, first):
            assert np.array_equal(a, b)
    # logits of about 4 at most: lse, entropies and log probabilities of 3 to 11, whose
    # exponentials are summed in chains of at most 16 and 6 joins and rounded once
    for start in (1, 3, 5):
        again, other = everything(start)
        assert np.array_equal(again, best)
        for a, b in zip(other[:4], first[:4]):
            assert np.all(np.abs(a - b) <= 2 * 2.0 ** -24 * (16 + 6 + 2 * 16))
        # (its exponential: one lse for another, and the result's rounding)
        p = np.abs(first[4]) + np.abs(grad.get())[:, None]
        step = np.finfo(dtype).eps
        assert np.all(np.abs(other[4] - first[4]) <= step * np.abs(first[4]) + 2.0 ** -17 * p + 1e-7)
        # (32 elements in 32 bits, or 64 bits throughout; half of it in the root)
        assert abs(other[5] - first[5]) <= 40 * 2.0 ** -24 * first[5]
        for a, b in zip(other[6:], first[6:]):               # rows as their elements lie
            assert np.array_equal(a, b)
