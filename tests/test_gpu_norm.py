"""Layer normalisation, alone and behind a residual sum of a dropped-out branch, against the formulas in 64 bits.

Tolerances are bounds of fp32 rounding (u = 2^-24 a step): N is the longest chain of additions of a row's sums (32 elements in a
thread, 5 shuffles and at most 16 warps; D / 512 elements a thread in rows longer than the registers hold).  An error of the mean of
N u mean|x| shifts every x - mean; what follows from it is carried through the formulas below.  Sums over rows have chains of at most
rows / 100 + 96 terms (148 SMs share the rows)."""
import ctypes

import numpy as np
import pytest

from tests.test_gpu_ops import env  # noqa: F401

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-5


def kept(shape, rate, seed):
    """The mask of the library's dropout generator."""
    z = np.arange(1, int(np.prod(shape)) + 1, dtype=np.uint64)
    with np.errstate(over="ignore"):
        z = z * np.uint64(0x9E3779B97F4A7C15) + np.uint64(seed) * np.uint64(0xD1342543DE82EF95)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        z ^= z >> np.uint64(31)
    return (((z >> np.uint64(40)).astype(np.float32) * np.float32(2.0 ** -24)) >= np.float32(rate)).reshape(shape)


def scale_of(rate):
    return np.float64(np.float32(1) / (np.float32(1) - np.float32(rate)))


def chain(D):
    return 64 + D // 512


def forward(x, gamma, beta, eps=EPS):
    """(y, bound of its error)"""
    x, gamma, beta = (np.asarray(v, np.float64) for v in (x, gamma, beta))
    D, n = x.shape[-1], chain(x.shape[-1])
    mean = x.mean(-1, keepdims=True)
    inv = 1 / np.sqrt(((x - mean) ** 2).mean(-1, keepdims=True) + eps)
    xh = (x - mean) * inv
    dxh = U * (inv * (n * np.abs(x).mean(-1, keepdims=True) + 3 * np.abs(x)) + (n + 8) * np.abs(xh))
    # an error e of the mean adds e^2 to the variance: second order, and with a variance far below eps next to nothing
    return gamma * xh + beta, np.abs(gamma) * dxh + 4 * U * (np.abs(gamma * xh) + np.abs(beta)) + 1e-30, xh, inv, dxh


def backward(x, gamma, dy, eps=EPS):
    _, _, xh, inv, dxh = forward(x, gamma, gamma, eps)
    gamma, dy = np.asarray(gamma, np.float64), np.asarray(dy, np.float64)
    D, n = x.shape[-1], chain(x.shape[-1])
    rows = int(np.prod(x.shape[:-1]))
    g = gamma * dy
    mean = lambda v: v.mean(-1, keepdims=True)     # noqa: E731
    mg, mgx = mean(g), mean(g * xh)
    dx = inv * (g - mg - xh * mgx)
    dmgx = U * (n + 4) * mean(np.abs(g * xh)) + mean(np.abs(g) * dxh)
    ddx = inv * (U * (6 * np.abs(g) + (n + 6) * mean(np.abs(g)) + 6 * np.abs(xh * mgx)) + np.abs(xh) * dmgx + dxh * np.abs(mgx)) + (n + 8) * U * np.abs(dx) + 1e-30
    flat = lambda v: v.reshape(rows, D)            # noqa: E731
    nr = rows / 100 + 96
    dgamma, dbeta = flat(dy * xh).sum(0), flat(dy).sum(0)
    ddgamma = flat(np.abs(dy) * dxh).sum(0) + U * nr * flat(np.abs(dy * xh)).sum(0) + 1e-30
    return (dx, dgamma, dbeta), (ddx, ddgamma, U * nr * flat(np.abs(dy)).sum(0) + 1e-30)


def within(got, want, bound, what):
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape, what
    over = np.abs(got - want) - bound
    assert not got.size or over.max() <= 0, "%s: off by %.3e at %s, where %.3e is allowed" % (
        what, np.abs(got - want).flat[over.argmax()], np.unravel_index(over.argmax(), over.shape), np.broadcast_to(bound, over.shape).flat[over.argmax()])


def inputs(shape, seed=0):
    rng = np.random.RandomState(seed + sum(shape))
    D = shape[-1]
    spread = np.exp(0.5 * rng.randn(D)) * np.where(rng.rand(D) < 0.02, 10, 1)
    x = (rng.randn(*shape) * spread + 0.3 * rng.randn(D)).astype(np.float32)
    return x, (1 + 0.1 * rng.randn(D)).astype(np.float32), (0.1 * rng.randn(D)).astype(np.float32), (0.1 * rng.randn(*shape)).astype(np.float32), rng


def view(env, array, offset_floats, shape):
    """An array over a part of another one's memory."""
    c = env.nd.DLArray()
    dims = (ctypes.c_int64 * len(shape))(*shape)
    c.data, c.ctx, c.ndim, c.shape = array.data_ptr + 4 * offset_floats, env.ctx, len(shape), ctypes.cast(dims, ctypes.POINTER(ctypes.c_int64))
    v = env.nd.NDArray(ctypes.pointer(c))
    v.is_freed, v._owner = True, (array, dims)
    return v


def place(env, value, misaligned=0):
    """`value` (or an empty array of that shape) on the GPU, `misaligned` floats behind a 16-byte boundary, NaN around it."""
    shape = value if isinstance(value, tuple) else value.shape
    size = int(np.prod(shape))
    whole = np.full(size + 12, np.nan, np.float32)
    if not isinstance(value, tuple):
        whole[4 + misaligned:4 + misaligned + size] = value.ravel()
    return view(env, env.nd.array(whole, env.ctx), 4 + misaligned, shape)


def read(arr):
    """What the array holds; fails if anything beside it was written."""
    whole = arr._owner[0].asnumpy()
    at = (arr.data_ptr - arr._owner[0].data_ptr) // 4
    size = int(np.prod(arr.shape))
    assert np.isnan(whole[:at]).all() and np.isnan(whole[at + size:]).all(), "written outside the array"
    return whole[at:at + size].reshape(arr.shape)


SHAPES = [(1, 1), (5, 1), (3, 2), (64, 3), (1, 4), (9, 5), (2, 31), (33, 32), (7, 33), (70, 127), (1, 128), (300, 129), (17, 130), (64, 256), (3, 257), (1003, 500), (40, 512),
          (5, 516), (4, 3, 5, 1000), (129, 1023), (6, 1024), (2, 1, 1028), (1, 2047), (300, 2048), (3, 2050), (2, 4096), (700, 4096), (5, 4097), (150, 8190), (2, 8191), (3, 8192), (1, 8196),
          (2, 16383), (170, 16384), (3, 16385), (1, 16388), (2, 40001), (2500, 64), (1,), (7,), (2048,), (310, 9001), (400, 12290), (160, 8194), (149, 12288), (1, 12292)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("misaligned", [0, 1])
def test_layer_norm(env, shape, misaligned):
    x, gamma, beta, dy, _ = inputs(shape)
    X, G, B, DY = (place(env, v, misaligned) for v in (x, gamma, beta, dy))
    Y, DX, DG, DB = (place(env, s, misaligned) for s in (shape, shape, gamma.shape, gamma.shape))
    env.gpu_op.layer_norm_forward(X, G, B, Y, EPS, env.stream)
    assert env.gpu_op.layer_norm_backward(X, G, DY, DX, DG, DB, EPS, env.stream) == 0
    want, bound = forward(x, gamma, beta)[:2]
    within(read(Y), want, bound, "y")
    for name, arr, w, b in zip(("dx", "dgamma", "dbeta"), (DX, DG, DB), *backward(x, gamma, dy)):
        within(read(arr), w, b, name)


@pytest.mark.parametrize("shape", [(1, 1), (64, 3), (1, 4), (7, 33), (300, 129), (64, 256), (17, 516), (4, 3, 5, 1000), (6, 1024), (300, 2048), (3, 2050), (700, 4096), (5, 8191), (3, 8192),
                                   (2, 16384), (3, 16385), (2500, 64), (310, 9001), (300, 12290), (160, 8196)])
@pytest.mark.parametrize("rate,seed,misaligned", [(0.0, 0, 0), (0.1, 7, 0), (0.5, 100, 1), (0.9, 2 ** 31 - 1, 0)])
def test_residual_norm(env, shape, rate, seed, misaligned):
    x, gamma, beta, dy, rng = inputs(shape)
    branch, dsum = rng.randn(*shape).astype(np.float32), (0.1 * rng.randn(*shape)).astype(np.float32)
    keep, scale = kept(shape, rate, seed), scale_of(rate)
    H, X, G, B, DY, DS = (place(env, v, misaligned) for v in (branch, x, gamma, beta, dy, dsum))
    S, Y, DH, DX, DG, DB = (place(env, s, misaligned) for s in (shape, shape, shape, shape, gamma.shape, gamma.shape))
    state = env.gpu_op.dropout_state(rate, seed)
    env.gpu_op.dropout_add_layer_norm_forward(H, X, G, B, S, Y, state, EPS, env.stream)
    s = read(S)
    want = x.astype(np.float64) + np.where(keep, branch * scale, 0)
    within(s, want, U * (np.abs(want) + np.abs(branch * scale)), "sum")
    y, bound = forward(s, gamma, beta)[:2]
    within(read(Y), y, bound, "y")
    assert env.gpu_op.dropout_add_layer_norm_backward(S, G, DY, DS, DH, DX, DG, DB, state, EPS, env.stream) == 0
    (dx, dgamma, dbeta), (bx, bg, bb) = backward(s, gamma, dy)
    total = dx + dsum
    bound = bx + U * np.abs(total)
    within(read(DX), total, bound, "dresidual")
    within(read(DH), np.where(keep, total * scale, 0), np.where(keep, bound * scale + U * np.abs(total * scale), 0), "dinput")
    within(read(DG), dgamma, bg, "dgamma")
    within(read(DB), dbeta, bb, "dbeta")
    # the mask is that of the dropout operator
    out = env.nd.empty(shape, env.ctx)
    if len(shape) == 2:
        inputd = env.gpu_op.get_input_descriptor(shape, "NCHW")
        env.gpu_op.dropout_forward(env.nd.array(np.ones(shape, np.float32), env.ctx), out, "NCHW", rate, seed, inputd, env.cudnn, env.stream)
        assert np.array_equal(out.asnumpy() != 0, keep)


@pytest.mark.parametrize("shape", [(37, 256), (5, 2050), (3, 16400)])
def test_results_that_are_not_asked_for(env, shape):
    x, gamma, beta, dy, rng = inputs(shape)
    X, G, B, DY, DS = (env.nd.array(v, env.ctx) for v in (x, gamma, beta, dy, dy[::-1].copy()))
    state = env.gpu_op.dropout_state(0.3, 5)

    def call(names, with_sum=True):
        a = {n: place(env, gamma.shape if n in ("dg", "db") else shape) if n in names else None for n in ("dh", "dx", "dg", "db")}
        env.gpu_op.dropout_add_layer_norm_backward(X, G, DY, DS if with_sum else None, a["dh"], a["dx"], a["dg"], a["db"], state, EPS, env.stream)
        p = {n: place(env, gamma.shape if n in ("dg", "db") else shape) if n in names else None for n in ("dx", "dg", "db")}
        env.gpu_op.layer_norm_backward(X, G, DY, p["dx"], p["dg"], p["db"], EPS, env.stream)
        return {n: read(v) for n, v in a.items() if v is not None}, {n: read(v) for n, v in p.items() if v is not None}

    whole, plain = call(("dh", "dx", "dg", "db"))
    for names in [(), ("dh",), ("dx",), ("dg",), ("db",), ("dg", "db"), ("dh", "db"), ("dx", "dg")]:
        for got, want in zip(call(names), (whole, plain)):
            for n, v in got.items():
                assert np.array_equal(v, want[n]), (names, n)
    # without a gradient from elsewhere the residual's gradient is the normalisation's own
    assert np.array_equal(call(("dx",), with_sum=False)[0]["dx"], plain["dx"])
    # the sum alone
    S, S2, Y = (place(env, shape) for _ in range(3))
    env.gpu_op.dropout_add_layer_norm_forward(DY, X, G, B, S, None, state, EPS, env.stream)
    env.gpu_op.dropout_add_layer_norm_forward(DY, X, G, B, S2, Y, state, EPS, env.stream)
    assert np.array_equal(read(S), read(S2))


@pytest.mark.parametrize("shape", [(301, 260), (1501, 1024), (9, 5000), (37, 16392)])
def test_the_same_bits_every_time_and_on_another_stream(env, shape):
    x, gamma, beta, dy, _ = inputs(shape)
    X, G, B, DY = (env.nd.array(v, env.ctx) for v in (x, gamma, beta, dy))
    other = env.gpu_op.create_cudaStream()
    seen = []
    for stream in (env.stream, other, env.stream, None):
        Y, DX, DG, DB = (env.nd.empty(s, env.ctx) for s in (shape, shape, gamma.shape, gamma.shape))
        env.gpu_op.device_synchronize()
        env.gpu_op.layer_norm_forward(X, G, B, Y, EPS, stream)
        env.gpu_op.layer_norm_backward(X, G, DY, DX, DG, DB, EPS, stream)
        env.gpu_op.device_synchronize()
        seen.append([v.asnumpy() for v in (Y, DX, DG, DB)])
    env.gpu_op.destroy_cudaStream(other)
    for again in seen[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(seen[0], again))


@pytest.mark.parametrize("D", [96, 1001, 16390])
def test_a_row_that_is_not_finite_stays_by_itself(env, D):
    x, gamma, beta, dy, _ = inputs((6, D))
    outs = []
    for bad in (None, np.inf, np.nan):
        v = x.copy()
        if bad is not None:
            v[2, D // 2] = bad
        X, G, B, DY = (env.nd.array(a, env.ctx) for a in (v, gamma, beta, dy))
        Y, DX = env.nd.empty(x.shape, env.ctx), env.nd.empty(x.shape, env.ctx)
        env.gpu_op.layer_norm_forward(X, G, B, Y, EPS, env.stream)
        env.gpu_op.layer_norm_backward(X, G, DY, DX, None, None, EPS, env.stream)
        outs.append((Y.asnumpy(), DX.asnumpy()))
    for y, dx in outs[1:]:
        for got, clean in ((y, outs[0][0]), (dx, outs[0][1])):
            assert np.isnan(got[2]).all()
            assert np.array_equal(np.delete(got, 2, 0), np.delete(clean, 2, 0))


def test_offsets_far_above_the_spread_and_constant_rows(env):
    """The mean is taken off before anything is squared: an offset of 1000 spreads costs what rounding of x itself costs."""
    rng = np.random.RandomState(3)
    x = np.concatenate([(1000 + rng.randn(4, 768)), np.full((3, 768), 12.3), np.zeros((1, 768))]).astype(np.float32)
    gamma, beta = np.ones(768, np.float32), np.zeros(768, np.float32)
    Y = env.nd.empty(x.shape, env.ctx)
    X, G, B = (env.nd.array(v, env.ctx) for v in (x, gamma, beta))
    for eps in (1e-5, 1e-2):
        env.gpu_op.layer_norm_forward(X, G, B, Y, eps, env.stream)
        want, bound, _, inv, _ = forward(x, gamma, beta, eps)
        within(Y.asnumpy(), want, bound, "y")
    assert np.array_equal(Y.asnumpy()[-1], beta)


def test_no_rows_and_no_columns(env):
    nd, op = env.nd, env.gpu_op
    G, B, DG, DB = (nd.array(np.ones(5, np.float32), env.ctx) for _ in range(4))
    X, Y = nd.empty((0, 5), env.ctx), nd.empty((0, 5), env.ctx)
    DX, DY = nd.empty((0, 5), env.ctx), nd.empty((0, 5), env.ctx)
    op.layer_norm_forward(X, G, B, Y, EPS, env.stream)
    op.layer_norm_backward(X, G, DY, DX, DG, DB, EPS, env.stream)
    assert not DG.asnumpy().any() and not DB.asnumpy().any()
    X, Y, G, B = nd.empty((4, 0), env.ctx), nd.empty((4, 0), env.ctx), nd.empty((0,), env.ctx), nd.empty((0,), env.ctx)
    op.layer_norm_forward(X, G, B, Y, EPS, env.stream)


@pytest.mark.parametrize("shape", [(6, 40), (3, 1030)])
def test_gradients_against_differences(env, shape):
    """Central differences of sum(y * c) in 64 bits (the formula's own, step 1e-5 relative): truncation 1e-9, cancellation 1e-10."""
    x, gamma, beta, c, rng = inputs(shape)
    X, G, DY = (env.nd.array(v, env.ctx) for v in (x, gamma, c))
    DX, DG, DB = (env.nd.empty(s, env.ctx) for s in (shape, gamma.shape, gamma.shape))
    env.gpu_op.layer_norm_backward(X, G, DY, DX, DG, DB, EPS, env.stream)
    loss = lambda x, g, b: float((forward(x, g, b)[0] * c).sum())     # noqa: E731
    (_, _, _), (bx, bg, bb) = backward(x, gamma, c)
    a64 = [v.astype(np.float64) for v in (x, gamma, beta)]
    for k, (got, bound) in enumerate(((DX.asnumpy(), bx), (DG.asnumpy(), bg), (DB.asnumpy(), bb))):
        for _ in range(6):
            at = tuple(rng.randint(0, n) for n in got.shape)
            sides = []
            for step in (1e-5, -1e-5):
                moved = [v.copy() for v in a64]
                moved[k][at] += step
                sides.append(loss(*moved))
            want = (sides[0] - sides[1]) / 2e-5
            assert abs(got[at] - want) <= bound[at] + 1e-7 * (1 + abs(want)), (k, at, got[at], want)


def test_elements_beyond_32_bits(env):
    """The last rows of an array of 2^31 + elements.  The numbers are a dropout of ones, made on the GPU."""
    D = 4096
    rows = (1 << 31) // D + 130
    op, nd = env.gpu_op, env.nd
    X, Y = nd.empty((rows, D), env.ctx), nd.empty((rows, D), env.ctx)
    if isinstance(X, int) or isinstance(Y, int):
        pytest.skip("not enough device memory")
    op.array_set(Y, 1.0, env.stream)
    op.dropout_forward(Y, X, "NCHW", 0.5, 3, op.get_input_descriptor((rows, D), "NCHW"), env.cudnn, env.stream)
    rng = np.random.RandomState(0)
    gamma, beta = (1 + 0.1 * rng.randn(D)).astype(np.float32), rng.randn(D).astype(np.float32)
    G, B, DG, DB = nd.array(gamma, env.ctx), nd.array(beta, env.ctx), nd.empty((D,), env.ctx), nd.empty((D,), env.ctx)
    last = slice((rows - 3) * D, rows * D)
    x = view(env, X, last.start, (3, D)).asnumpy()
    op.layer_norm_forward(X, G, B, Y, EPS, env.stream)
    y, bound = forward(x, gamma, beta)[:2]
    within(view(env, Y, last.start, (3, D)).asnumpy(), y, bound, "y")
    # backward in place of y: the gradient is x itself
    assert op.layer_norm_backward(X, G, X, Y, DG, DB, EPS, env.stream) == 0
    (dx, _, _), (bx, _, _) = backward(x, gamma, x)
    within(view(env, Y, last.start, (3, D)).asnumpy(), dx, bx, "dx")
    # dbeta is the sum of x: twice the count of kept elements, exact in fp32 up to 2^24
    assert np.all(np.abs(DB.asnumpy() - rows) < 8 * np.sqrt(rows))
    del X, Y
    op.release_cached_memory()
