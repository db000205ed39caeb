"""Layer norms whose arrays lie differently between 16-byte boundaries, and constant rows.

The kernels choose their access width by all arrays of a call together, and copy rows of odd widths in the 16-byte pieces that they lie in, which begin
somewhere else in every array.  Tolerances are those of test_gpu_norm."""
import numpy as np
import pytest

from tests.test_gpu_norm import EPS, U, backward, chain, forward, inputs, kept, place, read, scale_of, within
from tests.test_gpu_ops import env  # noqa: F401

pytestmark = pytest.mark.gpu
# floats behind a boundary: x, gamma, beta or the sum's gradient, dy, y or dresidual, dinput, dgamma, dbeta
PLACES = [(1, 0, 2, 3, 0, 1, 2, 0), (3, 1, 0, 2, 1, 0, 3, 2), (0, 3, 1, 0, 3, 2, 1, 0), (2, 0, 3, 1, 0, 3, 0, 1), (0, 0, 0, 0, 1, 0, 0, 0), (0, 0, 0, 2, 0, 0, 0, 0), (2, 2, 2, 2, 2, 2, 2, 2)]
# one row, few rows (a cluster), more than the rings of all SMs hold
SHAPES = [(1, 33), (700, 33), (5, 130), (300, 130), (2, 1029), (1300, 1029), (9, 1028), (3, 2048), (400, 4097), (7, 8191), (300, 8192), (200, 9001), (160, 8196), (3, 16384), (4, 16387)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("at", PLACES)
def test_layer_norm(env, shape, at):
    x, gamma, beta, dy, _ = inputs(shape)
    X, G, B, DY = (place(env, v, o) for v, o in zip((x, gamma, beta, dy), at))
    Y, DX, DG, DB = (place(env, s, o) for s, o in zip((shape, shape, gamma.shape, gamma.shape), at[4:]))
    env.gpu_op.layer_norm_forward(X, G, B, Y, EPS, env.stream)
    assert env.gpu_op.layer_norm_backward(X, G, DY, DX, DG, DB, EPS, env.stream) == 0
    want, bound = forward(x, gamma, beta)[:2]
    within(read(Y), want, bound, "y")
    for name, arr, w, b in zip(("dx", "dgamma", "dbeta"), (DX, DG, DB), *backward(x, gamma, dy)):
        within(read(arr), w, b, name)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("at", PLACES)
def test_residual_norm(env, shape, at):
    x, gamma, beta, dy, rng = inputs(shape)
    branch, dsum = rng.randn(*shape).astype(np.float32), (0.1 * rng.randn(*shape)).astype(np.float32)
    keep, scale = kept(shape, 0.3, 7), scale_of(0.3)
    X, G, DS, DY, H = (place(env, v, o) for v, o in zip((x, gamma, dsum, dy, branch), at))
    B, S, Y = place(env, beta, at[1]), place(env, shape, at[0]), place(env, shape, at[5])
    DX, DH, DG, DB = (place(env, s, o) for s, o in zip((shape, shape, gamma.shape, gamma.shape), at[4:]))
    state = env.gpu_op.dropout_state(0.3, 7)
    env.gpu_op.dropout_add_layer_norm_forward(H, X, G, B, S, Y, state, EPS, env.stream)
    s = read(S)
    want = x.astype(np.float64) + np.where(keep, branch * scale, 0)
    within(s, want, U * (np.abs(want) + np.abs(branch * scale)), "sum")
    within(read(Y), *forward(s, gamma, beta)[:2], "y")
    assert env.gpu_op.dropout_add_layer_norm_backward(S, G, DY, DS, DH, DX, DG, DB, state, EPS, env.stream) == 0
    (dx, dgamma, dbeta), (bx, bg, bb) = backward(s, gamma, dy)
    total = dx + dsum
    bound = bx + U * np.abs(total)
    within(read(DX), total, bound, "dresidual")
    within(read(DH), np.where(keep, total * scale, 0), np.where(keep, bound * scale + U * np.abs(total * scale), 0), "dinput")
    within(read(DG), dgamma, bg, "dgamma")
    within(read(DB), dbeta, bb, "dbeta")


@pytest.mark.parametrize("D", [3, 100, 768, 2050, 9001, 16400])
@pytest.mark.parametrize("value", [0.0, 12.3, -1e5, 1e15])
def test_constant_rows(env, D, value):
    """What is left of such a row is the error of its mean, e <= n u |value|, the same in every element: normalised it is e / sqrt(e^2 + eps), at most e / sqrt(eps)
    and at most one.  Without an eps the formula is 0 / 0: NaN, or that one.  The rows beside them are what they are alone."""
    rng = np.random.RandomState(D)
    x = np.concatenate([np.full((2, D), value), rng.randn(3, D)]).astype(np.float32)
    gamma, beta, dy = (1 + 0.1 * rng.randn(D)).astype(np.float32), (0.1 * rng.randn(D)).astype(np.float32), rng.randn(5, D).astype(np.float32)
    X, G, B, DY = (env.dev(v) for v in (x, gamma, beta, dy))
    Y, DX = env.empty(x.shape), env.empty(x.shape)
    n = chain(D)
    for eps in (1e-5, 0.0):
        env.gpu_op.layer_norm_forward(X, G, B, Y, eps, env.stream)
        env.gpu_op.layer_norm_backward(X, G, DY, DX, None, None, eps, env.stream)
        y, dx = Y.asnumpy(), DX.asnumpy()
        within(y[2:], *forward(x[2:], gamma, beta, eps)[:2], "y")
        (want, _, _), (bound, _, _) = backward(x[2:], gamma, dy[2:], eps)
        within(dx[2:], want, bound, "dx")
        left = min(1.0, n * U * abs(value) / np.sqrt(eps)) if eps else 1.0
        bound = left * (1 + (n + 8) * U) * np.abs(gamma) + 4 * U * (np.abs(gamma) + np.abs(beta))
        assert ((np.abs(y[:2] - beta) <= bound) | (np.isnan(y[:2]) if eps == 0 else False)).all()
