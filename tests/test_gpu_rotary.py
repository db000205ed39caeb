"""Rotary positions, alone and behind the norms of heads, against the formulas in 64 bits.

Tolerances count roundings, u = 2^-24 each: an angle reduced to an eighth of a turn is rounded by u / 2 of less than 1, its sine and cosine by
2 u, the amplitude's product by u, and a rotated value is two products and a sum of those: 8 u A (|a| + |b|).  A head's sum of squares has chains of 8
elements in a thread and 5 of shuffles, its root and reciprocal 2 u: 20 u of the normed value.  dgamma is added up over at most tokens x heads / 100 +
200 terms in a row (every fourth of an SM's share, up to 64 groups of a block, eights of the blocks and up to 32 sums of those)."""
import ctypes

import numpy as np
import pytest

from oracle import ops
from tests.test_gpu_norm import place, read, view, within
from tests.test_gpu_ops import env  # noqa: F401

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-6

# head_dim, rotated, layout, scaling
SHAPES = [(1, 0, "half", "none"), (2, 2, "half", "none"), (3, 2, "interleaved", "none"), (16, 16, "half", "linear"), (33, 20, "half", "none"), (64, 64, "interleaved", "parts"),
          (64, 64, "half", "stretched"), (72, 40, "interleaved", "none"), (80, 64, "half", "parts"), (90, 30, "half", "linear"), (96, 96, "interleaved", "stretched"),
          (128, 128, "half", "parts"), (128, 0, "half", "none"), (130, 66, "half", "none"), (256, 256, "half", "none"), (256, 128, "interleaved", "linear"), (251, 250, "interleaved", "none")]


def state_of(env, D, rotated, layout, scaling):
    return env.gpu_op.rotary_state(D, rotated, layout, 10000.0, scaling, 4.0, 512)


def turns_of(env, D, rotated, scaling, tokens, length, start, positions):
    f, amplitude = env.gpu_op.rotary_frequencies(rotated, 10000.0, scaling, 4.0, 512)
    return ops.rotary_angles(tokens, length, start, positions, f), amplitude


def spread(x, D, rotated, layout, amplitude):
    """A (|a| + |b|) of every element's pair; behind the rotated part the element's own magnitude."""
    y = np.abs(x.reshape(x.shape[0], -1, D))
    m = rotated // 2
    z = y.copy()
    a, b = (slice(0, m), slice(m, 2 * m)) if layout == "half" else (slice(0, 2 * m, 2), slice(1, 2 * m, 2))
    z[..., a] = z[..., b] = amplitude * (y[..., a] + y[..., b])
    return z.reshape(x.shape)


@pytest.mark.parametrize("D,rotated,layout,scaling", SHAPES)
@pytest.mark.parametrize("batch,length,heads,start,given,misaligned", [(1, 1, 1, 0, False, 0), (3, 7, 3, 5, False, 1), (2, 40, 12, 123456, False, 2), (1, 301, 5, 0, True, 0)])
def test_rotation(env, D, rotated, layout, scaling, batch, length, heads, start, given, misaligned):
    rng = np.random.RandomState(D + length)
    tokens = batch * length
    x = rng.randn(tokens, heads * D).astype(np.float32)
    positions = (rng.rand(tokens) * 3e6 - 1e6).astype(np.float32) if given else None
    angles, amplitude = turns_of(env, D, rotated, scaling, tokens, length, start, positions)
    state = state_of(env, D, rotated, layout, scaling)
    X, Y, DX = place(env, x, misaligned), place(env, x.shape, misaligned), place(env, x.shape, misaligned)
    P = None if positions is None else place(env, positions)
    env.gpu_op.rotary_forward(X, P, Y, length, start, state, env.stream)
    env.gpu_op.rotary_backward(X, P, DX, length, start, state, env.stream)
    env.gpu_op.device_synchronize()
    x = x.astype(np.float64)
    bound = 8 * U * spread(x, D, rotated, layout, amplitude) + 1e-30
    within(read(Y), ops.rotary(x, D, angles, amplitude, layout), bound, "y")
    within(read(DX), ops.rotary(x, D, angles, amplitude, layout, back=True), bound, "dx")
    m = rotated
    assert np.array_equal(read(Y).reshape(tokens, heads, D)[..., m:], x.reshape(tokens, heads, D)[..., m:])


def norm_bounds(x, gamma, dy, D, rotated, layout, angles, amplitude):
    x, gamma, dy = (np.asarray(v, np.float64) for v in (x, gamma, dy))
    y = ops.head_norm_rotary(x, gamma, D, angles, amplitude, layout, EPS)
    dx, dgamma = ops.head_norm_rotary_backward(x, gamma, dy, D, angles, amplitude, layout, EPS)
    h = x.reshape(x.shape[0], -1, D)
    inv = 1 / np.sqrt((h * h).mean(-1, keepdims=True) + EPS)
    n = h * inv
    ey = 30 * U * spread((n * gamma).reshape(x.shape), D, rotated, layout, amplitude)
    u = ops.rotary(dy, D, angles, amplitude, layout, back=True).reshape(h.shape)
    eu = 8 * U * spread(dy, D, rotated, layout, amplitude).reshape(h.shape)
    g = gamma * u
    eg = np.abs(gamma) * eu + U * np.abs(g)
    mean = lambda v: v.mean(-1, keepdims=True)     # noqa: E731
    dot = mean(g * n)
    edot = mean(eg * np.abs(n) + 20 * U * np.abs(g * n)) + 20 * U * mean(np.abs(g * n))
    edx = inv * (eg + np.abs(n) * edot + 24 * U * np.abs(n * dot) + 2 * U * np.abs(g)) + 24 * U * np.abs(dx).reshape(h.shape)
    chain = h.shape[0] * h.shape[1] / 100 + 200
    edg = (eu * np.abs(n) + (20 + chain) * U * np.abs(u * n)).sum((0, 1))
    return (y, dx, dgamma), (ey + 1e-30, edx.reshape(x.shape) + 1e-30, edg + 1e-30)


def both(env, q, k, gq, gk, dq, dk, positions, length, start, state, misaligned=0, which=(True,) * 4):
    on = lambda v: None if v is None else place(env, v, misaligned)       # noqa: E731
    Q, K, GQ, GK, DQ, DK, P = (on(v) for v in (q, k, gq, gk, dq, dk, positions))
    YQ, YK = place(env, q.shape, misaligned), None if k is None else place(env, k.shape, misaligned)
    env.gpu_op.head_norm_rotary_forward(Q, K, GQ, GK, P, YQ, YK, length, start, EPS, state, env.stream)
    results = [place(env, v.shape, misaligned) if w and v is not None else None for v, w in zip((q, k, gq, gk), which)]
    assert not env.gpu_op.head_norm_rotary_backward(Q, K, GQ, GK, P, DQ, DK, *results, length, start, EPS, state, env.stream)
    env.gpu_op.device_synchronize()
    return [None if v is None else read(v) for v in (YQ, YK, *results)]


@pytest.mark.parametrize("D,rotated,layout,scaling", SHAPES)
@pytest.mark.parametrize("tokens,length,heads,kv_heads,start,misaligned", [(1, 1, 1, 1, 7, 0), (30, 10, 6, 2, 0, 1), (64, 64, 8, 8, 100000, 0), (700, 350, 3, 1, 0, 2)])
def test_normed_heads(env, D, rotated, layout, scaling, tokens, length, heads, kv_heads, start, misaligned):
    rng = np.random.RandomState(D + tokens)
    q, k, dq, dk = (rng.randn(tokens, n * D).astype(np.float32) for n in (heads, kv_heads, heads, kv_heads))
    q *= np.exp(rng.randn(*q.shape)).astype(np.float32)
    gq, gk = ((1 + 0.3 * rng.randn(D)).astype(np.float32) for _ in range(2))
    angles, amplitude = turns_of(env, D, rotated, scaling, tokens, length, start, None)
    got = both(env, q, k, gq, gk, dq, dk, None, length, start, state_of(env, D, rotated, layout, scaling), misaligned)
    for name, x, g, d, at in (("q", q, gq, dq, (0, 2, 4)), ("k", k, gk, dk, (1, 3, 5))):
        want, bound = norm_bounds(x, g, d, D, rotated, layout, angles, amplitude)
        for what, w, e, i in zip(("y", "dx", "dgamma"), want, bound, at):
            within(got[i], w, e, what + " of " + name)


def test_queries_alone_and_one_gradient_alone(env):
    rng = np.random.RandomState(4)
    q, k, dq, dk = (rng.randn(900, n * 64).astype(np.float32) for n in (6, 2, 6, 2))
    gq, gk = rng.randn(64).astype(np.float32), rng.randn(64).astype(np.float32)
    state = state_of(env, 64, 64, "half", "none")
    at = (rng.rand(900) * 1000).astype(np.float32)
    whole = both(env, q, k, gq, gk, dq, dk, at, 450, 3, state)
    again = both(env, q, k, gq, gk, dq, dk, at, 450, 3, state)
    for a, b in zip(whole, again):
        assert np.array_equal(a, b)
    alone = both(env, q, None, gq, None, dq, None, at, 450, 3, state)
    assert np.array_equal(alone[0], whole[0]) and np.array_equal(alone[2], whole[2])
    # dgamma is added up over as many blocks as there are for it
    np.testing.assert_allclose(alone[4], whole[4], rtol=0, atol=1e-4)
    for i in range(4):
        one = both(env, q, k, gq, gk, dq, dk, at, 450, 3, state, which=[j == i for j in range(4)])
        assert all((v is None) == (j != i) for j, v in enumerate(one[2:]))
        if i < 2:
            assert np.array_equal(one[2 + i], whole[2 + i])
        else:
            np.testing.assert_allclose(one[2 + i], whole[2 + i], rtol=0, atol=1e-4)


def test_no_tokens(env):
    nd, op = env.nd, env.gpu_op
    state = op.rotary_state(8)
    E, G, D = nd.empty((0, 16), env.ctx), nd.array(np.ones(8, np.float32), env.ctx), nd.array(np.ones(8, np.float32), env.ctx)
    outs = [nd.empty((0, 16), env.ctx) for _ in range(4)]
    op.rotary_forward(E, None, outs[0], 4, 0, state, env.stream)
    op.head_norm_rotary_forward(E, E, G, G, None, outs[0], outs[1], 4, 0, EPS, state, env.stream)
    DK = nd.array(np.ones(8, np.float32), env.ctx)
    assert not op.head_norm_rotary_backward(E, E, G, G, None, E, E, outs[2], outs[3], D, DK, 4, 0, EPS, state, env.stream)
    assert not D.asnumpy().any() and not DK.asnumpy().any()


def test_a_token_that_is_not_finite_stays_by_itself(env):
    rng = np.random.RandomState(1)
    q, k = rng.randn(50, 4 * 32).astype(np.float32), rng.randn(50, 2 * 32).astype(np.float32)
    g, state = np.ones(32, np.float32), state_of(env, 32, 32, "half", "none")
    clean = both(env, q, k, g, g, q, k, None, 50, 0, state)
    for bad in (np.nan, np.inf):
        q2 = q.copy()
        q2[7, 33] = bad                            # head 1 of token 7
        got = both(env, q2, k, g, g, q, k, None, 50, 0, state)
        for i in (0, 2):
            heads, want = got[i].reshape(50, 4, 32), clean[i].reshape(50, 4, 32)
            # an infinity makes the reciprocal root 0: the head's finite elements become 0 by the formula, infinity times 0 NaN
            assert not np.isfinite(heads[7, 1]).all() and (np.isnan(bad) <= np.isnan(heads[7, 1]).all())
            heads[7, 1] = want[7, 1]
            assert np.array_equal(heads, want)
        assert np.array_equal(got[1], clean[1]) and np.array_equal(got[3], clean[3]) and np.array_equal(got[5], clean[5]) and np.isnan(got[4]).any()


def test_a_state_used_again_with_other_values(env):
    rng = np.random.RandomState(2)
    x = rng.randn(20, 64).astype(np.float32)
    X, Y = place(env, x), place(env, x.shape)
    state = env.gpu_op.rotary_state(64)
    env.gpu_op.rotary_forward(X, None, Y, 20, 0, state, env.stream)
    assert env.gpu_op.rotary_state(16, 8, "interleaved", state=state) is state
    env.gpu_op.rotary_forward(X, None, Y, 20, 0, state, env.stream)
    env.gpu_op.device_synchronize()
    f, amplitude = env.gpu_op.rotary_frequencies(8)
    want = ops.rotary(x.astype(np.float64), 16, ops.rotary_angles(20, 20, 0, None, f), amplitude, "interleaved")
    within(read(Y), want, 8 * U * spread(x, 16, 8, "interleaved", amplitude) + 1e-30, "y")


def test_products_take_the_maxima_that_these_kernels_leave(env):
    """A product behind the rotation scales by the largest magnitude that the rotation noted: the bits of a product that looks for it itself."""
    rng = np.random.RandomState(3)
    op, nd = env.gpu_op, env.nd
    x, w = (1e3 * rng.randn(512, 256)).astype(np.float32), rng.randn(256, 384).astype(np.float32)
    k, g = (1e-3 * rng.randn(512, 128)).astype(np.float32), np.full(64, 1e4, np.float32)
    X, W, Y, Z, K, G = (nd.array(v, env.ctx) if isinstance(v, np.ndarray) else nd.empty(v, env.ctx) for v in (x, w, x.shape, (512, 384), k, g))
    YK, ZK, WK = nd.empty(k.shape, env.ctx), nd.empty((512, 384), env.ctx), nd.array(w[:128].copy(), env.ctx)
    state = op.rotary_state(64)
    op.set_contraction_path(2)
    try:
        for _ in range(3):
            op.head_norm_rotary_forward(X, K, G, G, None, Y, YK, 512, 0, EPS, state, env.stream)
            op.matrix_multiply(Y, False, W, False, Z, env.cublas, env.stream)
            op.matrix_multiply(YK, False, WK, False, ZK, env.cublas, env.stream)
        noted = Z.asnumpy(), ZK.asnumpy()
        for y, w_, z, at in ((Y, W, Z, 0), (YK, WK, ZK, 1)):
            fresh = nd.array(y.asnumpy(), env.ctx)
            op.matrix_multiply(fresh, False, w_, False, z, env.cublas, env.stream)
            assert np.array_equal(z.asnumpy(), noted[at])
    finally:
        op.set_contraction_path(0)


@pytest.mark.parametrize("offset", [5, 64])
def test_part_of_a_block_that_was_freed(env, offset):
    """What is known of an array that was a part of another goes with that: the next array there has other magnitudes."""
    M, K, N = 1300, 768, 256
    rng = np.random.RandomState(0)

    def part(value):
        whole = np.zeros(M * K + 128, np.float32)
        whole[offset:offset + M * K] = value.ravel()
        return view(env, env.nd.array(whole, env.ctx), offset, (M, K))
    env.gpu_op.set_contraction_path(2)
    small = part((2.0 ** -90 * rng.randn(M, K)).astype(np.float32))
    out = part(np.zeros((M, K), np.float32))
    env.gpu_op.rotary_forward(small, None, out, M, 0, env.gpu_op.rotary_state(64), env.stream)
    env.gpu_op.device_synchronize()
    at = out.data_ptr
    del out
    a, b = rng.randn(M, K).astype(np.float32), rng.randn(K, N).astype(np.float32)
    A, B, C = part(a), env.nd.array(b, env.ctx), env.nd.empty((M, N), env.ctx)
    assert A.data_ptr == at                      # the block is used again
    env.gpu_op.matrix_multiply(A, False, B, False, C, env.cublas, env.stream)
    env.gpu_op.set_contraction_path(0)
    want, magnitude = a.astype(np.float64) @ b.astype(np.float64), np.abs(a).astype(np.float64) @ np.abs(b).astype(np.float64)
    within(C.asnumpy(), want, (4 + 3 * K / 8) * U * magnitude, "product")
