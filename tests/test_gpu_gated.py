"""The gated dense layer, and graphs of it with layer norms, on the GPU.

Tolerances: a product is within 1e-4 |want| + 8 u sum|a||b| (u = 2^-24), the bound of every dense contraction here; what follows from it is
held to the formulas in 64 bits on the projections that the call itself left, a few roundings each (the exponential, the error
function, the division: 2 to 4 u; erfc far below zero has its argument's rounding times 2 x^2)."""
import numpy as np
import pytest

from tests.test_gpu_norm import place, read, view, within
from tests.test_gpu_ops import close_dot, env  # noqa: F401

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ACTIVATIONS = ["sigmoid", "relu", "tanh", "silu", "gelu"]


def inputs(M, K, F, seed=0):
    rng = np.random.RandomState(seed + M + K + F)
    return rng.randn(M, K).astype(np.float32), (rng.randn(K, 2 * F) * max(K, 1) ** -0.5).astype(np.float32), (0.1 * rng.randn(M, F)).astype(np.float32)


def value_bound(activation, g):
    """(value, derivative, bounds of their errors)"""
    from oracle import ops
    value, slope = ops.gate(activation, g)
    far = 2 * np.minimum(g, 0) ** 2 if activation == "gelu" else np.abs(g) if activation in ("sigmoid", "silu", "tanh") else 0
    # the derivative of silu and gelu is a sum of two terms of at most (1 + |g|)
    parts = np.abs(slope) if activation in ("sigmoid", "relu", "tanh") else np.abs(value / np.where(g == 0, 1, g)) + np.abs(slope - value / np.where(g == 0, 1, g))
    return value, slope, (8 + far) * U * np.abs(value) + 1e-37, (12 + 2 * far) * U * parts + 1e-37


def check(env, M, K, F, activation, misaligned=0, path=0, arithmetic="3xfp16", seed=0):
    x, w, dout = inputs(M, K, F, seed)
    op = env.gpu_op
    X, W, D = (place(env, v, misaligned) for v in (x, w, dout))
    Z, H, H2, DX, DW = (place(env, s, misaligned) for s in ((M, 2 * F), (M, F), (M, F), (M, K), (K, 2 * F)))
    op.set_contraction_path(path)
    op.set_tensor_arithmetic(arithmetic)
    try:
        assert op.gated_linear_forward(X, W, Z, H, activation, env.stream) == 0
        assert op.gated_linear_forward(X, W, None, H2, activation, env.stream) == 0
        assert op.gated_linear_backward(X, W, Z, D, DX, DW, activation, env.stream) == 0
        env.gpu_op.device_synchronize()
    finally:
        op.set_contraction_path(0)
        op.set_tensor_arithmetic("3xfp16")
    x64, w64, d64 = x.astype(np.float64), w.astype(np.float64), dout.astype(np.float64)
    z = read(Z)
    if not z.size:
        return
    close_dot(z, x64 @ w64, np.abs(x64) @ np.abs(w64), what="gates")
    z = z.astype(np.float64)
    g, v = z[:, :F], z[:, F:]
    value, slope, bv, bs = value_bound(activation, g)
    within(read(H), value * v, bv * np.abs(v) + 2 * U * np.abs(value * v) + 1e-37, "out")
    # the same products, the same bits: what is kept changes nothing
    assert np.array_equal(read(H), read(H2))
    dz = np.concatenate([d64 * v * slope, d64 * value], axis=1)
    bound = np.concatenate([np.abs(d64 * v) * bs, np.abs(d64) * bv], axis=1) + 4 * U * np.abs(dz)
    for name, got, want, size, slack in (("dx", DX, dz @ w64.T, np.abs(dz) @ np.abs(w64).T, bound @ np.abs(w64).T), ("dw", DW, x64.T @ dz, np.abs(x64).T @ np.abs(dz), np.abs(x64).T @ bound)):
        close_dot(read(got), want, size + slack / (8 * U), what=name)


SMALL = [(1, 1, 1), (1, 7, 3), (3, 1, 5), (5, 9, 2), (16, 33, 31), (17, 64, 32), (64, 100, 33), (33, 65, 64), (130, 129, 65), (7, 1000, 130)]
LARGE = [(1, 1024, 1024), (2, 1500, 1002), (9, 1024, 2048), (16, 2052, 514), (64, 784, 256), (100, 300, 1000), (300, 520, 500), (777, 500, 1003), (129, 1030, 1024), (1000, 784, 132), (2500, 256, 516),
         (512, 512, 2048), (1300, 768, 1536), (4000, 512, 1000), (1664, 2048, 2080), (3333, 130, 700), (5000, 4100, 96)]


@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("M,K,F", SMALL)
def test_small_layers(env, M, K, F, activation):
    check(env, M, K, F, activation)


@pytest.mark.parametrize("k", range(len(LARGE)))
def test_large_layers(env, k):
    check(env, *LARGE[k], ACTIVATIONS[k % 5])


@pytest.mark.parametrize("activation", ACTIVATIONS)
def test_every_activation_on_the_tensor_cores(env, activation):
    check(env, 1200, 300, 1100, activation)
    check(env, 300, 520, 499, activation)                    # few tiles, cut over clusters


@pytest.mark.parametrize("M,K,F", [(64, 784, 256), (777, 500, 1003), (1200, 300, 1100), (3, 900, 700), (400, 300, 602)])
@pytest.mark.parametrize("misaligned,path,arithmetic", [(1, 0, "3xfp16"), (0, 1, "3xfp16"), (0, 0, "3xtf32"), (1, 0, "3xtf32")])
def test_alignment_engines_and_arithmetics(env, M, K, F, misaligned, path, arithmetic):
    check(env, M, K, F, "silu", misaligned, path, arithmetic)


@pytest.mark.parametrize("M,K,F", [(64, 300, 150), (130, 129, 125), (128, 128, 130), (200, 70, 2000), (3000, 64, 33)])      # 4e6 multiply-adds are the least it takes
def test_forced_onto_the_tensor_cores(env, M, K, F):
    check(env, M, K, F, "gelu", path=2)


@pytest.mark.parametrize("M,K,F", [(4000, 16, 70), (16, 512, 600), (17, 40, 4000), (1000, 20, 130), (129, 17, 999)])
def test_short_reductions_on_the_tensor_cores(env, M, K, F):
    """Less than one step of the reduction in one product or another."""
    check(env, M, K, F, "silu", path=2)


@pytest.mark.parametrize("M,K,F", [(8000, 16, 16), (2500, 96, 80), (1501, 77, 53), (3001, 33, 9), (30, 500, 40), (32, 512, 2048), (40, 2100, 1024), (100, 1999, 500), (256, 256, 1000), (500, 512, 512),
                                   (8, 100, 8000), (600, 8, 1000), (16, 100, 2000), (65, 30, 1600)])
def test_between_the_paths(env, M, K, F):
    """Long batches whose weight gradient is cut, and sizes on both sides of where the tensor path begins to pay."""
    check(env, M, K, F, "tanh")


@pytest.mark.parametrize("misaligned", [0, 1])
@pytest.mark.parametrize("M,K,F", [(1, 622, 4027), (1, 624, 4028), (3, 1001, 777), (8, 515, 1025), (13, 1023, 701), (1, 66, 8191), (5, 130, 5003), (1, 64, 8192), (6, 120, 7698), (16, 900, 1002), (1, 25, 6935), (8, 13, 3001), (12, 8, 2999), (40, 27, 1801)])
def test_few_rows_against_weights_of_every_width(env, M, K, F, misaligned):
    check(env, M, K, F, "gelu", misaligned)


def test_rows_beyond_the_small_grid(env):
    check(env, 65535 * 32 + 70, 2, 3, "relu")


def test_projections_beyond_32_bits(env):
    """2^31 + projections.  The inputs are zero but for the last three rows, so those alone make the gradient of the weights."""
    K, F = 64, 8192
    M = (1 << 31) // (2 * F) + 130
    op, nd = env.gpu_op, env.nd
    shapes = [(M, K), (M, 2 * F), (M, F), (M, F), (M, K)]
    arrays = []
    for s in shapes:
        arrays.append(nd.empty(s, env.ctx))
        if isinstance(arrays[-1], int):
            pytest.skip("not enough device memory")
    X, Z, H, D, DX = arrays
    x, w, dout = inputs(3, K, F)
    W, DW = nd.array(w, env.ctx), nd.empty((K, 2 * F), env.ctx)
    op.array_set(X, 0.0, env.stream)
    op.array_set(D, 0.5, env.stream)
    op.device_synchronize()
    view(env, X, (M - 3) * K, (3, K))[:] = x
    view(env, D, (M - 3) * F, (3, F))[:] = dout
    assert op.gated_linear_forward(X, W, Z, H, "sigmoid", env.stream) == 0
    z = view(env, Z, (M - 3) * 2 * F, (3, 2 * F)).asnumpy()
    x64, w64 = x.astype(np.float64), w.astype(np.float64)
    close_dot(z, x64 @ w64, np.abs(x64) @ np.abs(w64), what="gates")
    z = z.astype(np.float64)
    value, slope, bv, bs = value_bound("sigmoid", z[:, :F])
    within(view(env, H, (M - 3) * F, (3, F)).asnumpy(), value * z[:, F:], bv * np.abs(z[:, F:]) + 2 * U * np.abs(value * z[:, F:]) + 1e-37, "out")
    assert not view(env, H, (M - 8) * F, (5, F)).asnumpy().any()
    assert op.gated_linear_backward(X, W, Z, D, DX, DW, "sigmoid", env.stream) == 0
    d64 = dout.astype(np.float64)
    dz = np.concatenate([d64 * z[:, F:] * slope, d64 * value], axis=1)
    bound = np.concatenate([np.abs(d64 * z[:, F:]) * bs, np.abs(d64) * bv], axis=1) + 4 * U * np.abs(dz)
    for name, got, want, size, slack in (("dx", view(env, DX, (M - 3) * K, (3, K)), dz @ w64.T, np.abs(dz) @ np.abs(w64).T, bound @ np.abs(w64).T),
                                         ("dw", DW, x64.T @ dz, np.abs(x64).T @ np.abs(dz), np.abs(x64).T @ bound)):
        close_dot(got.asnumpy(), want, size + slack / (8 * U), what=name)
    del X, Z, H, D, DX, arrays
    op.release_cached_memory()


def test_no_rows_against_large_weights(env):
    op, nd = env.gpu_op, env.nd
    W, DW = nd.array(np.ones((1024, 2048), np.float32), env.ctx), nd.array(np.ones((1024, 2048), np.float32), env.ctx)
    X, Z, H, DX = (nd.empty(s, env.ctx) for s in ((0, 1024), (0, 2048), (0, 1024), (0, 1024)))
    assert op.gated_linear_forward(X, W, Z, H, "silu", env.stream) == 0
    assert op.gated_linear_backward(X, W, Z, H, DX, DW, "silu", env.stream) == 0
    assert not DW.asnumpy().any()


def test_a_capture_without_a_call_before_it(env):
    """The first use of a stream is a capture: its scratch is made in it."""
    import ctypes
    import torch
    for M, K, F in ((40, 96, 64), (4, 1024, 2048), (600, 512, 520)):
        x, w, dout = inputs(M, K, F)
        X, W, D = (env.nd.array(v, env.ctx) for v in (x, w, dout))
        Z, H, DX, DW = (env.nd.empty(s, env.ctx) for s in ((M, 2 * F), (M, F), (M, K), (K, 2 * F)))
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        cell = ctypes.pointer(ctypes.c_void_p(side.cuda_stream))
        env.gpu_op.device_synchronize()
        with torch.cuda.graph(graph, stream=side):
            assert env.gpu_op.gated_linear_forward(X, W, Z, H, "silu", cell) == 0
            assert env.gpu_op.gated_linear_backward(X, W, Z, D, DX, DW, "silu", cell) == 0
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        got = [v.asnumpy() for v in (Z, H, DX, DW)]
        env.gpu_op.gated_linear_forward(X, W, Z, H, "silu", env.stream)
        env.gpu_op.gated_linear_backward(X, W, Z, D, DX, DW, "silu", env.stream)
        assert all(np.array_equal(g, v.asnumpy()) for g, v in zip(got, (Z, H, DX, DW)))


def test_no_rows_no_inputs_no_outputs(env):
    op, nd = env.gpu_op, env.nd
    for M, K, F in ((0, 5, 4), (3, 5, 0), (3, 0, 2000), (0, 7, 2001)):
        arrays = [nd.empty(s, env.ctx) for s in ((M, K), (K, 2 * F), (M, 2 * F), (M, F), (M, K), (K, 2 * F), (M, F))]
        X, W, Z, H, DX, DW, D = arrays
        for a in (X, W, DX, DW):
            if 0 not in a.shape:
                a[:] = np.ones(a.shape, np.float32)
        op.gated_linear_forward(X, W, Z, H, "silu", env.stream)
        op.gated_linear_backward(X, W, Z, D, DX, DW, "silu", env.stream)
        for a in (DX, DW):
            if 0 not in a.shape:
                assert not a.asnumpy().any()
    X, W, Z, H = nd.empty((3, 0), env.ctx), nd.empty((0, 8), env.ctx), nd.empty((3, 8), env.ctx), nd.empty((3, 4), env.ctx)
    op.gated_linear_forward(X, W, Z, H, "sigmoid", env.stream)
    assert not Z.asnumpy().any() and not H.asnumpy().any()


@pytest.mark.parametrize("M,K,F", [(5, 40, 24), (9, 1024, 2048), (777, 500, 1003), (1300, 768, 1536), (1, 622, 4027), (7, 130, 2999), (8, 1024, 1024), (16, 645, 831), (4000, 20, 30), (300, 520, 500), (40, 27, 1801)])
def test_one_gradient_alone_and_the_same_bits_every_time(env, M, K, F):
    x, w, dout = inputs(M, K, F)
    op = env.gpu_op
    X, W, D = (env.nd.array(v, env.ctx) for v in (x, w, dout))
    seen = []
    for names in (("dx", "dw"), ("dx",), ("dw",), ("dx", "dw")):
        Z, H = env.nd.empty((M, 2 * F), env.ctx), env.nd.empty((M, F), env.ctx)
        DX, DW = (env.nd.empty(s, env.ctx) if n in names else None for n, s in (("dx", (M, K)), ("dw", (K, 2 * F))))
        op.gated_linear_forward(X, W, Z, H, "tanh", env.stream)
        op.gated_linear_backward(X, W, Z, D, DX, DW, "tanh", env.stream)
        seen.append([a.asnumpy() if a is not None else None for a in (Z, H, DX, DW)])
    for again in seen[1:]:
        for a, b in zip(seen[0], again):
            assert b is None or np.array_equal(a, b)


def test_extreme_projections(env):
    """Where the activations saturate: values and slopes stay finite and of the right size."""
    g = np.array([0.0, 1e-30, -1e-30, 1e-4, -1e-4, 1.0, -1.0, 5.0, -5.0, 12.0, -12.0, 30.0, -30.0, 80.0, -80.0, 1e4, -1e4, 1e30, -1e30], np.float32)
    n = len(g)
    for activation in ACTIVATIONS:
        Z = env.nd.array(np.concatenate([g, np.full(n, 2.0, np.float32)])[None, :], env.ctx)
        D = env.nd.array(np.ones((1, n), np.float32), env.ctx)
        X, W = env.nd.array(np.ones((1, 1), np.float32), env.ctx), env.nd.array(np.ones((1, 2 * n), np.float32), env.ctx)
        DW = env.nd.empty((1, 2 * n), env.ctx)
        env.gpu_op.gated_linear_backward(X, W, Z, D, None, DW, activation, env.stream)
        got = DW.asnumpy()[0].astype(np.float64)             # x is one: dW = dz
        with np.errstate(over="ignore", under="ignore"):
            value, slope, bv, bs = value_bound(activation, g.astype(np.float64))
        tiny = np.abs(value) < 1e-36                            # below the smallest normal numbers
        assert np.all(np.isfinite(got)), activation
        assert np.all(np.abs(got[:n] - 2 * slope) <= np.minimum(2 * bs, 1e-4) + 1e-36 + 4 * U * np.abs(slope)), activation
        assert np.all((np.abs(got[n:] - value) <= bv + 4 * U * np.abs(value)) | tiny), activation


@pytest.mark.parametrize("activation", ["sigmoid", "silu", "tanh"])
def test_slopes_of_many_projections(env, activation):
    """2^17 gates: the reciprocal of every size of 1 + exp(-|g|) against 64 bits."""
    n = 1 << 17
    g = np.linspace(-30, 30, n).astype(np.float32)
    Z = env.nd.array(np.concatenate([g, np.full(n, 1.0, np.float32)])[None, :], env.ctx)
    D, X, W = (env.nd.array(np.ones(s, np.float32), env.ctx) for s in ((1, n), (1, 1), (1, 2 * n)))
    DW = env.nd.empty((1, 2 * n), env.ctx)
    env.gpu_op.gated_linear_backward(X, W, Z, D, None, DW, activation, env.stream)
    got = DW.asnumpy()[0].astype(np.float64)                 # x is one: dW = dz
    value, slope, bv, bs = value_bound(activation, g.astype(np.float64))
    within(got[:n], slope, bs + 4 * U * np.abs(slope), "slope")
    within(got[n:], value, bv + 4 * U * np.abs(value), "value")


def test_the_call_does_not_wait_where_products_are_held(env):
    M, K, F = 40, 96, 64
    x, w, dout = inputs(M, K, F)
    op = env.gpu_op
    X, W, D = (env.nd.array(v, env.ctx) for v in (x, w, dout))
    got = []
    for hold in (False, True):
        Z, H, DX, DW = (env.nd.empty(s, env.ctx) for s in ((M, 2 * F), (M, F), (M, K), (K, 2 * F)))
        op.hold_products(hold)
        op.gated_linear_forward(X, W, Z, H, "silu", env.stream)
        op.gated_linear_backward(X, W, Z, D, DX, DW, "silu", env.stream)
        got.append([a.asnumpy() for a in (Z, H, DX, DW)])
        if hold:
            op.hold_products(False)
            op.launch_held(env.stream)
    assert all(np.array_equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("M,K,F", [(40, 96, 64), (9, 1024, 2048), (700, 512, 520), (20, 1024, 4100), (3000, 32, 48), (3, 700, 1001), (200, 9001, 16)])
def test_a_captured_block_replayed_on_other_data(env, M, K, F):
    """Norm, gated layer and both backward calls in a graph that the caller captures: its replays have the bits of ordinary calls whatever the
    sizes of the numbers were at the capture, before it and in the replays in between."""
    import ctypes
    import torch
    nd, op = env.nd, env.gpu_op
    rng = np.random.RandomState(M)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    cell = ctypes.pointer(ctypes.c_void_p(side.cuda_stream))
    shapes = {"h": (M, K), "r": (M, K), "g": (K,), "b": (K,), "s": (M, K), "y": (M, K), "w": (K, 2 * F), "z": (M, 2 * F), "o": (M, F), "do": (M, F), "dy": (M, K), "dw": (K, 2 * F),
              "dh": (M, K), "dr": (M, K), "dg": (K,), "db": (K,)}
    a = {n: nd.array(rng.randn(*s).astype(np.float32), env.ctx) for n, s in shapes.items()}
    state = op.dropout_state(0.3, 4)

    def work(stream):
        op.dropout_add_layer_norm_forward(a["h"], a["r"], a["g"], a["b"], a["s"], a["y"], state, 1e-5, stream)
        op.gated_linear_forward(a["y"], a["w"], a["z"], a["o"], "silu", stream)
        op.gated_linear_backward(a["y"], a["w"], a["z"], a["do"], a["dy"], a["dw"], "silu", stream)
        op.dropout_add_layer_norm_backward(a["s"], a["g"], a["dy"], None, a["dh"], a["dr"], a["dg"], a["db"], state, 1e-5, stream)

    def fill(size):
        for n in ("h", "r", "g", "w", "do"):
            a[n][:] = (size * rng.randn(*shapes[n])).astype(np.float32)

    results = ("s", "y", "z", "o", "dy", "dw", "dh", "dr", "dg", "db")
    fill(30.0)
    work(cell)                                               # ordinary calls that leave their maxima
    op.device_synchronize()
    with torch.cuda.graph(graph, stream=side):
        work(cell)
    for size in (1.0, 1e4, 1e-3, 0.5):
        fill(size)
        for n in results:
            a[n][:] = np.full(shapes[n], np.nan, np.float32)
        graph.replay()
        torch.cuda.synchronize()
        got = {n: a[n].asnumpy() for n in results}
        work(env.stream)
        op.device_synchronize()
        for n in results:
            assert np.isfinite(got[n]).all(), (size, n)
            np.testing.assert_array_equal(got[n], a[n].asnumpy(), err_msg="%s at %g" % (n, size))


@pytest.mark.parametrize("M,K,F", [(40, 96, 64), (9, 1024, 2048), (700, 512, 520)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_row_that_is_not_finite_stays_by_itself(env, M, K, F, bad):
    """The other rows keep their precision: the scale of the tensor path is taken from finite values."""
    x, w, dout = inputs(M, K, F)
    x *= np.float32(1e-3)
    row = M // 2
    x[row, K // 3] = bad
    X, W, D = (env.nd.array(v, env.ctx) for v in (x, w, dout))
    Z, H, DX, DW = (env.nd.empty(s, env.ctx) for s in ((M, 2 * F), (M, F), (M, K), (K, 2 * F)))
    env.gpu_op.gated_linear_forward(X, W, Z, H, "silu", env.stream)
    env.gpu_op.gated_linear_backward(X, W, Z, D, DX, DW, "silu", env.stream)
    z, rest = Z.asnumpy(), np.arange(M) != row
    assert not np.isfinite(z[row]).any() and not np.isfinite(H.asnumpy()[row]).all()
    x64, w64 = x[rest].astype(np.float64), w.astype(np.float64)
    close_dot(z[rest], x64 @ w64, np.abs(x64) @ np.abs(w64), what="gates")
    assert np.isfinite(H.asnumpy()[rest]).all() and np.isfinite(DX.asnumpy()[rest]).all()


def test_two_streams_at_once(env):
    """Calls on two streams from two threads: scratch, states and counters are each stream's own."""
    import threading
    nd, op, runs = env.nd, env.gpu_op, 12
    cells = [env.stream, op.create_cudaStream()]
    want, got, errors = [], [], []

    def work(k, seen, stream):
        x, w, dout = inputs((700, 333)[k], 512, 520, seed=k)
        X, W, D = (nd.array(v, env.ctx) for v in (x, w, dout))
        G, B = (nd.array(np.ones(512, np.float32), env.ctx) for _ in range(2))
        Z, H, DX, DW, Y, DN, DG, DB = (nd.empty(s, env.ctx) for s in ((len(x), 1040), (len(x), 520), x.shape, w.shape, x.shape, x.shape, (512,), (512,)))
        op.device_synchronize()
        for _ in range(runs):
            op.layer_norm_forward(X, G, B, Y, 1e-5, stream)
            op.gated_linear_forward(Y, W, Z, H, "gelu", stream)
            op.gated_linear_backward(Y, W, Z, D, DX, DW, "gelu", stream)
            op.layer_norm_backward(X, G, DX, DN, DG, DB, 1e-5, stream)
        op.device_synchronize()
        seen.append((k, [v.asnumpy() for v in (Z, H, DX, DW, DN, DG, DB)]))

    def guarded(k, seen, stream):
        try:
            work(k, seen, stream)
        except Exception as e:       # noqa: BLE001
            errors.append(e)

    for k in range(2):
        work(k, want, cells[k])
    threads = [threading.Thread(target=guarded, args=(k, got, cells[k])) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for k, arrays in got:
        assert all(np.array_equal(a, b) for a, b in zip(arrays, dict(want)[k]))


# ---- graphs ---------------------------------------------------------------------------------------------------------
def block_step(monkeypatch, recorded=False, steps=1, plan=None, optimizer="sgd", **kind):
    import queue
    import random
    from tests.block_graph import Block
    from tinyflow_b200 import autodiff as ad, gpu_op, ndarray, step_graph
    monkeypatch.setattr(step_graph, "ENABLED", recorded)
    random.seed(5)
    block = Block(**kind)
    control = queue.Queue()
    ex = ad.Executor(block.loss, block.y, 0.01, control, None, None, optimizer=optimizer)
    ctx = ndarray.gpu(0)
    feed = {n: ndarray.array(v, ctx) for n, v in block.values.items()}
    for var in block.parameters:
        for moment in ex.Variable_node_to_mv.get(var, ()):
            feed[moment] = ndarray.array(np.zeros_like(block.values[var]), ctx)
    if plan:
        ex.infer_shape({n: v.shape for n, v in feed.items()})
        control.put(plan(ex))
    losses = [ex.run(feed)[0] for _ in range(steps)]
    gpu_op.device_synchronize()
    replayed = any(f.recording or any(b.recording for b in f.batches.values()) for f in ex._recordings.sets.values())
    return block, ex, [v.asnumpy() for v in losses], {n.name: feed[n].asnumpy() for n in block.parameters}, replayed


@pytest.mark.parametrize("kind", [{}, dict(batch=300, width=260, hidden=516, dropout=0.5, activations=("relu", "silu", "sigmoid"))])
def test_every_node_of_a_step_against_the_oracle(env, monkeypatch, kind):
    from oracle.graph_eval import OracleExecutor
    block, ex, losses, _, _ = block_step(monkeypatch, **kind)
    orc = OracleExecutor(ex.topo_order, np.float64)
    value = lambda n: block.values[n].astype(np.float64) if n in block.values and n.isw == 2 else ex.value_of(n).asnumpy().astype(np.float64)     # noqa: E731
    # parameters were updated behind their last reader: evaluated at their first values
    first = {n: v.astype(np.float64) for n, v in block.values.items()}
    checked = 0
    for node in ex.topo_order:
        if not node.inputs or node.issgd:
            continue
        ins = [first[i] if i in first else value(i) for i in node.inputs]
        want = np.asarray(orc._eval(node, ins), np.float64)
        got = value(node).reshape(want.shape)
        name = type(node.op).__name__
        if name == "GatedLinearBackwardOp":
            wants = [want] + [np.asarray(p, np.float64) for p in orc.parts[node]]
        if name in ("MatMulOp", "GatedLinearBackwardOp", "GatedLinearForwardOp") or (name == "PartOp" and "Gated" in type(node.inputs[0].op).__name__):
            tolerance = 2e-5 * np.linalg.norm(want) / np.sqrt(want.size) + 1e-4 * np.abs(want)
        else:
            tolerance = 1e-4 * np.maximum(np.abs(want), 1e-2 * max([np.abs(want).max()] + [np.abs(i).max() for i in ins]))
        assert np.all(np.abs(got - want) <= tolerance), (node.index, node.name)
        checked += 1
    assert checked > 30


@pytest.mark.parametrize("optimizer", ["sgd", "adam"])
def test_a_replayed_step_has_the_bits_of_the_ordinary_one(env, monkeypatch, optimizer):
    runs = [block_step(monkeypatch, recorded, 9, optimizer=optimizer, dropout=0.3) for recorded in (False, True)]
    assert runs[1][4] and not runs[0][4]
    assert all(np.array_equal(a, b) for a, b in zip(runs[0][2], runs[1][2]))
    assert all(np.array_equal(v, runs[1][3][n]) for n, v in runs[0][3].items())


def test_a_replayed_step_of_a_long_batch(env, monkeypatch):
    """Clusters of 16 in a recorded step.  The summed loss of so many rows makes the last steps overshoot to NaN, which both runs have to do alike."""
    kind = dict(batch=2500, width=32, hidden=40, dropout=0.3)
    runs = [block_step(monkeypatch, recorded, 9, **kind) for recorded in (False, True)]
    assert runs[1][4] and not runs[0][4]
    assert all(np.isfinite(v).all() for v in runs[0][2][:6])
    assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(runs[0][2], runs[1][2]))
    assert all(np.array_equal(v, runs[1][3][n], equal_nan=True) for n, v in runs[0][3].items())


def _plan_swap(ex):
    from tinyflow_b200 import memory_plan
    return memory_plan.vdnn_plan(ex, policy="all", prefetch=4, min_bytes=1)


def _plan_recompute(ex):
    """Every result of a forward operator that has several is released behind its last forward reader and computed again in front of
    the first one of the backward pass, where its own inputs are still there."""
    users = {n: [] for n in ex.topo_order}
    for n in ex.topo_order:
        for i in n.inputs:
            users[i].append(n.index)
    release, recompute = [], []
    for n in ex.topo_order:
        whole = n.inputs[0] if type(n.op).__name__ in ("PartOp", "NormalisedSumOp") else n
        if not type(whole.op).__name__.endswith("ForwardOp") or not hasattr(whole.op, "parts") or n.index >= ex.targetloss.index:
            continue
        if type(n.op).__name__ != "NormalisedSumOp":
            continue
        forward, backward = [u for u in users[n] if u <= ex.targetloss.index], [u for u in users[n] if u > ex.targetloss.index]
        if forward and backward:
            release.append((max(forward), n.index))
            recompute.append((min(backward), n.index))
    assert recompute
    return [], release, recompute


@pytest.mark.parametrize("plan", [_plan_swap, _plan_recompute])
def test_a_memory_plan_changes_no_bits(env, monkeypatch, plan):
    want = block_step(monkeypatch, steps=3, dropout=0.4)
    got = block_step(monkeypatch, steps=3, dropout=0.4, plan=plan)
    assert all(np.array_equal(a, b) for a, b in zip(want[2], got[2]))
    assert all(np.array_equal(v, got[3][n]) for n, v in want[3].items())


def test_training_with_other_batches_in_turn(env, monkeypatch):
    """Feeds of two sizes one after the other: shapes, descriptors and arrays of each are its own."""
    import random
    from tests.block_graph import Block
    from tinyflow_b200 import autodiff as ad, ndarray
    block = Block(batch=40, dropout=0.0)
    ctx = ndarray.gpu(0)

    def run(ex, rows):
        feed = {n: ndarray.array(v[:rows] if n.isw == 2 else v, ctx) for n, v in block.values.items()}
        random.seed(1)
        loss, _ = ex.run(feed)
        return loss.asnumpy(), [feed[p].asnumpy() for p in block.parameters]

    one = ad.Executor(block.loss, block.y, 0.01, optimizer="sgd")
    both = [run(one, rows) for rows in (40, 11, 40, 11)]
    for rows, got in zip((40, 11, 40, 11), both):
        want = run(ad.Executor(block.loss, block.y, 0.01, optimizer="sgd"), rows)
        assert np.array_equal(got[0], want[0]) and all(np.array_equal(a, b) for a, b in zip(got[1], want[1]))
