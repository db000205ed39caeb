"""The largest magnitudes that operators leave behind for the products that read their results: what they are taken of, and how long they hold.

A product scales its operands by a power of two that comes from that maximum; a maximum that is too small lets finite numbers overflow
the 16-bit halves (above 2^15 / scale), one that is far too large costs the small ones their digits.  So results are compared bit by bit with
those of a run whose maximum is known to be right."""
import ctypes

import numpy as np
import pytest

from tests.test_gpu_norm import view
from tests.test_gpu_ops import env  # noqa: F401

pytestmark = pytest.mark.gpu
M, K, F = 700, 512, 520                 # the tensor path, forward and backward
ROW = 333


def flat(env, array):
    """The same memory as a matrix of M rows."""
    return view(env, array, 0, (M, K))


def by_relu(env, x):
    y = env.empty(x.shape)
    env.gpu_op.relu(env.dev(x), y)
    return y


def by_activation(env, x):
    y = env.empty(x.shape)
    env.gpu_op.activation_forward(env.dev(x), y, "relu", env.gpu_op.activation_get_cudnnlist(x.shape, "NCHW", "relu"), env.cudnn, env.stream)
    return y


def by_dropout(env, x):
    y = env.empty(x.shape)
    env.gpu_op.dropout_forward(env.dev(x), y, "NCHW", 0.3, 5, env.gpu_op.get_input_descriptor(x.shape, "NCHW"), env.cudnn, env.stream)
    return y


def by_sum_and_relu(env, x):
    total, y = env.empty(x.shape), env.empty(x.shape)
    half = env.dev(x * np.float32(0.5))
    env.gpu_op.matrix_elementwise_add(half, half, total, env.stream)
    env.gpu_op.activation_forward(total, y, "relu", env.gpu_op.activation_get_cudnnlist(x.shape, "NCHW", "relu"), env.cudnn, env.stream)
    return y


def by_relu_gradient(env, x):
    y = env.empty(x.shape)
    env.gpu_op.relu_gradient(env.dev(np.where(np.arange(K) % 3, 1, -1) * np.ones_like(x)), env.dev(x), y)
    return y


def by_concatenation(env, x):
    y = env.empty((M, K, 1, 1))
    env.gpu_op.concat_forward(env.dev(x[:, :200, None, None]), env.dev(x[:, 200:, None, None]), y, env.stream)
    return flat(env, y)


def by_split(env, x):
    y = env.empty((M, K, 1, 1))
    whole = np.concatenate([x, x[:, :8]], axis=1)[:, :, None, None]
    env.gpu_op.concat_a_backward(env.dev(x[:, :, None, None]), env.dev(whole[:, K:]), env.dev(whole), y, env.stream)
    return flat(env, y)


def by_mean(env, x):
    shape = (M, 8, 8, 8)
    out, cell = env.gpu_op.pooling_2d_forward_get_out_shape(shape, "NCHW", "mean", 1, 1, 1, 1, 3, 3)
    assert tuple(out) == shape
    y = env.empty(shape)
    env.gpu_op.pooling_2d_forward(env.dev(x.reshape(shape)), y, cell, env.cudnn, env.stream)
    return flat(env, y)


def by_convolution(env, x):
    shape = (M, 32, 4, 4)
    out, cell = env.gpu_op.convolution_2d_forward_get_out_shape(shape, (32, 32, 1, 1), "NCHW", "VALID", 1, 1)
    assert tuple(out) == shape
    y = env.empty(shape)
    env.gpu_op.convolution_2d_forward(env.dev(x.reshape(shape)), env.dev(np.random.RandomState(7).randn(32, 32, 1, 1)), y, cell, env.cudnn, env.stream)
    return flat(env, y)


def by_upload(env, x):
    return env.dev(x)


PRODUCERS = [by_relu, by_activation, by_dropout, by_sum_and_relu, by_relu_gradient, by_concatenation, by_split, by_mean, by_convolution, by_upload]


def layer(env, X, w, dout, forms=("gated", "product")):
    """Results of a gated layer, of its gradient and of a plain product, all of them rows of X."""
    W, D = env.dev(w), env.dev(dout)
    Z, H, DX, DW, C = (env.empty(s) for s in ((M, 2 * F), (M, F), (M, K), (K, 2 * F), (M, 2 * F)))
    env.gpu_op.gated_linear_forward(X, W, Z, H, "silu", env.stream)
    env.gpu_op.gated_linear_backward(X, W, Z, D, DX, DW, "silu", env.stream)
    env.gpu_op.matrix_multiply(X, False, W, False, C, env.cublas, env.stream)
    env.gpu_op.device_synchronize()
    return {"gates": Z.asnumpy(), "out": H.asnumpy(), "dx": DX.asnumpy(), "product": C.asnumpy()}, DW.asnumpy()


def operands(size):
    rng = np.random.RandomState(11)
    x = (size * rng.randn(M, K)).astype(np.float32)
    return x, (rng.randn(K, 2 * F) * K ** -0.5).astype(np.float32), (0.1 * rng.randn(M, F)).astype(np.float32)


@pytest.mark.parametrize("producer", PRODUCERS)
@pytest.mark.parametrize("size", [1e5, 1e-5])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_a_row_that_is_not_finite_leaves_the_others_their_bits(env, producer, size, bad):
    """Whichever operator wrote the rows.  The clean run has numbers in the row that are not the largest."""
    x, w, dout = operands(size)
    x[ROW] *= np.float32(0.1)
    clean, _ = layer(env, producer(env, x), w, dout)
    x[ROW] = bad
    got, _ = layer(env, producer(env, x), w, dout)
    rest = np.arange(M) != ROW
    for name, v in got.items():
        assert np.isfinite(v[rest]).all() and not np.isfinite(v[ROW]).any(), name
        np.testing.assert_array_equal(v[rest], clean[name][rest], err_msg=name)


@pytest.mark.parametrize("rule", ["sgd", "sgd many", "adam"])
def test_a_weight_that_is_not_finite_leaves_the_other_columns_their_bits(env, rule):
    x, w, dout = operands(1e5)
    w *= np.float32(1e5)
    column = 77
    w[9, column] = 1
    runs = []
    for bad in (False, True):
        g = np.zeros_like(w)
        if bad:
            g[9, column] = np.inf
        W, G = env.dev(w), env.dev(g)
        if rule == "sgd":
            env.gpu_op.sgd_update(W, G, 1.0, env.stream)
        elif rule == "sgd many":
            env.gpu_op.sgd_update_many(*(env.gpu_op.handle_array([v]) for v in (W, G)), 1.0, env.stream)
        else:
            m, v = env.dev(g), env.dev(np.ones_like(w))
            env.gpu_op.adam_compute(W, m, v, 0.9, 0.999, 1e-8, 1.0, env.stream)
        X, Z, H = env.dev(x), env.empty((M, 2 * F)), env.empty((M, F))
        env.gpu_op.gated_linear_forward(X, W, Z, H, "relu", env.stream)
        runs.append((Z.asnumpy(), H.asnumpy()))
    for clean, got in zip(*runs):
        rest = np.arange(clean.shape[1]) != column
        assert np.isfinite(clean).all() and not np.isfinite(got[:, column]).all()
        np.testing.assert_array_equal(got[:, rest], clean[:, rest])


# ---- arrays that a graph of the caller's own writes -------------------------------------------------------------------
def into(env, kind, x, y, stream):
    """The call that writes y (M x K) from x of that size."""
    op, ones = env.gpu_op, env.ones
    as4 = lambda a, *s: view(env, a, 0, s)                 # noqa: E731
    if kind == "relu":
        cell = op.activation_get_cudnnlist((M, K), "NCHW", "relu")
        return lambda: op.activation_forward(x, y, "relu", cell, env.cudnn, stream)
    if kind == "dropout":
        inputd = op.get_input_descriptor((M, K), "NCHW")
        return lambda: op.dropout_forward(x, y, "NCHW", 0.3, 5, inputd, env.cudnn, stream)
    if kind == "concat":
        a, b, whole = as4(x, M, K // 2, 1, 1), as4(x, M, K // 2, 1, 1), as4(y, M, K, 1, 1)
        return lambda: op.concat_forward(a, b, whole, stream)
    if kind == "mean":
        _, cell = op.pooling_2d_forward_get_out_shape((M, 8, 8, 8), "NCHW", "mean", 1, 1, 1, 1, 3, 3)
        return lambda: op.pooling_2d_forward(as4(x, M, 8, 8, 8), as4(y, M, 8, 8, 8), cell, env.cudnn, stream)
    if kind == "norm":                                     # gamma is what sizes its result
        gamma = view(env, x, 0, (K,))
        return lambda: op.layer_norm_forward(env.noise, gamma, gamma, y, 1e-5, stream)
    if kind == "residual norm":
        gamma, total, state = view(env, x, 0, (K,)), env.empty((M, K)), op.dropout_state(0.2, 3)
        return lambda: op.dropout_add_layer_norm_forward(env.noise, env.noise, gamma, gamma, total, y, state, 1e-5, stream)
    if kind == "norm gradient":
        return lambda: op.layer_norm_backward(env.noise, ones, x, y, None, None, 1e-5, stream)
    if kind == "gated small":                              # one launch of the CUDA-core kernel
        a, w = view(env, x, 0, (M, 8)), env.weight8
        return lambda: op.gated_linear_forward(a, w, None, y, "relu", stream)
    if kind == "gated":
        return lambda: op.gated_linear_forward(x, env.weight, None, y, "relu", stream)
    if kind == "copy":
        return lambda: op.copy_on_stream(x, y, stream)
    assert kind == "sum of squares"
    return lambda: op.matrix_elementwise_multiply(x, ones2(env, x), y, stream)


def ones2(env, like):
    if not hasattr(env, "ones_"):
        env.ones_ = env.dev(np.ones((M, K)))
    return env.ones_


@pytest.fixture(scope="module")
def stage(env):
    rng = np.random.RandomState(2)
    env.ones = env.dev(np.ones(K))
    env.noise = env.dev(rng.randn(M, K))
    env.weight8, env.weight = env.dev(rng.randn(8, 2 * K)), env.dev(rng.randn(K, 2 * K) * K ** -0.5)
    ones2(env, None)
    return env


KINDS = ["relu", "dropout", "concat", "mean", "norm", "residual norm", "norm gradient", "gated small", "gated", "copy", "sum of squares"]


def capture(call_on):
    """A graph of call_on(stream cell)() on a stream of its own."""
    import torch
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    cell = ctypes.pointer(ctypes.c_void_p(side.cuda_stream))
    call = call_on(cell)
    with torch.cuda.graph(graph, stream=side):
        call()
    graph.side = side
    return graph


def replay(graph):
    import torch
    graph.replay()
    torch.cuda.synchronize()


def same_as_a_copy(env, y, what):
    """What reads y has the bits that it has on an uploaded copy of y."""
    results = []
    rng = np.random.RandomState(8)
    w, dout = (rng.randn(K, 2 * F) * K ** -0.5).astype(np.float32), (0.1 * rng.randn(M, F)).astype(np.float32)
    for X in (y, env.dev(y.asnumpy())):
        got, dw = layer(env, X, w, dout)
        results.append(dict(got, dweight=dw))
    for name, v in results[0].items():
        assert np.isfinite(v).all(), (what, name)
        np.testing.assert_array_equal(v, results[1][name], err_msg="%s, %s" % (what, name))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("sizes", [(1.0, 1e4), (1e4, 1.0), (1e-3, 1e3)])
def test_a_replay_that_rewrites_an_array(stage, kind, sizes):
    """Ordinary call, then a replay of the same call on numbers of another size, and the same the other way round: what reads the array
    afterwards scales by what is there."""
    env = stage
    rng = np.random.RandomState(4)
    x, y = env.empty((M, K)), env.empty((M, K))
    numbers = rng.randn(M, K).astype(np.float32)

    def fill(size):
        x[:] = numbers * np.float32(size)

    fill(sizes[0])
    ordinary = into(env, kind, x, y, env.stream)
    for _ in range(2):
        ordinary()
    env.gpu_op.device_synchronize()
    graph = capture(lambda cell: into(env, kind, x, y, cell))
    for turn in range(3):
        fill(sizes[0])
        ordinary()                                         # leaves what it knows of y
        if turn:
            same_as_a_copy(env, y, "ordinary, turn %d" % turn)
        fill(sizes[1])
        replay(graph)
        same_as_a_copy(env, y, "replayed, turn %d" % turn)
        fill(sizes[0])
        replay(graph)
        same_as_a_copy(env, y, "replayed again, turn %d" % turn)


def test_an_array_in_the_place_of_one_that_a_replay_wrote(stage):
    """Freed memory has nothing of its past: what is written there by ordinary calls hands its maximum on again (a launch less)."""
    env = stage
    w, h = by_relu(env, np.ones((K, 2 * F), np.float32)), env.empty((M, F))
    x = env.dev(np.random.RandomState(5).randn(M, K))

    def launches(y):
        into(env, "relu", x, y, env.stream)()
        before = env.gpu_op.launch_count()
        env.gpu_op.gated_linear_forward(y, w, None, h, "relu", env.stream)
        return env.gpu_op.launch_count() - before

    y = env.empty((M, K))
    clean = launches(y)
    graph = capture(lambda cell: into(env, "relu", x, y, cell))
    assert launches(y) == clean + 1
    at = y.data_ptr
    del graph
    y.free_gpu()
    taken = []
    while not taken or taken[-1].data_ptr != at:
        taken.append(env.empty((M, K)))
        assert len(taken) < 100
    assert launches(taken[-1]) == clean


@pytest.mark.parametrize("last", ["sum", "relu gradient"])
def test_a_capture_that_ends_with_a_call_that_would_wait(stage, last):
    """Large sums and gradients of a ReLU wait for one call outside a capture; inside, their kernel is part of the graph."""
    env = stage
    rng = np.random.RandomState(6)
    a, b, out = env.dev(rng.randn(M, K)), env.dev(rng.randn(M, K)), env.dev(np.zeros((M, K)))
    cell_of = env.gpu_op.activation_get_cudnnlist((M, K), "NCHW", "relu")

    def call_on(stream):
        if last == "sum":
            return lambda: env.gpu_op.matrix_elementwise_add(a, b, out, stream)
        return lambda: env.gpu_op.activation_backward(a, out, a, b, "relu", cell_of, env.cudnn, stream)

    env.gpu_op.device_synchronize()
    graph = capture(call_on)
    for size in (1.0, 3.0):
        a[:] = (size * rng.randn(M, K)).astype(np.float32)
        out[:] = np.full((M, K), np.nan, np.float32)
        replay(graph)
        x, y = a.asnumpy(), b.asnumpy()
        np.testing.assert_array_equal(out.asnumpy(), x + y if last == "sum" else np.where(x > 0, y, 0))


# N, C, H, W, filters, window, stride: 1x1 and windows, strided phases, patches of few channels, the CUDA cores' own kernels
CONVOLUTIONS = [(8, 64, 14, 14, 96, 1, 1), (4, 32, 20, 20, 64, 3, 1), (4, 32, 21, 21, 64, 3, 2), (4, 3, 32, 32, 64, 7, 2), (4, 3, 30, 30, 16, 3, 1)]


@pytest.mark.parametrize("geometry", CONVOLUTIONS)
@pytest.mark.parametrize("before", [False, True])
def test_captured_convolutions(stage, geometry, before):
    """All three calls of a layer in a graph: replays on numbers of any size have the bits of ordinary calls on a descriptor of their own,
    and so have ordinary calls on the graph's descriptor in between.  before: those come ahead of the capture, too."""
    env = stage
    op = env.gpu_op
    N, C, H, W, filters, window, stride = geometry
    rng = np.random.RandomState(C + window)
    shapes = (N, C, H, W), (filters, C, window, window)
    padding = "SAME" if stride == 1 else "VALID"
    out, cell = op.convolution_2d_forward_get_out_shape(*shapes, "NCHW", padding, stride, stride)
    other = op.convolution_2d_forward_get_out_shape(*shapes, "NCHW", padding, stride, stride)[1]
    x, w, dy = (env.empty(s) for s in shapes + (tuple(out),))
    numbers = [rng.randn(*v.shape).astype(np.float32) for v in (x, w, dy)]
    results = {k: [env.empty(s) for s in (tuple(out),) + shapes] for k in ("graph", "same", "other")}

    def fill(size):
        for v, n in zip((x, w, dy), numbers):
            v[:] = n * np.float32(size)

    def calls(descriptor, into, stream):
        def run():
            assert op.convolution_2d_forward(x, w, into[0], descriptor, env.cudnn, stream) == 0
            assert op.convolution_backward_data(x, dy, w, into[1], descriptor, env.cudnn, stream) == 0
            assert op.convolution_backward_filter(x, dy, w, into[2], descriptor, env.cudnn, stream) == 0
        return run

    fill(30.0)
    if before:
        calls(cell, results["same"], env.stream)()
    op.device_synchronize()
    graph = capture(lambda stream: calls(cell, results["graph"], stream))
    for size in (1.0, 1e4, 1e-3, 0.5):
        fill(size)
        calls(other, results["other"], env.stream)()
        replay(graph)
        calls(cell, results["same"], env.stream)()
        replay(graph)
        op.device_synchronize()
        for k in ("graph", "same"):
            for name, got, want in zip(("y", "dx", "dw"), results[k], results["other"]):
                np.testing.assert_array_equal(got.asnumpy(), want.asnumpy(), err_msg="%s of %s at %g" % (name, k, size))


def test_a_replay_between_a_convolutions_calls(stage):
    """The descriptor's packs are what the replay left: the gradient behind it takes them anew from its own arrays."""
    env = stage
    op, rng = env.gpu_op, np.random.RandomState(9)
    shapes = (4, 32, 20, 20), (64, 32, 3, 3)
    out, cell = op.convolution_2d_forward_get_out_shape(*shapes, "NCHW", "SAME", 1, 1)
    other = op.convolution_2d_forward_get_out_shape(*shapes, "NCHW", "SAME", 1, 1)[1]
    x, x2, w, w2, dy = (env.dev(rng.randn(*s)) for s in (shapes[0], shapes[0], shapes[1], shapes[1], out))
    y, y2, got, want = env.empty(out), env.empty(out), [env.empty(s) for s in shapes], [env.empty(s) for s in shapes]
    op.device_synchronize()
    graph = capture(lambda stream: lambda: op.convolution_2d_forward(x2, w2, y2, cell, env.cudnn, stream))
    for descriptor, into in ((cell, got), (other, want)):
        op.convolution_2d_forward(x, w, y, descriptor, env.cudnn, env.stream)
        op.device_synchronize()
        replay(graph)
        op.convolution_backward_data(x, dy, w, into[0], descriptor, env.cudnn, env.stream)
        op.convolution_backward_filter(x, dy, w, into[1], descriptor, env.cudnn, env.stream)
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a.asnumpy(), b.asnumpy())


def test_a_replay_between_the_calls_of_a_pooling(stage):
    env = stage
    op, rng = env.gpu_op, np.random.RandomState(10)
    shape = (5, 7, 18, 18)
    out, cell = op.pooling_2d_forward_get_out_shape(shape, "NCHW", "max", 0, 0, 2, 2, 2, 2)
    other = op.pooling_2d_forward_get_out_shape(shape, "NCHW", "max", 0, 0, 2, 2, 2, 2)[1]
    x, x2, dy = (env.dev(rng.randn(*s)) for s in (shape, shape, out))
    y, y2, got, want = env.empty(out), env.empty(out), env.empty(shape), env.empty(shape)
    op.device_synchronize()
    graph = capture(lambda stream: lambda: op.pooling_2d_forward(x2, y2, cell, env.cudnn, stream))
    for descriptor, into in ((cell, got), (other, want)):
        op.pooling_2d_forward(x, y, descriptor, env.cudnn, env.stream)
        op.device_synchronize()
        replay(graph)
        op.pooling_2d_backward(x, y, dy, into, descriptor, env.cudnn, env.stream)
    np.testing.assert_array_equal(got.asnumpy(), want.asnumpy())


# ---- calls that are short of memory -------------------------------------------------------------------------------------
class FullDevice:
    """No scratch on any stream and no byte left in the pool."""
    def __init__(self, env):
        self.env = env

    def __enter__(self):
        op = self.env.gpu_op
        op.device_synchronize()
        op.set_memory_limit(1)
        assert isinstance(self.env.empty((1 << 30,)), int)                 # the scratch of every stream goes back
        op.release_cached_memory()
        op.set_memory_limit(sum(op.allocator_stats()))

    def __exit__(self, *error):
        self.env.gpu_op.set_memory_limit(0)


def product_bits(env, y, w):
    out = env.empty((y.shape[0], w.shape[1]))
    env.gpu_op.matrix_multiply(y, False, w, False, out, env.cublas, env.stream)
    return out.asnumpy()


@pytest.mark.parametrize("D", [512, 9000, 16400])
@pytest.mark.parametrize("form", ["norm", "residual norm"])
def test_norm_gradients_short_of_memory(stage, D, form):
    """They leave no maximum behind: the next write of the array begins with a clear word."""
    env = stage
    op, rows = env.gpu_op, 300
    rng = np.random.RandomState(D)
    x, y, big, small = (env.dev(size * rng.randn(rows, D)) for size in (1.0, 1.0, 1e4, 1e-4))
    gamma, dg, db, w = env.dev(np.ones(D)), env.empty((D,)), env.empty((D,)), env.dev(rng.randn(D, 1024))
    other, state = op.create_cudaStream(), op.dropout_state(0.5, 1)
    with FullDevice(env):
        op.relu(big, y)
        if form == "norm":
            assert op.layer_norm_backward(x, gamma, big, y, dg, db, 1e-5, other) > 0
        else:
            assert op.dropout_add_layer_norm_backward(x, gamma, big, None, y, None, dg, db, state, 1e-5, other) > 0
    op.relu(small, y)
    np.testing.assert_array_equal(product_bits(env, y, w), product_bits(env, env.dev(y.asnumpy()), w))
    op.destroy_cudaStream(other)


def test_a_convolution_short_of_memory(stage):
    env = stage
    op, rng = env.gpu_op, np.random.RandomState(3)
    shapes = (16, 256, 28, 28), (256, 256, 3, 3)
    out, cell = op.convolution_2d_forward_get_out_shape(*shapes, "NCHW", "SAME", 1, 1)
    next_cell = op.convolution_2d_forward_get_out_shape(out, (64, 256, 1, 1), "NCHW", "VALID", 1, 1)[1]
    act = op.activation_get_cudnnlist(out, "NCHW", "relu")
    x, w, w2, big, small = (env.dev(size * rng.randn(*s)) for size, s in ((1, shapes[0]), (1, shapes[1]), (1, (64, 256, 1, 1)), (1e6, out), (1e-6, out)))
    y, r, z = env.empty(out), env.empty(out), env.empty((16, 64, 28, 28))
    other = op.create_cudaStream()
    for _ in range(2):                                     # the ReLU in front of the second layer asks for the maximum of the first one's output
        assert op.convolution_2d_forward(x, w, y, cell, env.cudnn, env.stream) == 0
        op.activation_forward(y, r, "relu", act, env.cudnn, env.stream)
        assert op.convolution_2d_forward(r, w2, z, next_cell, env.cudnn, env.stream) == 0
    with FullDevice(env):
        op.relu(big, y)
        assert op.convolution_2d_forward(x, w, y, cell, env.cudnn, other) > 0
    op.relu(small, y)
    rows = view(env, y, 0, (256 * 16, 28 * 28))
    w3 = env.dev(rng.randn(28 * 28, 64))
    np.testing.assert_array_equal(product_bits(env, rows, w3), product_bits(env, env.dev(rows.asnumpy()), w3))
    op.destroy_cudaStream(other)


def test_a_write_that_the_library_does_not_see(stage):
    """By another library over the same memory, and through an array that begins elsewhere in it: announced, it is taken as it is."""
    import torch
    env = stage
    rng = np.random.RandomState(12)
    numbers = rng.randn(M, K).astype(np.float32)

    class Memory:
        def __init__(self, array):
            self.__cuda_array_interface__ = {"data": (array.data_ptr, False), "shape": array.shape, "typestr": "<f4", "version": 2}

    y = by_relu(env, numbers)
    env.gpu_op.device_synchronize()
    torch.as_tensor(Memory(y), device="cuda").copy_(torch.from_numpy(numbers * np.float32(1e5)).cuda())
    torch.cuda.synchronize()
    env.gpu_op.array_written(y)
    same_as_a_copy(env, y, "another library")
    whole = env.empty((M + 4, K))
    part = view(env, whole, 4 * K, (M, K))
    env.gpu_op.relu(env.dev(numbers), part)
    env.gpu_op.relu(env.dev(np.concatenate([numbers[:4], numbers * np.float32(1e5)])), whole)
    env.gpu_op.array_written(part)
    same_as_a_copy(env, part, "elsewhere in the same memory")


def test_a_captured_first_call_teaches_the_next_nothing(stage):
    """The first ordinary step behind it has the bits of the second: both know the first layer's maximum, from which the ReLU's pack takes its scale."""
    env = stage
    op, rng = env.gpu_op, np.random.RandomState(13)
    shapes = (13, 64, 40, 40), (64, 64, 1, 1)
    out, first = op.convolution_2d_forward_get_out_shape(*shapes, "NCHW", "VALID", 1, 1)
    second = op.convolution_2d_forward_get_out_shape(out, (64, 64, 1, 1), "NCHW", "VALID", 1, 1)[1]
    act = op.activation_get_cudnnlist(out, "NCHW", "relu")
    x = np.abs(rng.randn(*shapes[0])) * np.where(rng.rand(*shapes[0]) < 0.5, 1, 0)
    w = np.zeros(shapes[1])
    w[np.arange(64), np.arange(64), 0, 0] = np.where(np.arange(64) < 2, -1e8, 1)       # two channels far below zero, which the ReLU takes away
    X, W, W2 = env.dev(x), env.dev(w), env.dev(rng.randn(64, 64, 1, 1))
    y, r, z, kept = env.empty(out), env.empty(out), env.empty(out), env.empty(out)
    op.device_synchronize()
    op.set_contraction_path(2)
    graph = capture(lambda stream: lambda: op.convolution_2d_forward(X, W, kept, first, env.cudnn, stream))
    steps = []
    op.set_contraction_path(2)
    try:
        for _ in range(4):
            before = op.fused_relu_pack_count()
            assert op.convolution_2d_forward(X, W, y, first, env.cudnn, env.stream) == 0
            op.activation_forward(y, r, "relu", act, env.cudnn, env.stream)
            assert op.convolution_2d_forward(r, W2, z, second, env.cudnn, env.stream) == 0
            steps.append(z.asnumpy())
        assert op.fused_relu_pack_count() == before + 1
    finally:
        op.set_contraction_path(0)
    replay(graph)
    np.testing.assert_array_equal(kept.asnumpy(), y.asnumpy())
    for again in steps[1:]:
        np.testing.assert_array_equal(steps[0], again)
