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
