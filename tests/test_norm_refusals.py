"""What the layer-norm calls refuse, before anything touches a device (the arrays here are only described)."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def op(lib_path):
    from tinyflow_b200 import gpu_op
    return gpu_op


def described(shape, at, device=0, kind=2):
    from tinyflow_b200 import ndarray as nd
    c = nd.DLArray()
    dims = (ctypes.c_int64 * max(1, len(shape)))(*shape)
    c.data, c.ctx, c.ndim, c.shape = at, nd.DLContext(device, kind), len(shape), ctypes.cast(dims, ctypes.POINTER(ctypes.c_int64))
    arr = nd.NDArray(ctypes.pointer(c))
    arr.is_freed, arr._owner = True, dims
    return arr


MB = 1 << 20


def arrays():
    big, small = (6, 40), (40,)
    return {"x": described(big, MB), "gamma": described(small, 2 * MB), "beta": described(small, 3 * MB), "y": described(big, 4 * MB), "dy": described(big, 5 * MB),
            "dx": described(big, 6 * MB), "dg": described(small, 7 * MB), "db": described(small, 8 * MB), "r": described(big, 9 * MB), "s": described(big, 10 * MB),
            "dh": described(big, 11 * MB), "ds": described(big, 12 * MB)}


def calls(op, a, eps=1e-5, state=None):
    state = state or op.dropout_state(0.5, 1)
    yield lambda: op.layer_norm_forward(a["x"], a["gamma"], a["beta"], a["y"], eps, None)
    yield lambda: op.layer_norm_backward(a["x"], a["gamma"], a["dy"], a["dx"], a["dg"], a["db"], eps, None)
    yield lambda: op.dropout_add_layer_norm_forward(a["x"], a["r"], a["gamma"], a["beta"], a["s"], a["y"], state, eps, None)
    yield lambda: op.dropout_add_layer_norm_backward(a["s"], a["gamma"], a["dy"], a["ds"], a["dh"], a["dx"], a["dg"], a["db"], state, eps, None)


USED = [("x", "gamma", "beta", "y"), ("x", "gamma", "dy", "dx", "dg", "db"), ("x", "r", "gamma", "beta", "s", "y"), ("s", "gamma", "dy", "ds", "dh", "dx", "dg", "db")]
WRITTEN = [("y",), ("dx", "dg", "db"), ("s", "y"), ("dh", "dx", "dg", "db")]


def refused(call, words):
    from tinyflow_b200._base import TinyflowError
    with pytest.raises(TinyflowError, match=words):
        call()


@pytest.mark.parametrize("k", range(4))
def test_arrays_elsewhere_of_another_size_or_without_memory(op, k):
    for name in USED[k]:
        for changed, words in ((dict(kind=1), "not on the GPU"), (dict(device=1), "another GPU"), (dict(at=0), "no memory"), (dict(at=MB + 2), "not aligned")):
            a = arrays()
            shape = a[name].shape
            a[name] = described(shape, **{"at": a[name].data_ptr, **changed})
            refused(list(calls(op, a))[k], words)
        a = arrays()
        first = name == USED[k][0]
        a[name] = described(tuple(n + 1 for n in a[name].shape), a[name].data_ptr)
        if not first:
            refused(list(calls(op, a))[k], "size")


@pytest.mark.parametrize("k", range(4))
def test_results_that_share_memory(op, k):
    for out in WRITTEN[k]:
        for other in USED[k]:
            if other == out:
                continue
            a = arrays()
            a[out] = described(a[out].shape, a[other].data_ptr + 4)
            refused(list(calls(op, a))[k], "shares memory")


@pytest.mark.parametrize("k", range(4))
def test_bad_numbers(op, k):
    for eps in (-1e-5, float("inf"), float("nan")):
        refused(list(calls(op, arrays(), eps=eps))[k], "eps")
    a = arrays()
    for name in ("x", "s"):
        a[name] = described((), MB)
    refused(list(calls(op, a))[k], "axis")


def test_states(op):
    from tinyflow_b200._base import new_cell
    for rate in (1.0, -0.1, float("nan")):
        refused(lambda: op.dropout_state(rate, 1), "rate")
    for k in (2, 3):
        refused(list(calls(op, arrays(), state=new_cell(3)))[k], "state")
    state = op.dropout_state(0.1, 1)
    assert op.dropout_state(0.2, 3, state) is state


def test_a_cell_that_holds_another_descriptor(op):
    """It keeps it: the state of a residual norm takes an empty cell, or one that holds such a state."""
    cell = op.activation_get_cudnnlist((2, 3), "NCHW", "relu")
    held = cell[0]
    refused(lambda: op.dropout_state(0.5, 1, cell), "another descriptor")
    import ctypes
    address = lambda c: ctypes.cast(c, ctypes.c_void_p).value        # noqa: E731
    assert address(cell[0]) == address(held)
    state = op.dropout_state(0.5, 1)
    assert op.dropout_state(0.25, 2, state) is state


def test_a_write_of_an_array_that_is_not_on_a_gpu(op):
    refused(lambda: op.array_written(described((2, 3), MB, kind=1)), "device array")
    refused(lambda: op.array_written(described((2, 3), 0)), "device array")
    op.array_written(described((2, 3), MB))
    op.array_written(described((0, 3), 0))
