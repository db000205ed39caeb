"""Rotations whose frequencies and amplitude the caller gives: on the CPU what is refused and graphs of them, on the GPU their kernels against the formula in 64 bits."""
import numpy as np
import pytest

from oracle import ops
from tests.test_gpu_norm import within
from tests.test_gpu_ops import env  # noqa: F401
from tests.test_norm_refusals import op, refused  # noqa: F401

U = 2.0 ** -24


def test_refusals(op):
    for bad in (dict(frequencies=[1.0, 0.1], rotated=6), dict(frequencies=[1.0], scaling="linear", factor=2.0), dict(frequencies=[1.0], rotated=0)):
        with pytest.raises(AssertionError):
            op.rotary_state(8, **bad)
    refused(lambda: op.rotary_state(8, frequencies=[1.0] * 5), "do not fit")
    refused(lambda: op.rotary_state(8, frequencies=[1.0, float("nan")]), "frequency 1")
    refused(lambda: op.rotary_state(8, amplitude=float("inf")), "amplitude")
    op.rotary_state(8, frequencies=[])


@pytest.mark.parametrize("rotation", [dict(frequencies=[0.7, 0.01], amplitude=1.3), dict(frequencies=np.array([0.3, 0.2, 0.1]), layout="interleaved"),
                                      dict(scaling="parts", factor=8.0, trained=64, high=4.0, amplitude=1.0)], ids=["given", "all pairs", "parts"])
@pytest.mark.parametrize("norm", [False, True])
def test_gradients_of_graphs_against_differences(rotation, norm):
    """Central differences in 64 bits, step 1e-5."""
    from oracle.graph_eval import OracleExecutor
    from tinyflow_b200 import autodiff as ad
    rng = np.random.RandomState(0)
    X, W, gq, gk, P = ad.Placeholder("X"), ad.Variable("W"), ad.Variable("gq"), ad.Variable("gk"), ad.Placeholder("P")
    values = {X: rng.randn(6, 5), W: rng.randn(5, 12), gq: 1 + rng.randn(6), gk: 1 + rng.randn(6), P: rng.randn(6, 12)}
    q = ad.matmul_op(X, W)
    if norm:
        q, k = ad.head_norm_rotary_op(q, q, gq, gk, 6, 3, start=40, **rotation)
        y = q * P + k
    else:
        y = ad.rotary_op(q, 6, 3, start=40, **rotation) * P
    loss = ad.reduce_sum_op(y)
    wanted = [W, gq, gk] if norm else [W]
    grads = ad.gradients(loss, wanted)
    got, order = OracleExecutor(ad.find_topo_sort(grads)).run(values), ad.find_topo_sort([loss])
    total = lambda v: float(OracleExecutor(order).run(v)[loss].sum())      # noqa: E731
    for w, g in zip(wanted, (got[n] for n in grads)):
        for _ in range(4):
            at = tuple(rng.randint(0, n) for n in values[w].shape)
            sides = []
            for step in (1e-5, -1e-5):
                moved = dict(values)
                moved[w] = values[w].copy()
                moved[w][at] += step
                sides.append(total(moved))
            want = (sides[0] - sides[1]) / 2e-5
            assert abs(g[at] - want) <= 1e-6 * (1 + abs(want))
    if not norm and rotation.get("amplitude") == 1.3:
        turned = ops.rotary(values[X] @ values[W], 6, ops.rotary_angles(6, 3, 40, None, [0.7, 0.01]), 1.3, "half")
        assert np.allclose(total(values), (turned * values[P]).sum(), rtol=1e-12)


@pytest.mark.gpu
@pytest.mark.parametrize("D, given", [(8, dict(frequencies=[0.5, -0.25, 3.0], amplitude=0.75)), (64, dict(frequencies=np.linspace(1, 0.001, 32))), (33, dict(frequencies=[1e3], layout="interleaved")),
                                      (128, dict(scaling="parts", factor=8.0, trained=4096, high=4.0, amplitude=1.0))], ids=["signs", "all", "one", "parts"])
def test_kernels(env, D, given):
    """As in test_gpu_rotary.py: 8 u A (|a| + |b|), here of the largest two elements of a head."""
    rng = np.random.RandomState(D)
    x = rng.randn(14, 3 * D).astype(np.float32)
    state = env.gpu_op.rotary_state(D, **given)
    f, amplitude = given.get("frequencies"), given.get("amplitude", 1.0)
    if f is None:
        f = env.gpu_op.rotary_frequencies(D, 10000.0, "parts", 8.0, 4096, 1.0, 4.0)[0]
    X, Y, B = env.dev(x), env.empty(x.shape), env.empty(x.shape)
    env.gpu_op.rotary_forward(X, None, Y, 7, 1000, state, env.stream)
    env.gpu_op.rotary_backward(X, None, B, 7, 1000, state, env.stream)
    angles, layout = ops.rotary_angles(14, 7, 1000, None, f), given.get("layout", "half")
    bound = 8 * U * 2 * max(1.0, amplitude) * np.abs(x).max()
    for got, back in ((Y, False), (B, True)):
        want = ops.rotary(x.astype(np.float64), D, angles, amplitude, layout, back)
        within(got.asnumpy(), want, np.full(x.shape, bound), "back" if back else "forward")
