"""Graphs of normed, rotated heads and attention: their gradients, as the graph forms them, against differences, on the CPU; and steps of them on the GPU."""
import numpy as np
import pytest

from tests.test_gpu_ops import env  # noqa: F401


class Attended:
    """Projections of packed documents, normed and rotated heads, attention over shared heads, and a residual."""

    def __init__(self, batch=2, length=9, width=12, heads=4, kv_heads=2, dim=6, classes=5, seed=0, positions=False, norm=True, documents=True, **attention):
        from tinyflow_b200 import autodiff as ad
        rng = np.random.RandomState(seed)
        rows = batch * length
        self.X, self.y_ = ad.Placeholder("X"), ad.Placeholder("y_")
        self.values = {}

        def given(node, value):
            self.values[node] = np.asarray(value, np.float32)
            return node

        def weight(name, *shape, around=0.0):
            return given(ad.Variable(name), around + rng.randn(*shape) * (0.2 if len(shape) == 1 else shape[0] ** -0.5))

        q, k, v = (ad.matmul_op(self.X, weight("W" + n, width, h * dim)) for n, h in (("q", heads), ("k", kv_heads), ("v", kv_heads)))
        at = given(ad.Placeholder("positions"), rng.permutation(rows)) if positions else None
        if norm:
            q, k = ad.head_norm_rotary_op(q, k, weight("gq", dim, around=1.0), weight("gk", dim, around=1.0), dim, length, at, rotated=4, scaling="linear", factor=2.0)
        else:
            q, k = (ad.rotary_op(x, dim, length, at, layout="interleaved") for x in (q, k))
        docs = np.repeat(np.arange(4), rows)[:: 4][:rows].astype(np.float32)
        docs.reshape(batch, length)[:, -1] = -1
        masks = dict(documents=given(ad.Placeholder("documents"), docs)) if documents else {}
        if attention.pop("bias", False):
            masks["slopes"] = given(ad.Placeholder("slopes"), 2.0 ** -np.arange(1, heads + 1))
        if "prefix" in attention:
            masks["prefix"] = given(ad.Placeholder("prefix"), np.full(batch, attention.pop("prefix")))
        self.attended = ad.attention_op(q, k, v, heads, length, kv_heads, **masks, **attention)
        h = ad.matmul_op(self.attended, weight("Wo", heads * dim, width)) + self.X
        self.y = ad.matmul_op(h, weight("Wc", width, classes))
        self.loss = ad.softmaxcrossentropy_op(self.y, self.y_)
        labels = np.zeros((rows, classes))
        labels[np.arange(rows), rng.randint(0, classes, rows)] = 1
        given(self.X, rng.randn(rows, width))
        given(self.y_, labels)
        self.parameters = [n for n in self.values if n.isw == 1]


KINDS = [dict(), dict(norm=False, positions=True, documents=False, window=4, cap=1.5), dict(positions=True, bias=True, causal=False, window=3), dict(documents=False, prefix=3, norm=False),
         dict(heads=3, kv_heads=3, scale=0.3)]


@pytest.mark.parametrize("kind", KINDS)
def test_gradients_against_differences(kind):
    """Central differences in 64 bits, step 1e-5: truncation of 1e-10 times a third derivative, cancellation of 1e-11."""
    from oracle.graph_eval import OracleExecutor
    from tinyflow_b200 import autodiff as ad
    g = Attended(**kind)
    grads = ad.gradients(g.loss, g.parameters)
    values = {n: v.astype(np.float64) for n, v in g.values.items()}
    got = OracleExecutor(ad.find_topo_sort(grads)).run(values)
    order = ad.find_topo_sort([g.loss])
    loss = lambda v: float(OracleExecutor(order).run(v)[g.loss].sum())      # noqa: E731
    rng = np.random.RandomState(1)
    batch = len(values[g.X])                 # the loss is a mean over rows, its gradient is the sum's
    for node, grad in zip(g.parameters, grads):
        assert got[grad].shape == values[node].shape
        for _ in range(4):
            at = tuple(rng.randint(0, n) for n in values[node].shape)
            sides = []
            for step in (1e-5, -1e-5):
                moved = dict(values)
                moved[node] = values[node].copy()
                moved[node][at] += step
                sides.append(loss(moved))
            want = (sides[0] - sides[1]) / 2e-5
            assert abs(got[grad][at] / batch - want) <= 1e-7 * (1 + abs(want)), (node.name, at)


def test_one_operator_takes_the_gradients_of_queries_and_keys():
    from tinyflow_b200 import autodiff as ad
    g = Attended()
    order = ad.find_topo_sort(ad.gradients(g.loss, g.parameters))
    kinds = [type(n.op).__name__ for n in order]
    assert kinds.count("HeadNormRotaryBackwardOp") == 1 and kinds.count("AttentionBackwardOp") == 1 and "KeysGradientOp" not in kinds


def test_keys_or_queries_that_nobody_reads():
    from oracle import ops
    from oracle.graph_eval import OracleExecutor
    from tinyflow_b200 import autodiff as ad
    rng = np.random.RandomState(0)
    q, k, gq, gk = (ad.Variable(n) for n in ("q", "k", "gq", "gk"))
    values = {q: rng.randn(6, 8), k: rng.randn(6, 4), gq: rng.randn(4), gk: rng.randn(4)}
    angles = ops.rotary_angles(6, 3, 0, None, [1.0, 0.01])
    for keys in (False, True):
        yq, yk = ad.head_norm_rotary_op(q, k, gq, gk, 4, 3)
        y = yk if keys else yq
        grads = ad.gradients(ad.reduce_sum_op(y * y), [q, k, gq, gk])
        got = [OracleExecutor(ad.find_topo_sort(grads)).run(dict(values))[n] for n in grads]
        x, gamma = (values[k], values[gk]) if keys else (values[q], values[gq])
        dy = 2 * ops.head_norm_rotary(x, gamma, 4, angles, 1.0, "half", 1e-6)
        dx, dg = ops.head_norm_rotary_backward(x, gamma, dy, 4, angles, 1.0, "half", 1e-6)
        np.testing.assert_allclose(got[1 if keys else 0], dx, rtol=1e-9, atol=1e-12)
        np.testing.assert_allclose(got[3 if keys else 2], dg, rtol=1e-9, atol=1e-12)
        assert not got[0 if keys else 1].any() and not got[2 if keys else 3].any()


def test_the_gradient_of_queries_by_name():
    """What reaches the normed queries themselves, with keys that are read beside them."""
    from oracle.graph_eval import OracleExecutor
    from tinyflow_b200 import autodiff as ad
    rng = np.random.RandomState(0)
    q, k, gq, gk = (ad.Variable(n) for n in ("q", "k", "gq", "gk"))
    values = {q: rng.randn(6, 8), k: rng.randn(6, 8), gq: rng.randn(4), gk: rng.randn(4)}
    yq, yk = ad.head_norm_rotary_op(q, k, gq, gk, 4, 3)
    dyq, dyk = ad.gradients(ad.reduce_sum_op(yq * yk + yk * yk), [yq, yk])
    got = OracleExecutor(ad.find_topo_sort([dyq, dyk])).run(values)
    np.testing.assert_allclose(got[dyq], got[yk], rtol=1e-12)
    np.testing.assert_allclose(got[dyk], got[yq] + 2 * got[yk], rtol=1e-12)


def test_shapes_and_the_executors_order(lib_path):
    from tinyflow_b200 import autodiff as ad, memory_plan
    g = Attended()
    ex = ad.Executor(g.loss, g.y, 0.1, optimizer="sgd")
    ex.infer_shape({n: v.shape for n, v in g.values.items()})
    for var in g.parameters:
        assert ex.node_to_shape_map[ex.Variable_node_to_grad[var]] == g.values[var].shape
    assert ex.node_to_shape_map[g.attended] == (18, 24) and ex.node_to_shape_map[g.attended.kept[0]] == (18 * 4, 2)
    memory_plan.check_plan(ex, memory_plan.vdnn_plan(ex, policy="all", min_bytes=1))
    for node in ex.topo_order:
        if type(node.op).__name__ in ("AttentionForwardOp", "HeadNormRotaryForwardOp", "AttentionBackwardOp", "HeadNormRotaryBackwardOp"):
            with pytest.raises(NotImplementedError):
                node.op.compute(node, [None] * 6, [None] * 4, None, None, None, use_numpy=True)


def step(monkeypatch, recorded, steps, optimizer="sgd", **kind):
    from tinyflow_b200 import autodiff as ad, gpu_op, ndarray, step_graph
    monkeypatch.setattr(step_graph, "ENABLED", recorded)
    g = Attended(**kind)
    ex = ad.Executor(g.loss, g.y, 1e-3, None, None, None, optimizer=optimizer)
    ctx = ndarray.gpu(0)
    feed = {n: ndarray.array(v, ctx) for n, v in g.values.items()}
    for var in g.parameters:
        for moment in ex.Variable_node_to_mv.get(var, ()):
            feed[moment] = ndarray.array(np.zeros_like(g.values[var]), ctx)
    losses = [ex.run(feed)[0] for _ in range(steps)]
    gpu_op.device_synchronize()
    replayed = any(f.recording or any(b.recording for b in f.batches.values()) for f in ex._recordings.sets.values())
    return g, ex, [v.asnumpy() for v in losses], {n.name: feed[n].asnumpy() for n in g.parameters}, replayed


LARGE = dict(batch=2, length=300, width=64, heads=4, kv_heads=2, dim=64, classes=7)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS + [LARGE, dict(LARGE, dim=128, cap=20.0, bias=True, window=100)])
def test_every_node_of_a_step_against_the_oracle(env, monkeypatch, kind):      # noqa: F811
    """Each node on the inputs it had: 1e-4 of the element with a floor of 1 % of the tensor's largest or its inputs', as the library's other operators; products 2e-5 of
    the tensor's rms beside it.  (The bounds of single roundings are in the operators' own tests.)"""
    from oracle.graph_eval import OracleExecutor
    g, ex, losses, _, _ = step(monkeypatch, False, 1, **kind)
    orc = OracleExecutor(ex.topo_order, np.float64)
    first = {n: v.astype(np.float64) for n, v in g.values.items()}
    value = lambda n: ex.value_of(n).asnumpy().astype(np.float64)     # noqa: E731
    for node in ex.topo_order:
        if not node.inputs or node.issgd:
            continue
        ins = [first[i] if i in first else value(i) for i in node.inputs]
        want = np.asarray(orc._eval(node, ins), np.float64)
        got = value(node).reshape(want.shape)
        tolerance = 2e-5 * np.linalg.norm(want) / np.sqrt(want.size) + 1e-4 * np.maximum(np.abs(want), 1e-2 * max([np.abs(want).max()] + [np.abs(i).max() for i in ins]))
        assert (np.abs(got - want) <= tolerance).all(), (node.index, node.name, float(np.abs(got - want).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("optimizer", ["sgd", "adam"])
@pytest.mark.parametrize("kind", [dict(positions=True, bias=True), LARGE, dict(LARGE, dim=40, cap=5.0, heads=8)])
def test_a_replayed_step_has_the_bits_of_the_ordinary_one(env, monkeypatch, optimizer, kind):      # noqa: F811
    runs = [step(monkeypatch, recorded, 8, optimizer, **kind) for recorded in (False, True)]
    assert runs[1][4] and not runs[0][4]
    assert all(np.isfinite(v).all() for v in runs[0][2])
    for a, b in zip(runs[0][2], runs[1][2]):
        np.testing.assert_array_equal(a, b)
    for name, v in runs[0][3].items():
        np.testing.assert_array_equal(v, runs[1][3][name], err_msg=name)


@pytest.mark.gpu
def test_results_computed_again(env, monkeypatch):      # noqa: F811
    """A plan that lets go of the attention's output and the rotated heads after their last forward reader and computes them again: no bit changes."""
    import queue
    from tinyflow_b200 import autodiff as ad, ndarray, step_graph
    monkeypatch.setattr(step_graph, "ENABLED", False)

    def train(planned):
        g = Attended(**LARGE)
        control = queue.Queue()
        ex = ad.Executor(g.loss, g.y, 1e-3, control, None, None, optimizer="sgd")
        feed = {n: ndarray.array(v, ndarray.gpu(0)) for n, v in g.values.items()}
        if planned:
            ex.infer_shape({n: v.shape for n, v in feed.items()})
            loss = ex.targetloss.index
            release, again = [], {}
            for n in reversed(ex.topo_order):              # what is computed again from another result needs that one back first
                if type(n.op).__name__ not in ("AttentionForwardOp", "HeadNormRotaryForwardOp") or n.index >= loss:
                    continue
                readers = [u.index for u in ex.topo_order if n in u.inputs and not (type(u.op).__name__ in ("PartOp", "NormedKeysOp"))]
                backward = [i for i in readers if i > loss]
                if backward:
                    release.append((max(i for i in readers + [n.index] if i <= loss), n.index))
                    again[n] = min(backward + [at for m, at in again.items() if n in m.inputs])
            assert len(again) == 2
            control.put(([], release, [(at, n.index) for n, at in reversed(list(again.items()))]))
        losses = [ex.run(feed)[0].asnumpy() for _ in range(3)]
        return losses, {n.name: feed[n].asnumpy() for n in g.parameters}

    plain, planned = train(False), train(True)
    for a, b in zip(plain[0], planned[0]):
        np.testing.assert_array_equal(a, b)
    for name, v in plain[1].items():
        np.testing.assert_array_equal(v, planned[1][name], err_msg=name)
