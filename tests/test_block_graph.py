"""Graphs of layer norms, residual norms and gated layers: their gradients, as the graph forms them, against differences, on the CPU."""
import numpy as np
import pytest

from tests.block_graph import Block


def gradient_order(block):
    from tinyflow_b200 import autodiff as ad
    grads = ad.gradients(block.loss, block.parameters)
    return grads, ad.find_topo_sort(grads + [block.loss])


def loss_of(block, order, values):
    from oracle.graph_eval import OracleExecutor
    from tinyflow_b200 import autodiff as ad
    return float(OracleExecutor(ad.find_topo_sort([block.loss])).run(values)[block.loss].sum())


@pytest.mark.parametrize("dropout", [0.0, 0.25])
@pytest.mark.parametrize("activations", [("silu", "gelu"), ("sigmoid", "tanh"), ("silu",)])
def test_gradients_against_differences(dropout, activations):
    """Central differences in 64 bits, step 1e-5: truncation of 1e-10 times a third derivative, cancellation of 1e-11."""
    from oracle.graph_eval import OracleExecutor
    block = Block(dropout=dropout, activations=activations)
    for k, node in enumerate(block.residuals):
        node.seed[0] = 3 + k
    grads, order = gradient_order(block)
    values = {n: v.astype(np.float64) for n, v in block.values.items()}
    got = OracleExecutor(order).run(values)
    rng = np.random.RandomState(1)
    batch = len(values[block.X])             # the loss is a mean over rows, its gradient is the sum's
    for node, grad in zip(block.parameters, grads):
        assert got[grad].shape == values[node].shape
        for _ in range(4):
            at = tuple(rng.randint(0, n) for n in values[node].shape)
            sides = []
            for step in (1e-5, -1e-5):
                moved = dict(values)
                moved[node] = values[node].copy()
                moved[node][at] += step
                sides.append(loss_of(block, order, moved))
            want = (sides[0] - sides[1]) / 2e-5
            assert abs(got[grad][at] / batch - want) <= 1e-7 * (1 + abs(want)), (node.name, at)


def test_what_reaches_a_residual_sum_is_added_by_the_norms_kernel():
    """Both gradients of a residual sum - through the norm and past it - come out of one operator: no sum is left between them."""
    block = Block()
    _, order = gradient_order(block)
    kinds = [type(n.op).__name__ for n in order]
    assert kinds.count("DropoutAddLayerNormBackwardOp") == 2 and all(len(n.inputs) == 4 for n in order if type(n.op).__name__ == "DropoutAddLayerNormBackwardOp")
    assert kinds.count("AddOp") == 2                      # the one in front of the last norm, and softmax - labels of the loss
    assert not any(k.startswith("Zeros") for k in kinds)


def test_a_norm_that_nobody_reads():
    from oracle.graph_eval import OracleExecutor
    from tinyflow_b200 import autodiff as ad
    rng = np.random.RandomState(2)
    h, r, g, b = (ad.Variable(n) for n in "hrgb")
    total, _ = ad.dropout_add_layer_norm_op(h, r, g, b, 0.5)
    total.seed[0] = 4
    loss = ad.reduce_sum_op(total * total)
    dh, dr = ad.gradients(loss, [h, r])
    values = {n: rng.randn(*s) for n, s in ((h, (3, 5)), (r, (3, 5)), (g, (5,)), (b, (5,)))}
    got = OracleExecutor(ad.find_topo_sort([dh, dr])).run(values)
    from oracle import ops
    keep = ops.dropout(np.ones((3, 5)), 0.5, 4)
    want = 2 * (values[r] + keep * values[h])
    np.testing.assert_allclose(got[dr], want, rtol=1e-12)
    np.testing.assert_allclose(got[dh], want * keep, rtol=1e-12)


def test_shapes_and_the_executors_order(lib_path):
    from tinyflow_b200 import autodiff as ad, memory_plan
    block = Block(batch=21, width=24, hidden=20)
    ex = ad.Executor(block.loss, block.y, 0.1, optimizer="sgd")
    ex.infer_shape({n: v.shape for n, v in block.values.items()})
    for var in block.parameters:
        assert ex.node_to_shape_map[ex.Variable_node_to_grad[var]] == block.values[var].shape
    for node in ex.topo_order:
        if type(node.op).__name__ == "PartOp" and type(node.inputs[0].op).__name__ == "GatedLinearForwardOp":
            assert ex.node_to_shape_map[node] == (21, 40)
    memory_plan.check_plan(ex, memory_plan.vdnn_plan(ex, policy="all", min_bytes=1))
    ad.Executor(block.loss, block.y, 0.1, optimizer="adam")             # a second one on the same graph
    total = block.residuals[0]
    again = ad.normalised_sum_op(total, total.inputs[2], total.inputs[3])
    with pytest.raises(ValueError, match="twice"):
        ad.Executor(block.loss + ad.reduce_sum_op(again), block.y, 0.1)
    gates = ad.part_op(next(n for n in ex.topo_order if type(n.op).__name__ == "GatedLinearForwardOp"), 1)
    with pytest.raises(NotImplementedError):
        ad.gradients(ad.reduce_sum_op(gates), [block.parameters[0]])


@pytest.mark.parametrize("op,inputs", [("layer_norm_op", 3), ("dropout_add_layer_norm_op", 4), ("gated_linear_op", 2)])
def test_there_is_no_cpu_path(op, inputs):
    from tinyflow_b200 import autodiff as ad
    node = getattr(ad, op)(*(ad.Variable("v%d" % i) for i in range(inputs)))
    node = node[0] if isinstance(node, tuple) else node
    with pytest.raises(NotImplementedError):
        node.op.compute(node, [None] * inputs, [None, None], None, None, None, use_numpy=True)


def residual_sum(readers):
    """(sum, its normalisation, inputs, loss): the loss reads the normalisation and, `readers` times, the sum."""
    from tinyflow_b200 import autodiff as ad
    h, r, g, b = (ad.Variable(n) for n in "hrgb")
    total, y = ad.dropout_add_layer_norm_op(h, r, g, b, 0.0)
    whole = y * y * y
    for _ in range(readers):
        whole = whole + total * total
    rng = np.random.RandomState(3)
    return total, y, {n: rng.randn(*s) for n, s in ((h, (3, 5)), (r, (3, 5)), (g, (5,)), (b, (5,)))}, ad.reduce_sum_op(whole)


@pytest.mark.parametrize("readers", [0, 1, 2])
def test_the_gradient_of_a_residual_sum_itself(readers):
    """Asked for by name it is what reaches the residual input (the sum is that plus the branch), once, however many read the sum."""
    from oracle.graph_eval import OracleExecutor
    from tinyflow_b200 import autodiff as ad
    total, y, values, loss = residual_sum(readers)
    h, r, g, b = values
    grads = ad.gradients(loss, [total, r, h, y, g, b])
    got = OracleExecutor(ad.find_topo_sort(grads + [loss])).run(values)
    dtotal, dr, dh, dy = (got[n] for n in grads[:4])
    np.testing.assert_allclose(dy, 3 * got[y] ** 2, rtol=1e-12)
    np.testing.assert_array_equal(dtotal, dr)
    np.testing.assert_array_equal(dtotal, dh)
    order = ad.find_topo_sort([loss])

    def at(**moved):
        return float(OracleExecutor(order).run({n: moved.get(n.name, v) for n, v in values.items()})[loss].sum())

    # central differences, step 1e-5: truncation of 1e-10 times a third derivative, cancellation of 1e-11 times the loss
    for node, grad in zip((r, g, b), (dtotal, got[grads[4]], got[grads[5]])):
        for i in np.ndindex(values[node].shape):
            sides = []
            for step in (1e-5, -1e-5):
                v = values[node].copy()
                v[i] += step
                sides.append(at(**{node.name: v}))
            want = (sides[0] - sides[1]) / 2e-5
            assert abs(grad[i] - want) <= 1e-7 * (1 + abs(want)), (node.name, i)


def test_two_normalisations_of_one_sum_and_gradients_taken_twice():
    from oracle import ops
    from oracle.graph_eval import OracleExecutor
    from tinyflow_b200 import autodiff as ad
    total, y, values, _ = residual_sum(0)
    h, r, g, b = values
    loss = ad.reduce_sum_op(y * y * y + ad.normalised_sum_op(total, g, b) * total)
    first, second = ad.gradients(loss, [total, g]), ad.gradients(loss, [total, g])
    got = OracleExecutor(ad.find_topo_sort(first + second)).run(values)
    s = values[h] + values[r]
    n = ops.layer_norm(s, values[g], values[b], 1e-5)[0]
    dx, dg, _ = ops.layer_norm_backward(s, values[g], 3 * n * n + s, 1e-5)
    for total_grad, gamma_grad in (first, second):
        np.testing.assert_allclose(got[total_grad], dx + n, rtol=1e-9, atol=1e-12)
        np.testing.assert_allclose(got[gamma_grad], dg, rtol=1e-9, atol=1e-12)
