"""Steps of graphs with operators of several results, on the executor's other roads: one update per parameter (data-parallel training, a step that is
timed), and the exchange of their gradients between ranks."""
import os
import sys

import numpy as np
import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _rank_step(block, values):
    """(loss gradients of every parameter, their names) of one rank, in 64 bits."""
    from oracle.graph_eval import OracleExecutor
    from tinyflow_b200 import autodiff as ad
    grads = ad.gradients(block.loss, block.parameters)
    got = OracleExecutor(ad.find_topo_sort(grads)).run({n: v.astype(np.float64) for n, v in values.items()})
    return {n.name: got[g] for n, g in zip(block.parameters, grads)}


def _gloo_rank(rank, world, port, q):
    import torch
    import torch.distributed as dist
    sys.path.insert(0, REPO)
    from tests.block_graph import Block
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    whole = Block(batch=24, dropout=0.0)
    mine = {n: (v[rank * 12:rank * 12 + 12] if n.isw == 2 else v) for n, v in whole.values.items()}
    out = {}
    for name, g in _rank_step(whole, mine).items():
        t = torch.tensor(g)
        dist.all_reduce(t)
        out[name] = t.numpy()
    if rank == 0:
        q.put(out)
    dist.destroy_process_group()


def test_gradients_of_two_ranks_add_up_to_the_whole_batchs():
    """Every part of an operator's results is a gradient of its own to the exchange.  World size 2 over gloo."""
    import multiprocessing as mp
    from tests.block_graph import Block
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = 29500 + (os.getpid() + 977) % 2000
    procs = [ctx.Process(target=_gloo_rank, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = q.get(timeout=120)
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    whole = Block(batch=24, dropout=0.0)
    want = _rank_step(whole, whole.values)
    assert set(got) == set(want) and len(got) == len(whole.parameters)
    for name in want:
        np.testing.assert_allclose(got[name], want[name], rtol=1e-9, atol=1e-12, err_msg=name)


@pytest.mark.gpu
@pytest.mark.parametrize("optimizer", ["sgd", "adam"])
@pytest.mark.parametrize("road", ["data parallel", "timed"])
def test_one_update_per_parameter(lib_path, monkeypatch, optimizer, road):
    """The nodes one by one, as in data-parallel training and in a timed step: the losses and parameters of the step that updates them together."""
    import queue
    import random
    from tests.block_graph import Block
    from tinyflow_b200 import autodiff as ad, gpu_op, ndarray, step_graph
    monkeypatch.setattr(step_graph, "ENABLED", False)
    ctx, runs = ndarray.gpu(0), []
    for other in (False, True):
        random.seed(3)
        block = Block(batch=60, dropout=0.3)
        messages = queue.Queue() if other and road == "timed" else None
        if other and road == "data parallel":
            monkeypatch.setattr(gpu_op, "data_parallel_active", lambda: True)
        ex = ad.Executor(block.loss, block.y, 0.01, None, messages, None, optimizer=optimizer)
        feed = {n: ndarray.array(v, ctx) for n, v in block.values.items()}
        for var in block.parameters:
            for moment in ex.Variable_node_to_mv.get(var, ()):
                feed[moment] = ndarray.array(np.zeros_like(block.values[var]), ctx)
        losses = [ex.run(feed)[0].asnumpy() for _ in range(4)]
        runs.append((losses, {n.name: feed[n].asnumpy() for n in block.parameters}))
    for a, b in zip(runs[0][0], runs[1][0]):
        assert np.isfinite(a).all()
        np.testing.assert_array_equal(a, b)
    for name, v in runs[0][1].items():
        np.testing.assert_array_equal(v, runs[1][1][name], err_msg=name)


@pytest.mark.gpu
def test_a_replayed_step_of_a_long_batch_that_stays_finite(lib_path, monkeypatch):
    """Clusters of 16 in a recorded step, with a rate at which the summed loss of 2500 rows does not overshoot."""
    from tests import test_gpu_gated
    from tinyflow_b200 import autodiff as ad

    class Slow(ad.Executor):
        def __init__(self, loss, y, rate, *rest, **more):
            super().__init__(loss, y, rate / 2500, *rest, **more)

    monkeypatch.setattr(ad, "Executor", Slow)
    kind = dict(batch=2500, width=32, hidden=40, dropout=0.3)
    runs = [test_gpu_gated.block_step(monkeypatch, recorded, 9, **kind) for recorded in (False, True)]
    assert runs[1][4] and not runs[0][4]
    assert all(np.isfinite(v).all() for v in runs[0][2]) and all(np.isfinite(v).all() for v in runs[0][3].values())
    assert all(np.array_equal(a, b) for a, b in zip(runs[0][2], runs[1][2]))
    assert all(np.array_equal(v, runs[1][3][n]) for n, v in runs[0][3].items())


def _plan_every_forward_result(ex, kind):
    """What a forward operator of several results has, released behind its last reader of the forward pass and computed again in front of the first one of
    the backward pass: its own array ("whole"), its further results ("parts"), or all of them."""
    users = {n: [] for n in ex.topo_order}
    for n in ex.topo_order:
        for i in n.inputs:
            users[i].append(n)
    release, again, loss = [], {}, ex.targetloss.index
    for n in reversed(ex.topo_order):                      # what is computed again from another result needs that one back first
        part = type(n.op).__name__ in ("PartOp", "NormalisedSumOp")
        whole = n.inputs[0] if part else n
        if type(whole.op).__name__ not in ("GatedLinearForwardOp", "DropoutAddLayerNormForwardOp") or n.index >= loss or kind not in ("all", "parts" if part else "whole"):
            continue
        if type(n.op).__name__ == "DropoutAddLayerNormForwardOp":
            continue                                       # the next sums read it, and it takes its own inputs
        readers = [u for u in users[n] if not (type(u.op).__name__ in ("PartOp", "NormalisedSumOp") and u.inputs[0] is n)]
        forward, backward = [u.index for u in readers if u.index <= loss], [u.index for u in readers if u.index > loss]
        if not backward:
            continue
        release.append((max(forward + [n.index]), n.index))
        again[n] = min(backward + [at for m, at in again.items() if n in (m.inputs[0].inputs if type(m.op).__name__ == "PartOp" else m.inputs)])
    assert again
    return [], release, [(at, n.index) for n, at in reversed(list(again.items()))]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["whole", "parts", "all"])
@pytest.mark.parametrize("optimizer", ["sgd", "adam"])
def test_results_computed_again(lib_path, monkeypatch, kind, optimizer):
    """A plan that lets go of every result it can: the bits of the step without one."""
    from tests import test_gpu_gated
    want = test_gpu_gated.block_step(monkeypatch, steps=3, dropout=0.4, optimizer=optimizer)
    got = test_gpu_gated.block_step(monkeypatch, steps=3, dropout=0.4, optimizer=optimizer, plan=lambda ex: _plan_every_forward_result(ex, kind))
    for a, b in zip(want[2], got[2]):
        np.testing.assert_array_equal(a, b)
    for name, v in want[3].items():
        np.testing.assert_array_equal(v, got[3][name], err_msg=name)
