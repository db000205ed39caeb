"""Attention and norms of heads with several calls in flight: each stream has scratch and counters of its own, and results are the bits of one call after another."""
import numpy as np
import pytest

from tests.test_gpu_attention import Case, env  # noqa: F401

pytestmark = pytest.mark.gpu

class Held:
    """Arrays of a case and both directions' calls on them."""

    def __init__(self, env, c):
        on = lambda v: None if v is None else env.nd.array(v, env.ctx)      # noqa: E731
        self.op, self.state, self.masks = env.gpu_op, c.state(env), [on(a) for a in (c.documents, c.prefix, c.slopes)]
        self.arrays, self.dout = [on(a) for a in (c.q, c.k, c.v)], on(c.dout)
        self.out, self.stats = env.nd.empty(c.q.shape, env.ctx), env.nd.empty((c.batch, c.heads, c.queries, 2), env.ctx)
        self.grads = [env.nd.empty(a.shape, env.ctx) for a in (c.q, c.k, c.v)]

    def step(self, stream):
        assert not self.op.attention_forward(*self.arrays, *self.masks, self.out, self.stats, self.state, stream)
        assert not self.op.attention_backward(*self.arrays, *self.masks, self.out, self.stats, self.dout, *self.grads, self.state, stream)

    def results(self):
        return [a.asnumpy() for a in (self.out, self.stats, *self.grads)]

    def spoil(self):
        for a in (self.out, self.stats, *self.grads):
            a[:] = np.full(a.shape, np.nan, np.float32)


SEVERAL = [dict(batch=2, queries=500, keys=500, heads=4, kv_heads=2, dim=64), dict(batch=1, queries=300, keys=300, heads=4, kv_heads=4, dim=128, documents="packed"), dict(batch=3, queries=40, keys=40, heads=2, kv_heads=1, dim=200),
           dict(batch=2, queries=3, keys=900, heads=8, kv_heads=2, dim=64), dict(batch=1, queries=700, keys=700, heads=8, kv_heads=1, dim=64, cap=5.0)]


def test_steps_on_several_streams_at_once(env):
    """Both directions, tokens that are apart among them: the bits of one after another."""
    cases = [Case(**k) for k in SEVERAL]
    cases[0].v[::7] *= np.float32(2.0 ** 20)
    held = [Held(env, c) for c in cases]
    for h in held:
        h.step(env.stream)
    env.gpu_op.device_synchronize()
    want = [h.results() for h in held]
    streams = [env.gpu_op.create_cudaStream() for _ in held]
    for h in held:
        h.spoil()
    env.gpu_op.device_synchronize()
    for _ in range(10):
        for h, s in zip(held, streams):
            h.step(s)
    env.gpu_op.device_synchronize()
    for h, w in zip(held, want):
        for got, a in zip(h.results(), w):
            assert np.array_equal(got, a)
    for s in streams:
        env.gpu_op.destroy_cudaStream(s)


def test_large_and_small_steps_in_turn_on_one_stream(env):
    """Scratch that grows while smaller calls are in flight."""
    cases = [Case(**k) for k in (SEVERAL[3], SEVERAL[2], SEVERAL[1], SEVERAL[0], SEVERAL[4])]
    held = [Held(env, c) for c in cases]
    for h in held:
        h.step(env.stream)
    env.gpu_op.device_synchronize()
    want = [h.results() for h in held]
    for h in held:
        h.spoil()
    env.gpu_op.device_synchronize()
    stream = env.gpu_op.create_cudaStream()
    for order in (range(5), reversed(range(5)), range(5)):
        for i in order:
            held[i].step(stream)
    env.gpu_op.device_synchronize()
    for h, w in zip(held, want):
        for got, a in zip(h.results(), w):
            assert np.array_equal(got, a)
    env.gpu_op.destroy_cudaStream(stream)


def test_norms_of_heads_on_several_streams_at_once(env):
    op, nd = env.gpu_op, env.nd
    rng = np.random.RandomState(0)
    on = lambda *s: nd.array(rng.randn(*s).astype(np.float32), env.ctx)      # noqa: E731
    calls = []
    for tokens, heads, kv, dim in ((3000, 8, 2, 64), (777, 6, 2, 80), (40, 4, 4, 33), (5000, 4, 1, 128)):
        q, k, gq, gk, dq, dk = on(tokens, heads * dim), on(tokens, kv * dim), on(dim), on(dim), on(tokens, heads * dim), on(tokens, kv * dim)
        out = [nd.empty(s, env.ctx) for s in ((tokens, heads * dim), (tokens, kv * dim), (dim,), (dim,))]
        state = op.rotary_state(dim)
        calls.append((out, lambda s, q=q, k=k, gq=gq, gk=gk, dq=dq, dk=dk, out=out, state=state:
                      op.head_norm_rotary_backward(q, k, gq, gk, None, dq, dk, *out, 50, 0, 1e-6, state, s)))
    for _, call in calls:
        assert not call(env.stream)
    op.device_synchronize()
    want = [[a.asnumpy() for a in out] for out, _ in calls]
    for out, _ in calls:
        for a in out:
            a[:] = np.full(a.shape, np.nan, np.float32)
    op.device_synchronize()
    streams = [op.create_cudaStream() for _ in calls]
    for i in range(20):
        for (_, call), s in zip(calls, streams[i % 2:] + streams[:i % 2]):
            assert not call(s)
        op.device_synchronize()                  # a call writes its results on another stream next
    op.device_synchronize()
    for (out, _), w in zip(calls, want):
        for a, b in zip(out, w):
            assert np.array_equal(a.asnumpy(), b)
    for s in streams:
        op.destroy_cudaStream(s)


@pytest.mark.parametrize("kind", [SEVERAL[0], SEVERAL[1], SEVERAL[4]], ids=["shared", "documents", "cap"])
def test_replays_of_a_captured_step_on_tokens_near_and_apart(env, kind):
    """Which way a tile goes is found in the data, so a replay goes another way than the capture did."""
    import ctypes

    import torch
    c = Case(**kind)
    h, graph, side = Held(env, c), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    cell = ctypes.pointer(ctypes.c_void_p(side.cuda_stream))
    with torch.cuda.graph(graph, stream=side):
        h.step(cell)
    rng = np.random.RandomState(2)
    for apart in (False, True, False, True):
        for a in (*h.arrays, h.dout):
            values = rng.randn(*a.shape).astype(np.float32)
            if apart:
                values *= (2.0 ** rng.randint(-12, 1, (len(values), 1))).astype(np.float32)
                values[5] *= np.float32(2.0 ** 10)
            a[:] = values
        h.spoil()
        graph.replay()
        torch.cuda.synchronize()
        got = h.results()
        h.spoil()
        h.step(env.stream)
        env.gpu_op.device_synchronize()
        for g, w in zip(got, h.results()):
            assert np.isfinite(g).all() and np.array_equal(g, w)
