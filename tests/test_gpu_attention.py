"""Attention and its gradients against the formulas in 64 bits.

Tolerances bound roundings, u = 2^-24 a step.  With M_ij = scale sum_d |q_id k_jd|:
* a product of D terms is off by at most (D + 16) u M: one rounding a term (exact kernels); on the tensor path the halves of a value leave
  2^-23 of it, what is dropped 2^-23 of a product, and of 3 D / 16 accumulations each truncates 2 u of the sum: (4 + 3 D / 8) u M, and values below
  2^-18 of a tensor's largest lose more: 2^-39 of that, D such terms;
* the score behind it by 6 u more for scale, cap, bias and the change of base (the tanh of the tensor path: 8 u of the cap, its values being formed
  from an exponential and a reciprocal of 2 ulp each and rounded below 1);
* a probability relative to itself by log 2 times the score's error, its row's mean of that, and 12 u: exponential, sum of T keys (64 in a row at
  once, T / 64 tiles after one another), reciprocal, product;
* sums over T keys or queries by (T / 16 + 96) u of the sum of magnitudes: chains of 64 in a tile, and the tiles.
Errors of the probabilities go into the sums as magnitudes, so the bounds are far from sharp; what they catch is a wrong formula, mask or index."""
import ctypes

import numpy as np
import pytest

from oracle import ops
from tests.test_gpu_norm import place, read, within
from tests.test_gpu_ops import env  # noqa: F401

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


class Case:
    def __init__(self, batch, queries, keys, heads, kv_heads, dim, causal=True, window=0, cap=0.0, bias=False, documents=None, prefix=None, seed=0, scale=None, spread=1.0):
        rng = np.random.RandomState(seed + 7 * queries + keys + dim)
        f = lambda *s: rng.randn(*s).astype(np.float32)      # noqa: E731
        self.q, self.k, self.v = spread * f(batch * queries, heads * dim), f(batch * keys, kv_heads * dim), f(batch * keys, kv_heads * dim)
        self.dout = f(batch * queries, heads * dim)
        if documents == "packed":
            documents = np.floor(np.arange(batch * keys) / max(1, keys // 3)).astype(np.float32)
            documents.reshape(batch, keys)[:, keys - keys // 10:] = -1
        elif documents == "mixed":
            documents = rng.randint(-1, 3, batch * keys).astype(np.float32)
        if prefix is not None:
            prefix = np.asarray(prefix, np.float32) * np.ones(batch, np.float32)
        self.documents, self.prefix = documents, prefix
        self.slopes = (2.0 ** -np.arange(1, heads + 1)).astype(np.float32) if bias else None
        self.batch, self.queries, self.keys, self.heads, self.kv_heads, self.dim = batch, queries, keys, heads, kv_heads, dim
        self.causal, self.window, self.cap = causal, window, cap
        self.scale = np.float32(dim ** -0.5 if scale is None else scale)

    def formula(self):
        return dict(length=self.queries, heads=self.heads, kv_heads=self.kv_heads, causal=self.causal, window=self.window, scale=np.float64(self.scale),
                    cap=np.float64(np.float32(self.cap)), documents=self.documents, prefix=self.prefix, slopes=self.slopes)

    def bounds(self):
        """((out, dq, dk, dv), their bounds)"""
        q, k, v, do = (np.asarray(a, np.float64) for a in (self.q, self.k, self.v, self.dout))
        out, _ = ops.attention(q, k, v, **self.formula())
        dq, dk, dv = ops.attention_backward(q, k, v, do, **self.formula())
        D, cap, chain_k, chain_q = self.dim, self.cap, (self.keys / 16 + 96) * U, (self.queries * self.heads / self.kv_heads / 16 + 96) * U
        e_out, e_dq, e_dk, e_dv = (np.zeros_like(a) for a in (out, dq, dk, dv))
        big = lambda a: float(np.abs(a).max()) if a.size else 0.0       # noqa: E731
        tiny = D * 2.0 ** -39
        for _, h, kv, rows, cols, p, inner, z, _, _ in ops.attention_parts(q, k, **self.formula()):
            m, t = slice(h * D, (h + 1) * D), slice(kv * D, (kv + 1) * D)
            Q, K, V, dO = q[rows, m], k[cols, t], v[cols, t], do[rows, m]
            s = float(self.scale)
            mag = s * np.abs(Q) @ np.abs(K).T
            ez = (D + 16) * U * mag + s * tiny * big(q) * big(k) + (8 * U * cap if cap else 0) + 6 * U * (np.abs(np.where(np.isfinite(z), z, 0)) + mag)
            ep = np.log(2) * np.log2(np.e) * ez + 12 * U + chain_k
            ep = ep + (p * ep).sum(1, keepdims=True)
            e_out[rows, m] = (p * ep) @ np.abs(V) + chain_k * p @ np.abs(V) + tiny * big(v)
            dp = dO @ V.T
            edp = (D + 16) * U * np.abs(dO) @ np.abs(V).T + tiny * big(do) * big(v)
            delta = (dO * out[rows, m]).sum(1, keepdims=True)
            edelta = (np.abs(dO) * e_out[rows, m]).sum(1, keepdims=True) + (D + 2) * U * (np.abs(dO) * np.abs(out[rows, m])).sum(1, keepdims=True)
            ds = s * inner * p * (dp - delta)
            # derivative of the cap: 1 - t^2, t off by the score's error over the cap and the tanh's own 8 u
            einner = 2 * (ez / cap + 10 * U) if cap else 0.0
            eds = s * p * (inner * (ep * np.abs(dp - delta) + edp + edelta + 4 * U * (np.abs(dp) + np.abs(delta))) + einner * np.abs(dp - delta))
            # halves of ds are scaled by a bound of the row or tile: what is below 2^-18 of it loses more
            low = 2.0 ** -36 * s * (np.abs(dO).sum() / max(1, len(dO)) + np.linalg.norm(dO, axis=1).max() * np.linalg.norm(V, axis=1).max() if V.size else 0.0)
            e_dq[rows, m] = eds @ np.abs(K) + chain_k * np.abs(ds) @ np.abs(K) + low * np.abs(K).sum(0) + tiny * np.abs(ds).sum(1, keepdims=True) * big(k)
            e_dk[cols, t] += eds.T @ np.abs(Q) + chain_q * np.abs(ds).T @ np.abs(Q) + low * np.abs(Q).sum(0) + tiny * np.abs(ds).sum(0)[:, None] * big(q)
            e_dv[cols, t] += (p * ep).T @ np.abs(dO) + chain_q * p.T @ np.abs(dO) + tiny * p.sum(0)[:, None] * big(do) + 2.0 ** -36 * np.abs(dO).sum(0)
        return (out, dq, dk, dv), tuple(e + 1e-30 for e in (e_out, e_dq, e_dk, e_dv))

    def state(self, env):
        return env.gpu_op.attention_state(self.queries, self.heads, self.kv_heads, self.causal, self.window, float(self.scale), self.cap)


def run(env, c, misaligned=0, backward=True, stream=None, which=(True, True, True)):
    """(out, dq, dk, dv) of the library; arrays have NaN around them, which nothing reads into a result or overwrites."""
    on = lambda v: None if v is None else place(env, v, misaligned)       # noqa: E731
    q, k, v, docs, prefix, slopes, dout = (on(a) for a in (c.q, c.k, c.v, c.documents, c.prefix, c.slopes, c.dout))
    out, stats = place(env, c.q.shape, misaligned), place(env, (c.batch, c.heads, c.queries, 2), misaligned)
    state, stream = c.state(env), stream or env.stream
    assert not env.gpu_op.attention_forward(q, k, v, docs, prefix, slopes, out, stats if backward else None, state, stream)
    if not backward:
        env.gpu_op.device_synchronize()
        return (read(out),)
    grads = [place(env, a.shape, misaligned) if w else None for a, w in zip((c.q, c.k, c.v), which)]
    assert not env.gpu_op.attention_backward(q, k, v, docs, prefix, slopes, out, stats, dout, *grads, state, stream)
    env.gpu_op.device_synchronize()
    return (read(out),) + tuple(None if g is None else read(g) for g in grads)


def check(env, c, **more):
    got = run(env, c, **more)
    want, bound = c.bounds()
    for name, g, w, e in zip(("out", "dq", "dk", "dv"), got, want, bound):
        if g is not None:
            within(g, w, e, name)
    return got


SMALL = [
    dict(batch=1, queries=1, keys=1, heads=1, kv_heads=1, dim=1),
    dict(batch=2, queries=3, keys=3, heads=2, kv_heads=1, dim=5),
    dict(batch=3, queries=17, keys=17, heads=4, kv_heads=2, dim=16, causal=False),
    dict(batch=2, queries=64, keys=64, heads=4, kv_heads=4, dim=64),
    dict(batch=1, queries=65, keys=129, heads=6, kv_heads=2, dim=72, bias=True),
    dict(batch=2, queries=40, keys=40, heads=3, kv_heads=3, dim=33, window=7),
    dict(batch=2, queries=40, keys=70, heads=3, kv_heads=1, dim=24, causal=False, window=9, cap=5.0),
    dict(batch=3, queries=50, keys=50, heads=2, kv_heads=1, dim=40, prefix=[0, 13.5, 90]),
    dict(batch=2, queries=45, keys=60, heads=2, kv_heads=2, dim=128, documents="packed", cap=3.0, bias=True),
    dict(batch=2, queries=61, keys=61, heads=4, kv_heads=1, dim=20, documents="mixed", causal=False, prefix=[5, 200]),
    dict(batch=1, queries=33, keys=20, heads=2, kv_heads=1, dim=64),
    dict(batch=1, queries=20, keys=75, heads=2, kv_heads=2, dim=200, window=30, prefix=[3]),
    dict(batch=1, queries=7, keys=300, heads=8, kv_heads=2, dim=256, bias=True),
]


LARGE = [
    dict(batch=1, queries=128, keys=128, heads=1, kv_heads=1, dim=64, causal=False),
    dict(batch=1, queries=128, keys=384, heads=1, kv_heads=1, dim=128),
    dict(batch=2, queries=256, keys=256, heads=4, kv_heads=2, dim=64),
    dict(batch=1, queries=300, keys=300, heads=6, kv_heads=2, dim=72, prefix=[100], bias=True),
    dict(batch=2, queries=333, keys=500, heads=2, kv_heads=1, dim=80, window=150, cap=4.0),
    dict(batch=2, queries=401, keys=401, heads=3, kv_heads=3, dim=33, causal=False, window=65, cap=20.0, bias=True),
    dict(batch=2, queries=517, keys=517, heads=2, kv_heads=2, dim=128, documents="packed"),
    dict(batch=2, queries=260, keys=517, heads=4, kv_heads=1, dim=16, documents="mixed", prefix=[30, 600], cap=2.0),
    dict(batch=1, queries=700, keys=130, heads=2, kv_heads=1, dim=96),
    dict(batch=1, queries=1025, keys=1025, heads=1, kv_heads=1, dim=128, bias=True, cap=30.0),
]
FEW = [
    dict(batch=3, queries=1, keys=1, heads=4, kv_heads=2, dim=64),
    dict(batch=2, queries=1, keys=1000, heads=8, kv_heads=2, dim=128),
    dict(batch=1, queries=1, keys=4097, heads=8, kv_heads=1, dim=64, bias=True, cap=30.0),
    dict(batch=9, queries=1, keys=130, heads=24, kv_heads=12, dim=72, window=50),
    dict(batch=2, queries=3, keys=700, heads=4, kv_heads=2, dim=33, causal=False, window=100, prefix=[0, 20]),
    dict(batch=2, queries=5, keys=611, heads=3, kv_heads=1, dim=80, documents="mixed"),
    dict(batch=2, queries=2, keys=900, heads=2, kv_heads=2, dim=256, prefix=[40, 1000], cap=5.0),
    dict(batch=1, queries=4, keys=3, heads=2, kv_heads=1, dim=16),
    dict(batch=40, queries=1, keys=65, heads=16, kv_heads=16, dim=128),
]
IDS = lambda k: "-".join("%s%s" % (n[0], v) for n, v in k.items())      # noqa: E731


@pytest.mark.parametrize("kind", FEW, ids=IDS)
@pytest.mark.parametrize("misaligned", [0, 1])
def test_few_queries(env, kind, misaligned):
    """The forward call of few queries; the backward call takes its statistics."""
    c = Case(**kind)
    check(env, c, misaligned=misaligned)


@pytest.fixture(params=["exact", "tensor"])
def path(request, env):
    env.gpu_op.set_contraction_path({"exact": 1, "tensor": 2}[request.param])
    yield request.param
    env.gpu_op.set_contraction_path(0)


@pytest.mark.parametrize("kind", SMALL + LARGE, ids=IDS)
def test_formula(env, path, kind):
    if path == "tensor" and kind["dim"] > 128:
        pytest.skip("heads of up to 128 elements")
    check(env, Case(**kind))
    assert env.gpu_op.tensor_path_error() == 0
    assert env.gpu_op.last_contraction_path() == {"exact": 1, "tensor": 2}[path]
