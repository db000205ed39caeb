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
        if isinstance(documents, str) and documents == "packed":
            documents = np.floor(np.arange(batch * keys) / max(1, keys // 3)).astype(np.float32)
            documents.reshape(batch, keys)[:, keys - keys // 10:] = -1
        elif isinstance(documents, str):
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
        big_q, big_k, big_v, big_do = (float(np.abs(a).max()) if a.size else 0.0 for a in (q, k, v, do))
        tiny = D * 2.0 ** -39
        for _, h, kv, rows, cols, p, inner, z, _, _ in ops.attention_parts(q, k, **self.formula()):
            m, t = slice(h * D, (h + 1) * D), slice(kv * D, (kv + 1) * D)
            Q, K, V, dO = q[rows, m], k[cols, t], v[cols, t], do[rows, m]
            s = abs(float(self.scale))               # every use of it is in a magnitude
            mag = s * np.abs(Q) @ np.abs(K).T
            ez = (D + 16) * U * mag + s * tiny * big_q * big_k + (8 * U * cap if cap else 0) + 6 * U * (np.abs(np.where(np.isfinite(z), z, 0)) + mag)
            ep = np.log(2) * np.log2(np.e) * ez + 12 * U + chain_k
            ep = ep + (p * ep).sum(1, keepdims=True)
            e_out[rows, m] = (p * ep) @ np.abs(V) + chain_k * p @ np.abs(V) + tiny * big_v
            dp = dO @ V.T
            edp = (D + 16) * U * np.abs(dO) @ np.abs(V).T + tiny * big_do * big_v
            delta = (dO * out[rows, m]).sum(1, keepdims=True)
            edelta = (np.abs(dO) * e_out[rows, m]).sum(1, keepdims=True) + (D + 2) * U * (np.abs(dO) * np.abs(out[rows, m])).sum(1, keepdims=True)
            ds = s * inner * p * (dp - delta)
            # derivative of the cap: 1 - t^2, t off by the score's error over the cap and the tanh's own 8 u
            einner = 2 * (ez / cap + 10 * U) if cap else 0.0
            eds = s * p * (inner * (ep * np.abs(dp - delta) + edp + edelta + 4 * U * (np.abs(dp) + np.abs(delta))) + einner * np.abs(dp - delta))
            # halves of ds are scaled by a bound of the row or tile: what is below 2^-18 of it loses more
            low = 2.0 ** -36 * s * (np.abs(dO).sum() / max(1, len(dO)) + np.linalg.norm(dO, axis=1).max() * np.linalg.norm(V, axis=1).max() if V.size else 0.0)
            e_dq[rows, m] = eds @ np.abs(K) + chain_k * np.abs(ds) @ np.abs(K) + low * np.abs(K).sum(0) + tiny * np.abs(ds).sum(1, keepdims=True) * big_k
            e_dk[cols, t] += eds.T @ np.abs(Q) + chain_q * np.abs(ds).T @ np.abs(Q) + low * np.abs(Q).sum(0) + tiny * np.abs(ds).sum(0)[:, None] * big_q
            e_dv[cols, t] += (p * ep).T @ np.abs(dO) + chain_q * p.T @ np.abs(dO) + tiny * p.sum(0)[:, None] * big_do + 2.0 ** -36 * np.abs(dO).sum(0)
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


@pytest.mark.parametrize("kind", [LARGE[3], LARGE[6], SMALL[4], SMALL[9]], ids=IDS)
@pytest.mark.parametrize("misaligned", [1, 2, 3])
def test_arrays_off_their_boundaries(env, path, kind, misaligned):
    check(env, Case(**kind), misaligned=misaligned)


@pytest.mark.parametrize("kind", [LARGE[2], LARGE[3], LARGE[7], SMALL[5], SMALL[11], FEW[1], FEW[5], dict(batch=1, queries=700, keys=700, heads=8, kv_heads=1, dim=64)], ids=IDS)
def test_the_same_bits_and_one_gradient_alone(env, kind):
    c = Case(**kind)
    whole = run(env, c)
    for a, b in zip(whole, run(env, c)):
        assert np.array_equal(a, b)
    assert np.array_equal(run(env, c, backward=False)[0], whole[0])
    for i in range(3):
        one = run(env, c, which=[j == i for j in range(3)])
        assert all((g is None) == (j != i) for j, g in enumerate(one[1:])) and np.array_equal(one[1 + i], whole[1 + i])
    none = run(env, c, which=(False,) * 3)
    assert none[1:] == (None, None, None)


@pytest.mark.parametrize("kind", [dict(batch=2, queries=5, keys=9, heads=4, kv_heads=2, dim=6, bias=True, cap=2.0), dict(batch=1, queries=130, keys=130, heads=2, kv_heads=1, dim=16, window=70, prefix=[9]),
                                  dict(batch=1, queries=200, keys=260, heads=2, kv_heads=2, dim=24, documents="packed", causal=False)], ids=IDS)
def test_gradients_against_differences(env, path, kind):
    """Central differences of sum(out * dout) in 64 bits, step 1e-5: truncation of 1e-10 times a third derivative, cancellation of 1e-11 times the loss."""
    c = Case(**kind)
    got, (_, bound) = run(env, c), c.bounds()
    rng = np.random.RandomState(0)
    a64 = [v.astype(np.float64) for v in (c.q, c.k, c.v)]
    loss = lambda q, k, v: float((ops.attention(q, k, v, **c.formula())[0] * c.dout).sum())      # noqa: E731
    for i in range(3):
        for _ in range(5):
            at = tuple(rng.randint(0, n) for n in a64[i].shape)
            sides = []
            for step in (1e-5, -1e-5):
                moved = [v.copy() for v in a64]
                moved[i][at] += step
                sides.append(loss(*moved))
            want = (sides[0] - sides[1]) / 2e-5
            assert abs(got[1 + i][at] - want) <= bound[1 + i][at] + 1e-6 * (1 + abs(want)), (i, at, got[1 + i][at], want)


def test_rows_that_see_nothing(env, path):
    """Padding, queries in front of the first key and windows behind the last: zeros, no gradient, and nothing of them in the others'."""
    for c in (Case(2, 200, 200, 4, 2, 40, documents="packed"), Case(1, 300, 100, 2, 1, 64), Case(1, 150, 150, 2, 1, 64, documents=np.full(150, -1, np.float32))):
        out, dq, dk, dv = check(env, c)
        want = ops.attention(*(np.asarray(a, np.float64) for a in (c.q, c.k, c.v)), **c.formula())
        empty = (want[1][..., 1] == 0)                      # batch, heads, queries
        assert empty.any()
        for got in (out, dq):
            rows = got.reshape(c.batch, c.queries, c.heads, c.dim).transpose(0, 2, 1, 3)
            assert not rows[empty].any()


@pytest.mark.parametrize("where", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("kind", [dict(batch=2, queries=70, keys=70, heads=4, kv_heads=2, dim=24, window=9), dict(batch=2, queries=300, keys=300, heads=4, kv_heads=2, dim=64, window=40)], ids=IDS)
def test_what_is_not_finite_reaches_what_depends_on_it_and_nothing_else(env, path, kind, where, bad):
    c = Case(**kind)
    clean = run(env, c)
    token, head = kind["queries"] + 30, 1                    # of the second sequence
    array = getattr(c, where)
    array[token, head * c.dim + 3] = bad
    got = run(env, c)
    first, W = kind["queries"], kind["window"]
    key_heads = [1] if where in "kv" else [head // 2]
    heads = [2, 3] if where in "kv" else [head]
    rows = list(range(token, token + W)) if where in "kv" else [token]              # queries that depend on it
    keys = sorted({j for i in rows for j in range(max(first, i - W + 1), i + 1)})
    view = lambda a, n: a.reshape(len(a), n, c.dim)         # noqa: E731
    for name, g, w, heads_of, n, touched in (("out", got[0], clean[0], heads, c.heads, rows if where != "dout" else []), ("dq", got[1], clean[1], heads, c.heads, rows),
                                             ("dk", got[2], clean[2], key_heads, c.kv_heads, keys), ("dv", got[3], clean[3], key_heads, c.kv_heads, keys)):
        g, w = view(g, n).copy(), view(w, n)
        for h in heads_of:
            for t in touched:
                if name in ("out", "dq"):
                    assert not np.isfinite(g[t, h]).all(), (name, t, h)
                g[t, h] = w[t, h]
        assert np.array_equal(g, w), name


@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("where", ["q", "k", "v"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_is_not_finite_reaches_the_answers_that_depend_on_it(env, where, bad, cap):
    """A score of minus infinity has no weight, and a cap makes it finite: the answer is not finite all the same."""
    c = Case(2, 2, 90, 4, 2, 24, window=60, cap=cap)
    clean, = run(env, c, backward=False)
    array = getattr(c, where)
    token, head = (3, 1) if where == "q" else (90 + 29, 1)   # of the second sequence: its last query; a key that its first query sees and its last does not
    array[token, head * c.dim + 3] = bad
    got, = run(env, c, backward=False)
    touched = [(3, 1)] if where == "q" else [(2, 2), (2, 3)]
    got, clean = got.reshape(4, 4, c.dim), clean.reshape(4, 4, c.dim)
    for at in touched:
        assert not np.isfinite(got[at]).all(), at
        got[at] = clean[at]
    assert np.array_equal(got, clean)


@pytest.mark.parametrize("queries, path", [(2, 1), (17, 1), (17, 2)])
def test_more_sequences_than_a_grid_has_rows(env, queries, path):
    c = Case(70001, queries, queries, 1, 1, 4)
    env.gpu_op.set_contraction_path(path)
    got = run(env, c)
    env.gpu_op.set_contraction_path(0)
    some = [0, 65534, 65535, 65536, 70000]
    few = Case(len(some), queries, queries, 1, 1, 4)
    take = lambda a: a.reshape(c.batch, queries, 4)[some].reshape(-1, 4)      # noqa: E731
    few.q, few.k, few.v, few.dout = (take(a) for a in (c.q, c.k, c.v, c.dout))
    want, bound = few.bounds()
    for name, g, w, e in zip(("out", "dq", "dk", "dv"), got, want, bound):
        within(take(g), w, e, name)


def test_unseen_keys_may_hold_anything(env, path):
    """Keys behind the last query's sight, of other documents and padding: NaN there changes no bit of the exact kernels' results.  On the tensor path a finite value there has
    a part in its tile's scale, a power of two, and NaN has none: values that were representable in 22 bits below 2^14 are so below 2^15, and the roundings are others of the same
    bounds."""
    c = Case(2, 180, 180, 4, 2, 64, documents="packed")
    clean = run(env, c)
    want, bound = c.bounds()
    padding = np.flatnonzero(c.documents < 0)
    for array in (c.k, c.v):
        array[padding] = np.nan
    for name, g, w, exact, e in zip(("out", "dq", "dk", "dv"), run(env, c), clean, want, bound):
        if path == "exact":
            assert np.array_equal(g, w), name
        within(g, exact, e, name)
    c = Case(1, 3, 400, 4, 2, 64, window=20)
    clean = run(env, c, backward=False)[0]
    c.k[:200] = np.inf
    c.v[:370] = np.nan
    assert np.array_equal(run(env, c, backward=False)[0], clean)


def test_values_of_every_size(env, path):
    """Each tile has scales of its own: tokens 2^60 apart, zeros, and scores beyond what an exponential takes."""
    c = Case(1, 400, 400, 2, 1, 64, spread=1.0)
    for array, size in ((c.v, 2.0 ** 40), (c.dout, 2.0 ** -50)):
        array *= np.float32(size)
    c.q[:128] *= np.float32(2.0 ** -30)
    c.q[128:256] = 0
    c.k[256:] *= np.float32(2.0 ** 20)
    c.q[256:] *= np.float32(2.0 ** -20)
    check(env, c)
    c = Case(1, 300, 300, 2, 2, 32, spread=40.0)               # one key takes all
    got = run(env, c)
    want, bound = c.bounds()
    within(got[0], want[0], bound[0], "out")
    assert all(np.isfinite(g).all() for g in got)
    c = Case(1, 200, 200, 2, 1, 32, spread=1e18, scale=1e-20)
    assert all(np.isfinite(g).all() for g in run(env, c))


def test_a_negative_scale_and_positive_biases(env, path):
    c = Case(2, 190, 190, 4, 2, 48, scale=-0.2, bias=True)
    c.slopes *= -0.3
    check(env, c)
    check(env, Case(1, 260, 260, 2, 2, 64, scale=-0.125))
    check(env, Case(1, 150, 150, 2, 2, 64, scale=0.0))


@pytest.mark.parametrize("kind", [SMALL[4], LARGE[3], LARGE[7], FEW[1]], ids=IDS)
def test_a_captured_pass_replayed_on_other_data(env, kind):
    import torch
    nd, op = env.nd, env.gpu_op
    c = Case(**kind)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    cell = ctypes.pointer(ctypes.c_void_p(side.cuda_stream))
    on = lambda v: None if v is None else nd.array(v, env.ctx)       # noqa: E731
    q, k, v, docs, prefix, slopes, dout = (on(a) for a in (c.q, c.k, c.v, c.documents, c.prefix, c.slopes, c.dout))
    out, stats = nd.empty(c.q.shape, env.ctx), nd.empty((c.batch, c.heads, c.queries, 2), env.ctx)
    grads = [nd.empty(a.shape, env.ctx) for a in (c.q, c.k, c.v)]
    state = c.state(env)

    def work(stream):
        assert not op.attention_forward(q, k, v, docs, prefix, slopes, out, stats, state, stream)
        assert not op.attention_backward(q, k, v, docs, prefix, slopes, out, stats, dout, *grads, state, stream)

    with torch.cuda.graph(graph, stream=side):                  # the first use of the stream
        work(cell)
    rng = np.random.RandomState(5)
    for size in (1.0, 1e3, 1e-4):
        for a in (q, k, v, dout):
            a[:] = (size * rng.randn(*a.shape)).astype(np.float32)
        for a in (out, stats, *grads):
            a[:] = np.full(a.shape, np.nan, np.float32)
        graph.replay()
        torch.cuda.synchronize()
        got = [a.asnumpy() for a in (out, stats, *grads)]
        work(env.stream)
        op.device_synchronize()
        for g, a in zip(got, (out, stats, *grads)):
            assert np.isfinite(g).all()
            assert np.array_equal(g, a.asnumpy())


def test_two_streams_at_once(env):
    """Each stream has scratch of its own."""
    cases = [Case(2, 500, 500, 4, 2, 64, seed=1), Case(1, 700, 700, 4, 4, 128, seed=2), Case(3, 1, 2000, 8, 2, 64, seed=3)]
    want = [run(env, c, backward=i < 2) for i, c in enumerate(cases)]
    streams = [env.gpu_op.create_cudaStream() for _ in cases]
    held = []
    for c, s in zip(cases, streams):
        on = [env.nd.array(a, env.ctx) for a in (c.q, c.k, c.v)]
        out, stats = env.nd.empty(c.q.shape, env.ctx), env.nd.empty((c.batch, c.heads, c.queries, 2), env.ctx)
        held.append((on, out, stats, c.state(env)))
    for _ in range(20):
        for (on, out, stats, state), s in zip(held, streams):
            env.gpu_op.attention_forward(*on, None, None, None, out, stats, state, s)
    env.gpu_op.device_synchronize()
    for (on, out, stats, state), w in zip(held, want):
        assert np.array_equal(out.asnumpy(), w[0])
    for s in streams:
        env.gpu_op.destroy_cudaStream(s)


def test_no_sequences_and_no_keys(env, path):
    nd, op = env.nd, env.gpu_op
    E, F = nd.empty((0, 16), env.ctx), nd.empty((0, 16), env.ctx)
    state = op.attention_state(4, 2, 2)
    assert not op.attention_forward(E, E, E, None, None, None, F, None, state, env.stream)
    if path == "tensor":
        return
    q, out, stats = nd.array(np.ones((8, 16), np.float32), env.ctx), nd.array(np.ones((8, 16), np.float32), env.ctx), nd.empty((2, 2, 4, 2), env.ctx)
    assert not op.attention_forward(q, E, E, None, None, None, out, stats, state, env.stream)
    assert not out.asnumpy().any() and not stats.asnumpy().any()
    dq, dk, dv = nd.array(np.ones((8, 16), np.float32), env.ctx), nd.empty((0, 16), env.ctx), nd.empty((0, 16), env.ctx)
    assert not op.attention_backward(q, E, E, None, None, None, out, stats, q, dq, dk, dv, state, env.stream)
    assert not dq.asnumpy().any()


def test_shortage_of_memory_is_reported(env):
    nd, op = env.nd, env.gpu_op
    q = nd.array(np.ones((4096, 64), np.float32), env.ctx)
    out, state = nd.empty((4096, 64), env.ctx), op.attention_state(4096, 1, 1)
    stream = op.create_cudaStream()
    op.release_cached_memory()
    op.set_memory_limit(1 << 20)               # less than the arrays hold: what other streams' scratch gives back does not help
    try:
        short = op.attention_forward(q, q, q, None, None, None, out, None, state, stream)
    finally:
        op.set_memory_limit(0)
    assert short > 0
    assert not op.attention_forward(q, q, q, None, None, None, out, None, state, stream)
    op.device_synchronize()
    op.destroy_cudaStream(stream)


def test_the_same_array_for_all_three(env, path):
    """Queries, keys and values may be one array."""
    c = Case(1, 200, 200, 2, 2, 64)
    c.k = c.v = c.q
    x = place(env, c.q)
    out, stats = place(env, c.q.shape), place(env, (1, 2, 200, 2))
    assert not env.gpu_op.attention_forward(x, x, x, None, None, None, out, stats, c.state(env), env.stream)
    env.gpu_op.device_synchronize()
    within(read(out), c.bounds()[0][0], c.bounds()[1][0], "out")


def test_elements_beyond_32_bits(env):
    """The last sequence of keys and values of 2^31 + elements, answered by one query each; what lies in front is a dropout of ones."""
    nd, op = env.nd, env.gpu_op
    D, G, keys = 128, 8, 4096
    batch = (1 << 31) // (D * G * keys) + 1
    K = nd.empty((batch * keys, G * D), env.ctx)
    V = nd.empty((batch * keys, G * D), env.ctx)
    if isinstance(K, int) or isinstance(V, int):
        pytest.skip("not enough device memory")
    op.array_set(V, 1.0, env.stream)
    op.dropout_forward(V, K, "NCHW", 0.5, 3, op.get_input_descriptor(K.shape, "NCHW"), env.cudnn, env.stream)
    from tests.test_gpu_norm import view
    rng = np.random.RandomState(0)
    last = {}
    for name, whole in (("k", K), ("v", V)):
        tail = view(env, whole, (batch - 1) * keys * G * D, (keys, G * D))
        last[name] = rng.randn(keys, G * D).astype(np.float32)
        tail[:] = last[name]
    q = np.concatenate([np.ones((batch - 1, G * D)), rng.randn(1, G * D)]).astype(np.float32)
    Q, out = nd.array(q, env.ctx), nd.empty(q.shape, env.ctx)
    assert not op.attention_forward(Q, K, V, None, None, None, out, None, op.attention_state(1, G, G, True, 0, D ** -0.5), env.stream)
    got = out.asnumpy()
    c = Case(1, 1, keys, G, G, D)
    c.q, c.k, c.v, c.dout = q[-1:], last["k"], last["v"], q[-1:]
    want, bound = c.bounds()
    within(got[-1:], want[0], bound[0], "out")
    np.testing.assert_allclose(got[:-1], 1.0, rtol=1e-5)
    del K, V
    op.release_cached_memory()
