"""Attention of values that differ in size from token to token, or are not finite, against the formulas in 64 bits.

Tolerances as in test_gpu_attention.py, but what is lost of small values is counted by token, not by the whole array: no value of one token may cost bits of another's that
does not depend on it.  On the tensor path a tile of 128 tokens shares a scale only where their largest magnitudes are near each other:
* queries, keys, values: the arrays here are within 16 of each other, or so far apart that every token has a scale of its own: an element is off by 2^-39 of 16 times
  its token's largest, twice for both operands of a product: 2^-34;
* output gradients over their row's sum: within 2^15: 2^-23;
* weights are off by 2^-38 of what scales them: 1 for the probabilities, for the gradients the norm of the row's output gradient times sqrt(D) times the largest value near it
  (dq), and up to 1024 times that of any query that the key sees (dk)."""
import numpy as np
import pytest

from oracle import ops
from tests.test_gpu_attention import IDS, U, Case, env, path, run  # noqa: F401
from tests.test_gpu_norm import within

pytestmark = pytest.mark.gpu


class Fine(Case):
    def bounds(self):
        q, k, v, do = (np.asarray(a, np.float64) for a in (self.q, self.k, self.v, self.dout))
        want = (ops.attention(q, k, v, **self.formula())[0],) + ops.attention_backward(q, k, v, do, **self.formula())
        D, cap, chain_k, chain_q = self.dim, self.cap, (self.keys / 16 + 96) * U, (self.queries * self.heads / self.kv_heads / 16 + 96) * U
        e_out, e_dq, e_dk, e_dv = (np.zeros_like(a) for a in want)
        near, s = 2.0 ** -34, abs(float(self.scale))
        for _, h, kv, rows, cols, p, inner, z, _, inv in ops.attention_parts(q, k, **self.formula()):
            m, t = slice(h * D, (h + 1) * D), slice(kv * D, (kv + 1) * D)
            Q, K, V, dO, inv = q[rows, m], k[cols, t], v[cols, t], do[rows, m], inv[:, None]
            seen = np.isfinite(z)
            qm, km, vm, dm = (np.abs(a).max(1) for a in (Q, K, V, dO))
            mag = s * np.abs(Q) @ np.abs(K).T
            ez = (D + 16) * U * mag + s * D * near * np.outer(qm, km) + (8 * U * cap if cap else 0) + 6 * U * (np.abs(np.where(seen, z, 0)) + mag)
            ep = ez + 12 * U + chain_k
            ep = ep + (p * ep).sum(1, keepdims=True)
            e_out[rows, m] = (p * ep) @ np.abs(V) + chain_k * p @ np.abs(V) + 2.0 ** -32 * (p @ vm)[:, None] + 2.0 ** -38 * inv * (seen @ np.abs(V))
            dp = dO @ V.T
            edp = (D + 16) * U * np.abs(dO) @ np.abs(V).T + D * 2.0 ** -23 * np.outer(dm, vm)
            delta = (dO * want[0][rows, m]).sum(1, keepdims=True)
            edelta = (np.abs(dO) * e_out[rows, m]).sum(1, keepdims=True) + (D + 2) * U * (np.abs(dO) * np.abs(want[0][rows, m])).sum(1, keepdims=True)
            ds = s * inner * p * (dp - delta)
            einner = 2 * (ez / cap + 10 * U) if cap else 0.0
            eds = s * p * (inner * (ep * np.abs(dp - delta) + edp + edelta + 4 * U * (np.abs(dp) + np.abs(delta))) + einner * np.abs(dp - delta))
            weight = s * 2.0 ** -38 * inv * seen * (16 * D ** 0.5 * np.outer(np.linalg.norm(dO, axis=1), vm) + np.abs(delta))
            e_dq[rows, m] = eds @ np.abs(K) + chain_k * np.abs(ds) @ np.abs(K) + weight @ np.abs(K) + 2.0 ** -32 * (np.abs(ds) @ km)[:, None]
            e_dk[cols, t] += eds.T @ np.abs(Q) + chain_q * np.abs(ds).T @ np.abs(Q) + 1024 * weight.T @ np.abs(Q) + 2.0 ** -32 * (np.abs(ds).T @ qm)[:, None]
            e_dv[cols, t] += (p * ep).T @ np.abs(dO) + chain_q * p.T @ np.abs(dO) + 2.0 ** -23 * (p.T @ dm)[:, None] + 2.0 ** -38 * (inv * seen).T @ np.abs(dO)
        return want, tuple(e + 1e-35 for e in (e_out, e_dq, e_dk, e_dv))


def check(got, want, bound, names=("out", "dq", "dk", "dv")):
    for name, g, w, e in zip(names, got, want, bound):
        assert np.isfinite(g).all(), name
        within(g, w, e, name)


# ---- what is not finite -----------------------------------------------------------------------------
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("kind", [dict(queries=40, dim=24), dict(queries=150, dim=64), dict(queries=24, dim=200)], ids=lambda k: "%(queries)d-%(dim)d" % k)
@pytest.mark.parametrize("first", [True, False])
def test_a_query_that_is_not_finite_has_no_answer(env, path, kind, bad, cap, first):
    """The first of its sequence, which sees one key, and one that sees several: the answer and the query's gradient are not finite, nor are the gradients of the keys that it sees,
    and everything else keeps its bits.  A score of minus infinity alone would have no weight, and a cap would make it finite."""
    if path == "tensor" and kind["dim"] > 128:
        pytest.skip("heads of up to 128 elements")
    c = Case(2, kind["queries"], kind["queries"], 4, 2, kind["dim"], window=6, cap=cap)
    clean = run(env, c)
    start = kind["queries"]
    token, head = start if first else start + 20, 1
    c.q[token, head * c.dim + 3] = bad
    got = run(env, c)
    keys = range(max(start, token - 5), token + 1)
    for name, g, w, n, touched in (("out", got[0], clean[0], 4, [(token, 1)]), ("dq", got[1], clean[1], 4, [(token, 1)]), ("dk", got[2], clean[2], 2, [(j, 0) for j in keys]),
                                   ("dv", got[3], clean[3], 2, [(j, 0) for j in keys])):
        g, w = g.reshape(len(g), n, c.dim).copy(), w.reshape(len(w), n, c.dim)
        for at in touched:
            assert not np.isfinite(g[at]).any() if name in ("out", "dq") else not np.isfinite(g[at]).all(), (name, at)
            g[at] = w[at]
        assert np.array_equal(g, w), name


@pytest.mark.parametrize("kind", [dict(queries=300, keys=300, heads=4, kv_heads=2, dim=64), dict(queries=260, keys=260, heads=2, kv_heads=2, dim=128, cap=5.0, bias=True),
                                  dict(queries=140, keys=200, heads=2, kv_heads=1, dim=40, causal=False, documents="packed")], ids=IDS)
def test_gradients_scale_with_the_output_gradient_bit_by_bit(env, path, kind):
    """A power of two times the output gradient is that times every gradient."""
    c = Case(2, **kind)
    whole = run(env, c)
    for size in (2.0 ** -3, 2.0 ** -20, 2.0 ** 10):
        scaled = Case(2, **kind)
        scaled.dout *= np.float32(size)
        for name, g, w in zip(("out", "dq", "dk", "dv"), run(env, scaled), whole):
            assert np.array_equal(g, w * np.float32(1 if name == "out" else size)), (name, size)


@pytest.mark.parametrize("dim", [64, 128])
def test_tokens_that_see_themselves_alone(env, path, dim):
    """Documents of one token: a probability of 1, so the value's gradient is the output gradient, but for the score's distance from itself.  That is z - max, where max is z rounded: half a step
    of |z| + 1, log 2 of it a change of the weight; 2 u each for the exponential, the reciprocal and their product; 2^-22 for both operands' halves and what their product drops, and
    2 u for each of three products' accumulations; 2^-32 of the largest value for those far below it."""
    c = Case(1, 512, 512, 2, 2, dim, documents=np.arange(512).astype(np.float32), seed=9)
    out, dq, dk, dv = run(env, c)
    z = np.abs((np.asarray(c.q, np.float64) * c.k).reshape(512, 2, dim).sum(-1)) * float(c.scale) * np.log2(np.e)
    allowed = np.repeat(U * (np.log(2) * (z + 1) + 6 + 4 + 6), dim, axis=1)
    within(dv, np.asarray(c.dout, np.float64), allowed * np.abs(c.dout) + 2.0 ** -32 * np.abs(c.dout).max(), "dv")
    within(out, np.asarray(c.v, np.float64), allowed * np.abs(c.v) + 2.0 ** -32 * np.abs(c.v).max(), "out")


@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 24, 2.0 ** 34, 2.0 ** 60, 2.0 ** 110])
@pytest.mark.parametrize("kind", [dict(queries=300, keys=300, heads=4, kv_heads=2, dim=64), dict(queries=150, keys=270, heads=2, kv_heads=1, dim=128, causal=False), dict(queries=2, keys=700, heads=4, kv_heads=2, dim=40),
                                  dict(queries=200, keys=200, heads=2, kv_heads=2, dim=48, bias=True)], ids=IDS)
def test_scores_of_any_size(env, path, kind, size):
    """Where the largest score is 150 above the next, in units of log 2, it takes all: the answer is its value, and the value's gradient the sum of the output gradients of the queries that it
    answers.  u: 2 each for exponential, sum, reciprocal and products, 4 for the halves, 6 for the accumulations, and the sum over queries (the calls of few queries form scores in an
    order of their own: their answers alone)."""
    c = Case(1, **kind)
    c.q *= np.float32(size ** 0.5)
    c.k *= np.float32(size ** 0.5)
    got = run(env, c)
    assert all(np.isfinite(g).all() for g in got)
    D, want, dv, allowed = c.dim, np.zeros(c.q.shape), np.zeros(c.v.shape), np.zeros(c.v.shape)
    clear = np.zeros((c.queries, c.heads), bool)
    for _, h, kv, rows, cols, p, _, z, _, _ in ops.attention_parts(c.q.astype(np.float64), c.k.astype(np.float64), **c.formula()):
        m, t = slice(h * D, (h + 1) * D), slice(kv * D, (kv + 1) * D)
        best = z.argmax(1)
        rest = z.copy()
        rest[np.arange(c.queries), best] = -np.inf
        noise = (D + 16) * U * float(c.scale) * np.log2(np.e) * (np.abs(c.q[:, m].astype(np.float64)) @ np.abs(c.k[:, t].astype(np.float64)).T).max(1)
        clear[:, h] = z.max(1) - rest.max(1) > 150 + 2 * noise
        want[:, m] = c.v[best, t]
    assert clear.mean() > (0.2 if size < 2.0 ** 20 else 0.9)
    of_out = np.repeat(clear, D, axis=1)
    within(got[0][of_out], want[of_out], 16 * U * np.abs(want[of_out]) + 2.0 ** -32 * np.abs(c.v).max(), "out")
    if c.queries * c.heads // c.kv_heads <= 16:
        return
    c.dout[~of_out] = 0
    got = run(env, c)
    for _, h, kv, rows, cols, p, _, z, _, _ in ops.attention_parts(c.q.astype(np.float64), c.k.astype(np.float64), **c.formula()):
        m, t = slice(h * D, (h + 1) * D), slice(kv * D, (kv + 1) * D)
        for i, j in enumerate(z.argmax(1)):
            dv[j, t] += c.dout[i, m]
            allowed[j, t] += np.abs(c.dout[i, m])
    within(got[3], dv, (16 + c.queries / 16 + 96) * U * allowed + 2.0 ** -30 * np.abs(c.dout).max(), "dv")


@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** -75, 2.0 ** -64, 2.0 ** 62, 2.0 ** 80])
@pytest.mark.parametrize("dim", [40, 128])
def test_output_gradients_whose_squares_leave_float32(env, path, dim, size):
    c = Fine(1, 400, 400, 2, 1, dim, causal=False, seed=10)
    want, bound = c.bounds()
    c.dout *= np.float32(size)
    got = run(env, c)
    check([g.astype(np.float64) / (size if i else 1) for i, g in enumerate(got)], want, bound)


@pytest.mark.parametrize("dim", [64, 128])
def test_tokens_that_see_themselves_alone_behind_a_cap(env, path, dim):
    """The same, with scores of 20 to 30 behind a cap of 30.  The score is what the answer's was, bit by bit, so its weight is 1."""
    c = Case(1, 512, 512, 2, 2, dim, documents=np.arange(512).astype(np.float32), cap=30.0, seed=9)
    c.k = (c.q * np.random.RandomState(1).uniform(3, 9, (512, 1))).astype(np.float32)
    out, dq, dk, dv = run(env, c)
    within(dv, np.asarray(c.dout, np.float64), 16 * U * np.abs(c.dout) + 2.0 ** -32 * np.abs(c.dout).max(), "dv")
    within(out, np.asarray(c.v, np.float64), 16 * U * np.abs(c.v) + 2.0 ** -32 * np.abs(c.v).max(), "out")


# ---- tokens of different sizes ---------------------------------------------------------------------
KINDS = [dict(heads=4, kv_heads=2, dim=64), dict(heads=2, kv_heads=2, dim=128, causal=False), dict(heads=3, kv_heads=1, dim=33, cap=4.0, bias=True), dict(heads=2, kv_heads=1, dim=96, causal=False, cap=20.0),
         dict(heads=1, kv_heads=1, dim=16, bias=True)]


def among_others(alone, lead, tail, seed=1):
    """Documents of `lead` and `tail` tokens around the tokens of `alone`, all of one row."""
    n, total = alone.queries, lead + alone.queries + tail
    c = Case(1, total, total, alone.heads, alone.kv_heads, alone.dim, alone.causal, cap=alone.cap, bias=alone.slopes is not None, seed=seed)
    c.documents = np.repeat([1.0, 2.0, 3.0], [lead, n, tail]).astype(np.float32)
    mine = slice(lead, lead + n)
    for name in ("q", "k", "v", "dout"):
        getattr(c, name)[mine] = getattr(alone, name)
    return c, mine, [t for t in range(total) if not lead <= t < lead + n]


@pytest.mark.parametrize("size", [2.0 ** 13, 2.0 ** 20, 2.0 ** 40, 2.0 ** 100, 2.0 ** -20])
@pytest.mark.parametrize("where", ["q", "k", "v", "all"])
@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_other_documents_of_any_size_cost_nothing(env, path, kind, where, size):
    alone = Fine(1, 140, 140, seed=3, **kind)
    want, bound = alone.bounds()
    c, mine, others = among_others(alone, 60, 75)
    clean = run(env, c)
    for name in ("q", "k", "v") if where == "all" else (where,):
        getattr(c, name)[others] *= np.float32(size ** 0.5 if where == "all" else size)
    got = run(env, c)
    check([g[mine] for g in got], want, bound)
    if path == "exact":
        for g, w in zip(got, clean):
            assert np.array_equal(g[mine], w[mine])


@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 60, 2.0 ** 120])
@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_padding_of_any_size_costs_nothing(env, path, kind, size):
    """Padding behind every sequence: no result depends on it."""
    c = Fine(2, 150, 150, documents=np.where(np.arange(300) % 150 < 141, 1.0, -1.0).astype(np.float32), seed=2, **kind)
    want, bound = c.bounds()
    padding = np.flatnonzero(c.documents < 0)
    for array in (c.q, c.k, c.v, c.dout):
        array[padding] *= np.float32(size)
    check(run(env, c), want, bound)


@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 60])
@pytest.mark.parametrize("kind", [k for k in KINDS if k.get("causal", True)], ids=IDS)
def test_tokens_behind_a_query_cost_nothing(env, path, kind, size):
    """Tokens 90 to 99 of 200 diverge: the answers and gradients of the queries in front of them."""
    c = Fine(1, 200, 200, seed=4, **kind)
    c.dout[90:] = 0                                        # the keys' gradients are those of the queries in front
    want, bound = c.bounds()
    for array in (c.q, c.k, c.v):
        array[90:100] *= np.float32(size)
    got = run(env, c)
    check([g[:90] for g in got], [w[:90] for w in want], [e[:90] for e in bound])


@pytest.mark.parametrize("where", ["v", "k", "q"])
@pytest.mark.parametrize("size", [2.0 ** 13, 2.0 ** 20, 2.0 ** 40, 2.0 ** -13, 2.0 ** -40])
@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_one_token_of_another_size_among_those_that_are_seen(env, path, kind, where, size):
    """What depends on the token is as near to the formula as its own magnitudes allow, what does not is not touched.  Larger queries and keys come with a smaller scale, so that scores stay
    in an exponential's range, and smaller others: their scores are next to nothing, whichever of them."""
    c = Fine(1, 200, 200, seed=5, scale=kind["dim"] ** -0.5 * (min(1.0, 1 / size) if where != "v" else 1.0), **kind)
    getattr(c, where)[37] *= np.float32(size)
    getattr(c, where)[161] *= np.float32(size)
    check(run(env, c), *c.bounds())


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_every_token_of_a_size_of_its_own(env, path, kind):
    """Values from 2^-30 to 2^30, queries and output gradients too, keys the other way around."""
    rng = np.random.RandomState(11)
    c = Fine(2, 270, 270, seed=6, **kind)
    sizes = lambda: (2.0 ** rng.randint(-30, 31, (540, 1))).astype(np.float32)      # noqa: E731
    c.v *= sizes()
    by_query = sizes()
    c.q *= by_query
    c.dout *= sizes()
    c.scale = np.float32(c.scale * 2.0 ** -30)
    check(run(env, c), *c.bounds())


@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("dim", [64, 128])
def test_sequences_and_heads_of_any_size_side_by_side(env, path, dim, shared):
    """One sequence and head diverges token by token; the others do not notice."""
    c = Fine(3, 260, 260, 4, 2 if shared else 4, dim, seed=7)
    want, bound = c.bounds()
    rows = slice(260, 520)
    sizes = (2.0 ** np.random.RandomState(3).randint(-40, 41, (260, 1))).astype(np.float32)
    for a in (c.q, c.k, c.v, c.dout):
        a[rows, :dim] *= sizes
    got = run(env, c)
    for name, g, w, e, n in zip(("out", "dq", "dk", "dv"), got, want, bound, (4, 4, c.kv_heads, c.kv_heads)):
        view = lambda a: np.delete(a.reshape(3, 260, n, dim), 0, axis=2)[1] if n > 1 else a[:0]      # noqa: E731
        for b in (0, 2):
            within(g[260 * b:260 * (b + 1)], w[260 * b:260 * (b + 1)], e[260 * b:260 * (b + 1)], name)
        if not shared:
            within(view(g), view(w), view(e), name)


# ---- gradients of different sizes -------------------------------------------------------------------
@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_a_document_of_smaller_gradients_keeps_its_bits(env, path, kind):
    """Output gradients of the others up to 2^50 larger."""
    alone = Fine(1, 140, 140, seed=3, **kind)
    want, bound = alone.bounds()
    for size in (2.0 ** 5, 2.0 ** 10, 2.0 ** 13, 2.0 ** 17, 2.0 ** 20, 2.0 ** 50):
        c, mine, others = among_others(alone, 60, 75)
        c.dout[others] *= np.float32(size)
        check([g[mine] for g in run(env, c)], want, bound)


@pytest.mark.parametrize("kind", KINDS[:4], ids=IDS)
def test_later_queries_of_smaller_gradients(env, path, kind):
    """Each query's output gradient half of the one's before: the last keys are seen by the smallest alone."""
    c = Fine(1, 100, 100, seed=8, **dict(kind, causal=True))
    c.dout *= (2.0 ** -np.arange(100)).astype(np.float32)[:, None]
    check(run(env, c), *c.bounds())


@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 22, 2.0 ** 40, 2.0 ** 100])
@pytest.mark.parametrize("kind", [dict(queries=130, keys=130, heads=4, kv_heads=2, dim=64), dict(queries=4, keys=300, heads=2, kv_heads=1, dim=40), dict(queries=200, keys=200, heads=2, kv_heads=2, dim=128, bias=True)], ids=IDS)
@pytest.mark.parametrize("first, second", [(1, 2), (2, 1), (0, 2), (0, 1)])
def test_scores_of_any_size_where_the_directions_run_on_different_kernels(env, kind, size, first, second):
    """Then their scores differ by roundings, which are more than an exponent of 1 from 2^20 on: probabilities are at most 1 all the same, so the values' gradients are at most the sum
    of the output gradients, and all are finite."""
    c = Case(1, **kind)
    c.q *= np.float32(size ** 0.5)
    c.k *= np.float32(size ** 0.5)
    on = lambda v: None if v is None else env.nd.array(v, env.ctx)      # noqa: E731
    q, k, v, dout, slopes = (on(a) for a in (c.q, c.k, c.v, c.dout, c.slopes))
    out, stats = env.nd.empty(c.q.shape, env.ctx), env.nd.empty((1, c.heads, c.queries, 2), env.ctx)
    grads = [env.nd.empty(a.shape, env.ctx) for a in (c.q, c.k, c.v)]
    state = c.state(env)
    try:
        env.gpu_op.set_contraction_path(first)
        assert not env.gpu_op.attention_forward(q, k, v, None, None, slopes, out, stats, state, env.stream)
        env.gpu_op.set_contraction_path(second)
        assert not env.gpu_op.attention_backward(q, k, v, None, None, slopes, out, stats, dout, *grads, state, env.stream)
    finally:
        env.gpu_op.set_contraction_path(0)
    for a in (out, *grads):
        assert np.isfinite(a.asnumpy()).all()
    total = np.abs(c.dout).reshape(c.queries, c.kv_heads, -1, c.dim).sum((0, 2)).reshape(-1)
    allowed = 2.0 ** -10                                     # the sums
    if size < 2.0 ** 20:                                     # below 2^16 weights are taken as they come, and both kernels' scores are off by (D + 16) u of their terms
        norms = [np.linalg.norm(a.reshape(len(a), -1, c.dim).astype(np.float64), axis=2).max() for a in (c.q, c.k)]
        allowed += 2.0 ** (2 * (c.dim + 16) * U * float(c.scale) * np.log2(np.e) * norms[0] * norms[1]) - 1
    assert (np.abs(grads[2].asnumpy()) <= total * (1 + allowed)).all()
