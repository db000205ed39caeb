"""Performance cases: the operators that mix tokens, through the wrappers that the graph calls.

Rotary positions, the norms of query and key heads with the rotation in the same pass, and attention.  Their arrays are what a matrix
product of all tokens makes: (sequences x length) rows of heads x head_dim columns.  One pass is a forward call, a backward call, or both
(a step).  Everything is float32, the one type of the library's arrays.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

own = False
EPS = 1e-6
MOST_SCORES = 1 << 28                        # sequences x heads x queries x keys of a drawn attention
MOST_ELEMENTS = 1 << 26                      # of a rotated tensor
LOG2E = math.log2(math.e)
BASE = 10000.0


def _rotary(name, direction, batch, length, heads, dim, rotated, layout, scaling="none", start=0):
    c = {"op": "rotary", "pass": direction, "batch": batch, "length": length, "heads": heads, "dim": dim, "rotated": rotated, "layout": layout,
         "scaling": scaling, "start": start}
    if name:
        c["name"] = name
    return c


def _norm(name, direction, batch, length, heads, kv_heads, dim, rotated, layout, scaling="none", start=0):
    c = {"op": "head_norm", "pass": direction, "batch": batch, "length": length, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotated": rotated,
         "layout": layout, "scaling": scaling, "start": start}
    if name:
        c["name"] = name
    return c


def _attention(name, direction, batch, queries, keys, heads, kv_heads, dim, mask, window=0, bias=False, cap=0.0):
    c = {"op": "attention", "pass": direction, "batch": batch, "queries": queries, "keys": keys, "heads": heads, "kv_heads": kv_heads, "dim": dim,
         "mask": mask, "window": window, "bias": bias, "cap": cap}
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one token of four sequences, far into them: latency
        _rotary("rotary fwd 4x1x8x64", "forward", 4, 1, 8, 64, 64, "interleaved", "none", 5000),
        # ragged: odd head width, part of the head
        _rotary("rotary step 3x333x5x90", "step", 3, 333, 5, 90, 30, "half", "linear"),
        # a layer's queries, scaled for a context longer than the trained one
        _rotary("rotary bwd 2x8192x16x128", "backward", 2, 8192, 16, 128, 128, "half", "parts"),
        # one token's queries and keys
        _norm("head norm fwd 2x1x16x128", "forward", 2, 1, 16, 4, 128, 128, "half", "none", 777),
        # a training step on a ragged batch
        _norm("head norm step 2x777x6x80", "step", 2, 777, 6, 2, 80, 40, "interleaved", "stretched"),
        # gradients of a layer over a long batch, shared key heads
        _norm("head norm bwd 4x4096x16x128", "backward", 4, 4096, 16, 4, 128, 128, "half"),
        # eight rows answered: one token each against what came before it, shared key-value heads
        _attention("attn fwd 8x1x4096", "forward", 8, 1, 4096, 32, 8, 128, "causal"),
        # a small batch of short sequences: latency
        _attention("attn step 4x64x64", "step", 4, 64, 64, 4, 4, 64, "causal"),
        # ragged: odd width and length, a bidirectional prefix, scores biased by distance
        _attention("attn step 2x777x777", "step", 2, 777, 777, 6, 2, 72, "prefix", 0, True),
        # several documents and padding packed into one long row
        _attention("attn fwd 1x8192 documents", "forward", 1, 8192, 8192, 8, 2, 64, "documents"),
        # gradients of a local layer with capped scores
        _attention("attn bwd 4x2048 window", "backward", 4, 2048, 2048, 8, 8, 64, "window", 512, False, 30.0),
        # a training step of a long layer
        _attention("attn step 2x4096x4096", "step", 2, 4096, 4096, 16, 4, 128, "causal"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.random()
    dim = rng.choice((16, 32, 40, 64, 64, 72, 80, 96, 128, 128, rng.randint(8, 128)))
    kv_heads, group = rng.choice((1, 2, 4, 8)), rng.choice((1, 1, 2, 4, 8))
    heads = kv_heads * group
    if kind < 0.4:
        direction = rng.choice(("forward", "backward", "step"))
        rotated = 2 * rng.randint(1, dim // 2) if rng.random() < 0.4 else dim // 2 * 2
        layout, scaling = rng.choice(("half", "interleaved")), rng.choice(("none", "linear", "stretched", "parts"))
        length = _log_int(rng, 1, 16384)
        batch = _log_int(rng, 1, max(1, min(64, MOST_ELEMENTS // (length * heads * dim))))
        start = rng.choice((0, 0, rng.randint(1, 100000)))
        if rng.random() < 0.5:
            return _rotary(None, direction, batch, length, heads, dim, rotated, layout, scaling, start)
        return _norm(None, direction, batch, length, heads, kv_heads, dim, rotated, layout, scaling, start)
    single = rng.random() < 0.3
    direction = "forward" if single else rng.choice(("forward", "backward", "step"))
    keys = _log_int(rng, 1 if direction == "forward" else 8, 8192)       # a row that sees one key has no gradient but rounding
    queries = rng.choice((1, 1, 2, 5)) if single else keys if rng.random() < 0.8 else _log_int(rng, min(8, keys), keys)
    queries = min(queries, keys)
    mask = rng.choice(("causal", "causal", "full", "window", "documents", "prefix"))
    while heads > 1 and heads * queries * keys > MOST_SCORES:
        heads, kv_heads = heads // 2, max(1, kv_heads // 2)
    batch = _log_int(rng, 1, max(1, min(32, MOST_SCORES // (heads * queries * keys), (1 << 23) // (keys * max(1, kv_heads)))))
    window = _log_int(rng, min(4, keys), keys) if mask == "window" else 0
    return _attention(None, direction, batch, queries, keys, heads, kv_heads, dim, mask, window, rng.random() < 0.3, rng.choice((0.0, 0.0, 30.0, 50.0)))


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _frequencies(case):
    """Turns of each pair per position, in 64 bits, and the factor of the rotated values."""
    pairs, factor, trained = case["rotated"] // 2, 8.0, 4096
    base, amplitude = BASE, 1.0
    if case["scaling"] == "stretched" and pairs > 1:
        base *= factor ** (pairs / (pairs - 1.0))
    f = base ** (-np.arange(pairs, dtype=np.float64) / pairs)
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "parts":               # pairs of many turns within the trained length stay, those of few are stretched
        kept = np.clip((trained * f / (2 * np.pi) - 1.0) / (32.0 - 1.0), 0.0, 1.0)
        f, amplitude = f * (kept + (1 - kept) / factor), 0.1 * math.log(factor) + 1.0
    return torch.from_numpy(f).cuda(), amplitude


def _documents(total, padding, gen):
    """Numbers of documents that follow one another, the last tokens padding (-1)."""
    cuts = torch.rand(total, generator=gen, device="cuda") < 6.0 / total
    numbers = torch.cumsum(cuts.int(), 0).float()
    numbers[total - padding:] = -1.0
    return numbers


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    backward = case["pass"] != "forward"
    dim, t = case["dim"], {}
    if case["op"] == "rotary":
        rows, cols = case["batch"] * case["length"], case["heads"] * dim
        if case["pass"] != "backward":
            t["x"] = normal(rows, cols)
        if backward:
            t["dout"] = normal(rows, cols).mul_(0.1)
        return t
    if case["op"] == "head_norm":
        rows = case["batch"] * case["length"]
        for name, heads in (("q", case["heads"]), ("k", case["kv_heads"])):
            t[name] = normal(rows, heads * dim) * (1.0 + 2.0 * torch.rand(heads * dim, generator=gen, device="cuda"))
            t["gamma_" + name] = 1.0 + 0.2 * normal(dim)
            if backward:
                t["dout_" + name] = normal(rows, heads * dim).mul_(0.1)
        return t
    b, tq, tk = case["batch"], case["queries"], case["keys"]
    # normed heads of a trained layer: some columns weigh more
    t["q"] = normal(b * tq, case["heads"] * dim) * (0.7 + 0.8 * torch.rand(case["heads"] * dim, generator=gen, device="cuda"))
    t["k"] = normal(b * tk, case["kv_heads"] * dim) * (0.7 + 0.8 * torch.rand(case["kv_heads"] * dim, generator=gen, device="cuda"))
    t["v"] = normal(b * tk, case["kv_heads"] * dim)
    if case["mask"] == "documents":
        t["documents"] = torch.cat([_documents(tk, tk // 20 if tq == tk else 0, gen) for _ in range(b)])      # no padding behind a token that is answered
    if case["mask"] == "prefix":
        t["prefix"] = torch.floor(torch.rand(b, generator=gen, device="cuda") * tk)
    if case["bias"]:
        t["slopes"] = torch.exp2(-8.0 * torch.arange(1, case["heads"] + 1, device="cuda") / case["heads"])
    if backward:
        t["dout"] = normal(b * tq, case["heads"] * dim).mul_(0.1)
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    state = {"case": case, "in": t, "kept": {}}
    if case["op"] != "attention":
        state["frequencies"], state["amplitude"] = _frequencies(case)
    elif case["pass"] == "backward":             # what the forward call left for the gradient
        t["out"], t["stats"] = _attention_forward(case, t)[:2]
    return state


# ---- plain form -------------------------------------------------------------------------------------------------------
def _turned(x, case, frequencies, amplitude, back=False):
    """x (rows, heads, dim) rotated by its position; `back`: by the opposite angle."""
    length, rotated = case["length"], case["rotated"]
    positions = (torch.arange(x.shape[0], device="cuda") % length + case["start"]).double()
    angles = (positions[:, None] * frequencies)[:, None, :]
    cos, sin = (torch.cos(angles) * amplitude).float(), (torch.sin(angles) * (-amplitude if back else amplitude)).float()
    out = x.clone()
    if case["layout"] == "half":
        a, b = x[..., :rotated // 2], x[..., rotated // 2:rotated]
        out[..., :rotated // 2], out[..., rotated // 2:rotated] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., 0:rotated:2], x[..., 1:rotated:2]
        out[..., 0:rotated:2], out[..., 1:rotated:2] = a * cos - b * sin, a * sin + b * cos
    return out


def _plain_rotary(state):
    case, t, out = state["case"], state["in"], {}
    if "x" in t:
        x = t["x"]
        out["out"] = _turned(x.reshape(x.shape[0], case["heads"], case["dim"]), case, state["frequencies"], state["amplitude"]).reshape(x.shape)
    if "dout" in t:
        d = t["dout"]
        out["dx"] = _turned(d.reshape(d.shape[0], case["heads"], case["dim"]), case, state["frequencies"], state["amplitude"], True).reshape(d.shape)
    return out


def _plain_head_norm(state):
    case, t, out = state["case"], state["in"], {}

    def one(name, heads):
        x = t[name].reshape(-1, heads, case["dim"])
        gamma = t["gamma_" + name]
        inv = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        if case["pass"] != "backward":
            out["out_" + name] = _turned(x * inv * gamma, case, state["frequencies"], state["amplitude"]).reshape(t[name].shape)
        if case["pass"] != "forward":
            u = _turned(t["dout_" + name].reshape(x.shape), case, state["frequencies"], state["amplitude"], True)
            n, g = x * inv, u * gamma
            out["d" + name] = (inv * (g - n * (g * n).mean(-1, keepdim=True))).reshape(t[name].shape)
            out["dgamma_" + name] = (u * n).sum((0, 1))

    one("q", case["heads"])
    one("k", case["kv_heads"])
    return out


def _split(x, batch, heads, dim):
    """(batch * length, heads * dim) -> batch, heads, length, dim"""
    return x.reshape(batch, -1, heads, dim).permute(0, 2, 1, 3)


def _joined(x):
    return x.permute(0, 2, 1, 3).reshape(x.shape[0] * x.shape[2], -1)


def _seen(case, t):
    """Truth value of each query and key: broadcasts to batch, heads, queries, keys."""
    b, tq, tk = case["batch"], case["queries"], case["keys"]
    i = torch.arange(tk - tq, tk, device="cuda")[:, None]
    j = torch.arange(tk, device="cuda")[None, :]
    seen = torch.ones((tq, tk), dtype=torch.bool, device="cuda") if case["mask"] == "full" else j <= i
    if case["window"]:
        seen = seen & (i - j < case["window"])
    seen = seen[None, None]
    if "prefix" in t:
        seen = seen | (j[None, None] < t["prefix"].reshape(b, 1, 1, 1))
    if "documents" in t:
        of = t["documents"].reshape(b, 1, tk)
        seen = seen & (of[:, :, tk - tq:, None] == of[:, :, None, :]) & (of[:, :, None, :] >= 0)
    return seen


def _scores(case, t):
    """The scores after cap and bias, in units of log 2, minus infinity where a query does not see the key; the cap's derivative or None."""
    b, h, tq, tk, dim = case["batch"], case["heads"], case["queries"], case["keys"], case["dim"]
    q, k = _split(t["q"], b, h, dim), _split(t["k"], b, case["kv_heads"], dim)
    z = torch.matmul(q.reshape(b, case["kv_heads"], -1, dim), k.transpose(-1, -2)).reshape(b, h, tq, tk)
    z = z * (1.0 / math.sqrt(dim))
    slope = None
    if case["cap"]:
        z = torch.tanh(z / case["cap"])
        slope = 1.0 - z * z
        z = z * case["cap"]
    if "slopes" in t:
        i, j = torch.arange(tk - tq, tk, device="cuda")[:, None], torch.arange(tk, device="cuda")[None, :]
        z = z - t["slopes"].reshape(1, h, 1, 1) * (i - j).abs().float()
    return torch.where(_seen(case, t), z * LOG2E, -math.inf), slope


def _attention_forward(case, t):
    b, h, tq, tk, dim = case["batch"], case["heads"], case["queries"], case["keys"], case["dim"]
    z, slope = _scores(case, t)
    most = z.amax(-1, keepdim=True)
    most = torch.where(torch.isinf(most), 0.0, most)
    p = torch.exp2(z - most)
    total = p.sum(-1, keepdim=True)
    inv = torch.where(total > 0, 1.0 / total, 0.0)
    p = p * inv
    v = _split(t["v"], b, case["kv_heads"], dim)
    out = torch.matmul(p.reshape(b, case["kv_heads"], -1, tk), v).reshape(b, h, tq, dim)
    return _joined(out), torch.cat((most, inv), -1), p, slope


def _plain_attention(state):
    case, t, got = state["case"], state["in"], {}
    b, h, g, tq, tk, dim = case["batch"], case["heads"], case["kv_heads"], case["queries"], case["keys"], case["dim"]
    if case["pass"] == "backward":
        z, slope = _scores(case, t)
        out, p = t["out"], torch.exp2(z - t["stats"][..., :1]) * t["stats"][..., 1:]
    else:
        out, _, p, slope = _attention_forward(case, t)
        got["out"] = out
    if case["pass"] != "forward":
        do = _split(t["dout"], b, h, dim)
        q, k, v = _split(t["q"], b, h, dim), _split(t["k"], b, g, dim), _split(t["v"], b, g, dim)
        dp = torch.matmul(do.reshape(b, g, -1, dim), v.transpose(-1, -2)).reshape(b, h, tq, tk)
        ds = p * (dp - (do * _split(out, b, h, dim)).sum(-1, keepdim=True)) * (1.0 / math.sqrt(dim))
        if slope is not None:
            ds = ds * slope
        ds, p = ds.reshape(b, g, -1, tk), p.reshape(b, g, -1, tk)
        got["dq"] = _joined(torch.matmul(ds, k).reshape(b, h, tq, dim))
        got["dk"] = _joined(torch.matmul(ds.transpose(-1, -2), q.reshape(b, g, -1, dim)))
        got["dv"] = _joined(torch.matmul(p.transpose(-1, -2), do.reshape(b, g, -1, dim)))
    return got


# ---- the framework's calls --------------------------------------------------------------------------------------------
class _Shared(object):
    """Device memory for torch: float32, contiguous; ``owner`` keeps it alive."""

    def __init__(self, array):
        self.owner = array
        self.__cuda_array_interface__ = {"data": (array.data_ptr, False), "shape": array.shape, "typestr": "<f4", "version": 2}


_stream = []


def _hand_over(state):
    """The inputs as the framework's arrays, over the same memory, the arrays of the results, the descriptor and the stream: what a program
    of the framework has instead of torch tensors.  Made at a state's first pass."""
    from tinyflow_b200 import gpu_op, ndarray
    case, t = state["case"], state["in"]
    torch.cuda.current_stream().synchronize()
    if not _stream:
        _stream.append(gpu_op.create_cudaStream())
    kept = state["kept"]

    def view(tensor):
        c = ndarray.DLArray()
        dims = (ctypes.c_int64 * tensor.dim())(*tensor.shape)
        c.data, c.ctx, c.ndim, c.shape = tensor.data_ptr(), ndarray.gpu(0), tensor.dim(), ctypes.cast(dims, ctypes.POINTER(ctypes.c_int64))
        array = ndarray.NDArray(ctypes.pointer(c))
        array.is_freed = True                        # torch frees it
        return array

    a = kept["arrays"] = {name: view(tensor) for name, tensor in t.items()}
    kept["out"] = {}

    def result(name, like, shown=True):
        a[name] = ndarray.empty(like if isinstance(like, tuple) else tuple(like.shape), ndarray.gpu(0))
        if shown:
            kept["out"][name] = torch.as_tensor(_Shared(a[name]), device="cuda")

    forward, backward = case["pass"] != "backward", case["pass"] != "forward"
    if case["op"] == "attention":
        if forward:
            result("out", t["q"])
            a["stats"] = None
            if backward:
                result("stats", (case["batch"], case["heads"], case["queries"], 2), False)
        if backward:
            result("dq", t["q"])
            result("dk", t["k"])
            result("dv", t["v"])
        kept["state"] = gpu_op.attention_state(case["queries"], case["heads"], case["kv_heads"], case["mask"] != "full", case["window"], 1.0 / math.sqrt(case["dim"]), case["cap"])
    else:
        for name in ("q", "k") if case["op"] == "head_norm" else ("",):
            if name:
                if forward:
                    result("out_" + name, t[name])
                if backward:
                    result("d" + name, t[name])
                    result("dgamma_" + name, t["gamma_" + name])
            else:
                if forward:
                    result("out", t["x"])
                if backward:
                    result("dx", t["dout"])
        kept["state"] = gpu_op.rotary_state(case["dim"], case["rotated"], case["layout"], BASE, case["scaling"], 8.0, 4096)
    kept["gpu_op"] = gpu_op
    return kept


def _framework(state):
    case, kept = state["case"], state["kept"] or _hand_over(state)
    a, gpu_op, held, stream = kept["arrays"], kept["gpu_op"], kept["state"], _stream[0]
    forward, backward = case["pass"] != "backward", case["pass"] != "forward"
    if case["op"] == "rotary":
        if forward:
            gpu_op.rotary_forward(a["x"], None, a["out"], case["length"], case["start"], held, stream)
        if backward:
            gpu_op.rotary_backward(a["dout"], None, a["dx"], case["length"], case["start"], held, stream)
    elif case["op"] == "head_norm":
        if forward:
            gpu_op.head_norm_rotary_forward(a["q"], a["k"], a["gamma_q"], a["gamma_k"], None, a["out_q"], a["out_k"], case["length"], case["start"], EPS, held, stream)
        if backward:
            gpu_op.head_norm_rotary_backward(a["q"], a["k"], a["gamma_q"], a["gamma_k"], None, a["dout_q"], a["dout_k"], a["dq"], a["dk"], a["dgamma_q"], a["dgamma_k"],
                                             case["length"], case["start"], EPS, held, stream)
    else:
        masks = a.get("documents"), a.get("prefix"), a.get("slopes")
        if forward:
            gpu_op.attention_forward(a["q"], a["k"], a["v"], *masks, a["out"], a["stats"], held, stream)
        if backward:
            gpu_op.attention_backward(a["q"], a["k"], a["v"], *masks, a["out"], a["stats"], a["dout"], a["dq"], a["dk"], a["dv"], held, stream)
    return kept["out"]


def run(state):
    if own:
        return _framework(state)
    return {"rotary": _plain_rotary, "head_norm": _plain_head_norm, "attention": _plain_attention}[state["case"]["op"]](state)


def work(case):
    forward, backward = case["pass"] != "backward", case["pass"] != "forward"
    if case["op"] != "attention":
        rows = case["batch"] * case["length"]
        size = rows * case["dim"] * (case["heads"] + case.get("kv_heads", 0))
        norm = case["op"] == "head_norm"
        floats = size * (2 * forward + (3 if norm else 2) * backward - (1 if norm and forward and backward else 0)) + (2 * case["dim"] * (forward + backward) if norm else 0)
        return {"bytes": 4 * floats, "flops": size * ((7 if norm else 3) * forward + (12 if norm else 3) * backward)}
    b, h, g, tq, tk, dim = case["batch"], case["heads"], case["kv_heads"], case["queries"], case["keys"], case["dim"]
    i = np.arange(tk - tq, tk, dtype=np.float64)
    last = np.full(tq, tk - 1.0) if case["mask"] == "full" else i
    pairs = float((last - (np.maximum(i - case["window"] + 1, 0) if case["window"] else 0) + 1).sum())
    if case["mask"] == "prefix":                 # a prefix of half the keys, on average
        pairs += float(np.maximum(tk / 2 - last - 1, 0).sum())
    if case["mask"] == "documents":              # seven documents a row
        pairs /= 7.0
    queries, keys = b * tq * h * dim, 2 * b * tk * g * dim
    floats = 0
    if forward:
        floats += 2 * queries + keys
    if backward:
        floats += (3 if forward else 4) * queries + keys + (0 if forward else keys)
    return {"bytes": 4 * floats, "flops": b * h * pairs * dim * (4 * forward + 10 * backward)}


# ---- the definitions, in 64 bits --------------------------------------------------------------------------------------
def _exact_turns(case):
    """Rotation of every position as matrices (length, dim, dim) would be large: cos and sin per element and the element that it is paired with."""
    dim, r = case["dim"], case["rotated"]
    m = r // 2
    factor, trained, base, amplitude = 8.0, 4096.0, BASE, 1.0
    e = torch.arange(m, dtype=torch.float64, device="cuda")
    if case["scaling"] == "stretched" and r > 2:
        base = base * factor ** (r / (r - 2))
    f = torch.exp(-2 * e / r * math.log(base))
    if case["scaling"] == "linear":
        f /= factor
    elif case["scaling"] == "parts":
        turns = trained * f / (2 * math.pi)
        ramp = ((turns - 1) / 31).clamp(0, 1)
        f = ramp * f + (1 - ramp) * f / factor
        amplitude = 1 + math.log(factor) / 10
    where = torch.arange(dim, device="cuda")
    pair, sign, number = where.clone(), torch.zeros(dim, dtype=torch.float64, device="cuda"), torch.full((dim,), -1, device="cuda")
    first = torch.arange(m, device="cuda") * (1 if case["layout"] == "half" else 2)
    second = first + (m if case["layout"] == "half" else 1)
    pair[first], pair[second] = second, first
    sign[first], sign[second] = -1.0, 1.0
    number[first] = number[second] = torch.arange(m, device="cuda")
    at = torch.arange(case["length"], dtype=torch.float64, device="cuda") + case["start"]
    angle = torch.outer(at, torch.cat((f, torch.zeros(1, dtype=torch.float64, device="cuda")))[number])
    times = torch.where(number >= 0, amplitude, 1.0)
    return torch.cos(angle) * times, torch.sin(angle) * sign * times, pair


def _exact_rotated(x, case, turns):
    cos, sin, pair = (v[:, None, :] if v.dim() == 2 else v for v in turns)
    x = x.reshape(case["batch"], case["length"], -1, case["dim"])
    return x * cos + x[..., pair] * sin


def _exact_heads(case, d):
    turns, got = _exact_turns(case), {}
    names = (("x", "out", "dout", "dx"),) if case["op"] == "rotary" else (("q", "out_q", "dout_q", "dq"), ("k", "out_k", "dout_k", "dk"))
    for x, y, dy, dx in names:
        like = d[x] if x in d else d[dy]
        leaf = (d[x] if x in d else torch.zeros_like(d[dy])).clone().requires_grad_()
        leaves = [leaf]
        with torch.enable_grad():
            rows = leaf.reshape(case["batch"], case["length"], -1, case["dim"])
            if case["op"] == "head_norm":
                gamma = d["gamma_" + x].requires_grad_()
                leaves.append(gamma)
                rows = rows / torch.sqrt((rows ** 2).sum(-1, keepdim=True) / case["dim"] + EPS) * gamma
            z = _exact_rotated(rows, case, turns).reshape(like.shape)
            if case["pass"] != "forward":
                grads = torch.autograd.grad(z, leaves, d[dy])
                got[dx] = grads[0]
                if len(grads) > 1:
                    got["dgamma_" + x] = grads[1]
        if case["pass"] != "backward":
            got[y] = z.detach()
    return got


def _exact_attention(case, d):
    """Sequence by sequence, each key-value head's group by itself."""
    b, h, g, tq, tk, dim = case["batch"], case["heads"], case["kv_heads"], case["queries"], case["keys"], case["dim"]
    q, k, v = d["q"].view(b, tq, g, h // g, dim), d["k"].view(b, tk, g, dim), d["v"].view(b, tk, g, dim)
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    do = d["dout"].view(q.shape) if "dout" in d else None
    place = torch.arange(tk, dtype=torch.float64, device="cuda")
    gap = place[tk - tq:, None] - place[None, :]
    for n in range(b):
        hidden = gap < 0 if case["mask"] != "full" else torch.zeros_like(gap, dtype=torch.bool)
        if case["window"]:
            hidden = hidden | (gap >= case["window"])
        if "prefix" in d:
            hidden = hidden & ~(place[None, :] < d["prefix"][n])
        if "documents" in d:
            of = d["documents"].view(b, tk)[n]
            hidden = hidden | (of[tk - tq:, None] != of[None, :]) | (of[None, :] < 0)
        blind = hidden.all(1, keepdim=True)
        for m in range(g):
            s = torch.einsum("qhd,kd->hqk", q[n, :, m], k[n, :, m]) / math.sqrt(dim)
            inner = None
            if case["cap"]:
                inner = torch.tanh(s / case["cap"])
                s = case["cap"] * inner
            if "slopes" in d:
                s = s - d["slopes"][m * (h // g):(m + 1) * (h // g), None, None] * gap.abs()
            s = s.masked_fill(hidden, -math.inf).masked_fill(blind, 0.0)
            p = torch.softmax(s, -1).masked_fill(hidden, 0.0)
            out[n, :, m] = torch.einsum("hqk,kd->qhd", p, v[n, :, m])
            if do is not None:
                dv[n, :, m] = torch.einsum("hqk,qhd->kd", p, do[n, :, m])
                dp = torch.einsum("qhd,kd->hqk", do[n, :, m], v[n, :, m])
                ds = p * (dp - (p * dp).sum(-1, keepdim=True))
                if inner is not None:
                    ds = ds * (1 - inner ** 2)
                dq[n, :, m] = torch.einsum("hqk,kd->qhd", ds, k[n, :, m]) / math.sqrt(dim)
                dk[n, :, m] = torch.einsum("hqk,qhd->kd", ds, q[n, :, m]) / math.sqrt(dim)
    got = {}
    if case["pass"] != "backward":
        got["out"] = out.view(d["q"].shape)
    if case["pass"] != "forward":
        got.update(dq=dq.view(d["q"].shape), dk=dk.view(d["k"].shape), dv=dv.view(d["v"].shape))
    return got


def exact(case, seed):
    d = {name: tensor.double() for name, tensor in _inputs(case, seed).items()}
    return _exact_attention(case, d) if case["op"] == "attention" else _exact_heads(case, d)
