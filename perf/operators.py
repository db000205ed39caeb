"""Performance cases: the operators of a pre-normalised residual block, through the wrappers that the graph calls.

Layer normalisation over the last axis, the residual sum of a dropped-out branch with the normalisation behind it, and the
gated dense layer out = act(x Wg) * (x Wv), weight = [Wg | Wv].  One pass is a forward call, a backward call, or both (a step).
Everything is float32, the one type of the library's arrays.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

own = False
EPS = 1e-5
MOST_ELEMENTS = 16384 * 4096                 # of a normalised tensor
MOST_PRODUCT = 8192 * 2048 * 8192            # rows x inputs x outputs of a gated layer
ACTIVATIONS = ("sigmoid", "relu", "tanh", "silu", "gelu")


def _norm(name, kind, direction, rows, cols, dropout=0.0, seed=0):
    c = {"op": kind, "pass": direction, "rows": rows, "cols": cols}
    if kind == "residual_norm":
        c.update(dropout=dropout, seed=seed)
    if name:
        c["name"] = name
    return c


def _gated(name, direction, rows, inputs, outputs, activation, keep=True):
    c = {"op": "gated", "pass": direction, "rows": rows, "inputs": inputs, "outputs": outputs, "activation": activation, "keep": keep}
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # hidden layer of the benchmark's perceptron at a small batch: latency
        _norm("norm fwd 64x256", "norm", "forward", 64, 256),
        # ragged rows that no 16-byte access fits
        _norm("norm fwd 1003x1029", "norm", "forward", 1003, 1029),
        # an ordinary layer's gradients
        _norm("norm bwd 4096x1024", "norm", "backward", 4096, 1024),
        # a wide layer over a long batch
        _norm("norm bwd 16384x4096", "norm", "backward", 16384, 4096),
        # a small batch in front of the next block
        _norm("residual fwd 32x768", "residual_norm", "forward", 32, 768, 0.1, 7),
        # odd widths
        _norm("residual bwd 1000x2050", "residual_norm", "backward", 1000, 2050, 0.5, 3),
        # forward and backward of a training step
        _norm("residual step 8192x2048", "residual_norm", "step", 8192, 2048, 0.2, 99),
        # one row answered: the weights are read once, nothing is kept for a gradient
        _gated("gated fwd 1x1024x4096", "forward", 1, 1024, 4096, "silu", False),
        # the perceptron's first layer, gated, at a small batch
        _gated("gated step 64x784x256", "step", 64, 784, 256, "sigmoid"),
        # ragged everywhere
        _gated("gated fwd 777x500x1003", "forward", 777, 500, 1003, "gelu"),
        # gradients of an ordinary layer
        _gated("gated bwd 2048x1024x4096", "backward", 2048, 1024, 4096, "gelu"),
        # a training step of a large one
        _gated("gated step 8192x2048x8192", "step", 8192, 2048, 8192, "silu"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    direction = rng.choice(("forward", "backward", "step"))
    if rng.random() < 0.55:
        cols = _log_int(rng, 2, 16384)
        rows = _log_int(rng, 1, min(32768, MOST_ELEMENTS // cols))
        if rng.random() < 0.5:
            return _norm(None, "norm", direction, rows, cols)
        return _norm(None, "residual_norm", direction, rows, cols, rng.choice((0.0, 0.1, 0.3, 0.5)), rng.randint(0, 100))
    inputs, outputs = _log_int(rng, 8, 4096), _log_int(rng, 8, 8192)
    rows = _log_int(rng, 1, min(8192, MOST_PRODUCT // (inputs * outputs)))
    return _gated(None, direction, rows, inputs, outputs, rng.choice(ACTIVATIONS), direction != "forward" or rng.random() < 0.5)


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    t = {}
    if case["op"] == "gated":
        rows, inputs, outputs = case["rows"], case["inputs"], case["outputs"]
        t["x"] = normal(rows, inputs)
        t["weight"] = normal(inputs, 2 * outputs).mul_(inputs ** -0.5)
        if case["pass"] != "forward":
            t["dout"] = normal(rows, outputs).mul_(0.1)
        return t
    rows, cols = case["rows"], case["cols"]
    # a residual stream: columns of different spread and offset, a few far larger than the rest
    spread = torch.exp(0.5 * normal(cols)) * torch.where(torch.rand(cols, generator=gen, device="cuda") < 0.01, 10.0, 1.0)
    t["x"] = normal(rows, cols) * spread + 0.3 * normal(cols)
    t["gamma"] = 1.0 + 0.1 * normal(cols)
    t["beta"] = 0.1 * normal(cols)
    if case["op"] == "residual_norm":
        t["branch"] = normal(rows, cols)
        if case["pass"] != "forward":
            t["dsum"] = 0.1 * normal(rows, cols)
    if case["pass"] != "forward":
        t["dout"] = 0.1 * normal(rows, cols)
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    if case["op"] == "gated" and case["pass"] == "backward":
        t["gates"] = t["x"] @ t["weight"]            # what the forward call left for the gradient
    return {"case": case, "in": t, "kept": {}}


# ---- plain form -------------------------------------------------------------------------------------------------------
def _kept(count, rate, seed):
    """Truth value per element: kept by the library's dropout generator (a 64-bit mix of index and seed, 24 bits of it)."""
    def wrapped(v):
        return v - (1 << 64) if v >= 1 << 63 else v

    def shifted(z, bits):                            # logical, not arithmetic
        return (z >> bits) & ((1 << (64 - bits)) - 1)

    z = torch.arange(1, count + 1, dtype=torch.int64, device="cuda") * wrapped(0x9E3779B97F4A7C15)
    z = z + wrapped(seed * 0xD1342543DE82EF95 & (1 << 64) - 1)
    z = (z ^ shifted(z, 30)) * wrapped(0xBF58476D1CE4E5B9)
    z = (z ^ shifted(z, 27)) * wrapped(0x94D049BB133111EB)
    z = z ^ shifted(z, 31)
    return shifted(z, 40).to(torch.float32) * (1.0 / 16777216.0) >= torch.tensor(rate, dtype=torch.float32, device="cuda")


def _scale(rate):
    return float(np.float32(1) / (np.float32(1) - np.float32(rate)))


def _normalised(x):
    centred = x - x.mean(-1, keepdim=True)
    inv = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    return centred * inv, inv


def _norm_gradients(x, gamma, dout):
    xhat, inv = _normalised(x)
    g = dout * gamma
    dx = inv * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    return dx, (dout * xhat).sum(0), dout.sum(0)


def _activation(kind, g):
    """The activation and its derivative."""
    if kind == "relu":
        return torch.clamp(g, min=0.0), (g > 0).to(g.dtype)
    if kind == "tanh":
        a = torch.tanh(g)
        return a, 1.0 - a * a
    if kind == "gelu":
        below = 0.5 * torch.erfc(-g * math.sqrt(0.5))
        return g * below, below + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    s = torch.sigmoid(g)
    if kind == "sigmoid":
        return s, s * (1.0 - s)
    return g * s, s * (1.0 + g * (1.0 - s))


def _plain(case, t):
    out = {}
    backward, forward = case["pass"] != "forward", case["pass"] != "backward"
    if case["op"] == "gated":
        n = case["outputs"]
        gates = t["x"] @ t["weight"] if forward else t["gates"]
        act, slope = _activation(case["activation"], gates[:, :n])
        if forward:
            out["out"] = act * gates[:, n:]
            if case["keep"]:
                out["gates"] = gates
        if backward:
            dgates = torch.cat((t["dout"] * gates[:, n:] * slope, t["dout"] * act), 1)
            out["dx"], out["dweight"] = dgates @ t["weight"].T, t["x"].T @ dgates
        return out
    x = t["x"]
    if case["op"] == "residual_norm":
        kept = _kept(x.numel(), case["dropout"], case["seed"]).reshape(x.shape)
        if forward:                                  # backward: x is the sum that the forward call left
            x = out["sum"] = x + torch.where(kept, t["branch"] * _scale(case["dropout"]), 0.0)
    if forward:
        out["out"] = _normalised(x)[0] * t["gamma"] + t["beta"]
    if backward:
        dx, out["dgamma"], out["dbeta"] = _norm_gradients(x, t["gamma"], t["dout"])
        if case["op"] == "residual_norm":
            dx = dx + t["dsum"]
            out["dbranch"] = torch.where(kept, dx * _scale(case["dropout"]), 0.0)
        out["dx"] = dx
    return out


# ---- the framework's calls --------------------------------------------------------------------------------------------
class _Shared(object):
    """Device memory for torch: float32, contiguous; ``owner`` keeps it alive."""

    def __init__(self, array):
        self.owner = array
        self.__cuda_array_interface__ = {"data": (array.data_ptr, False), "shape": array.shape, "typestr": "<f4", "version": 2}


_stream = []


def _hand_over(state):
    """The inputs as the framework's arrays, over the same memory, the arrays of the results, and the stream: what a program of
    the framework has instead of torch tensors.  Made at a state's first pass."""
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

    def result(name, like):
        array = ndarray.empty(like if isinstance(like, tuple) else tuple(like.shape), ndarray.gpu(0))
        kept["out"][name] = torch.as_tensor(_Shared(array), device="cuda")
        return array

    kept["out"] = {}
    a = kept["arrays"] = {name: view(tensor) for name, tensor in t.items()}
    forward, backward = case["pass"] != "backward", case["pass"] != "forward"
    if case["op"] == "gated":
        if forward:
            a["out"] = result("out", (case["rows"], case["outputs"]))
            a["gates"] = result("gates", (case["rows"], 2 * case["outputs"])) if case["keep"] else None
        if backward:
            a["dx"], a["dweight"] = result("dx", t["x"]), result("dweight", t["weight"])
    else:
        if forward:
            a["out"] = result("out", t["x"])
            if case["op"] == "residual_norm":
                a["sum"] = result("sum", t["x"])
        elif case["op"] == "residual_norm":
            a["sum"] = a["x"]
        if backward:
            a["dx"], a["dgamma"], a["dbeta"] = result("dx", t["x"]), result("dgamma", t["gamma"]), result("dbeta", t["gamma"])
            if case["op"] == "residual_norm":
                a["dbranch"] = result("dbranch", t["x"])
    if case["op"] == "residual_norm":
        kept["dropout"] = gpu_op.dropout_state(case["dropout"], case["seed"])
    kept["gpu_op"] = gpu_op
    return kept


def _framework(state):
    case, kept = state["case"], state["kept"] or _hand_over(state)
    a, gpu_op, stream = kept["arrays"], kept["gpu_op"], _stream[0]
    forward, backward = case["pass"] != "backward", case["pass"] != "forward"
    if case["op"] == "gated":
        if forward:
            gpu_op.gated_linear_forward(a["x"], a["weight"], a["gates"], a["out"], case["activation"], stream)
        if backward:
            gpu_op.gated_linear_backward(a["x"], a["weight"], a["gates"], a["dout"], a["dx"], a["dweight"], case["activation"], stream)
    elif case["op"] == "norm":
        if forward:
            gpu_op.layer_norm_forward(a["x"], a["gamma"], a["beta"], a["out"], EPS, stream)
        if backward:
            gpu_op.layer_norm_backward(a["x"], a["gamma"], a["dout"], a["dx"], a["dgamma"], a["dbeta"], EPS, stream)
    else:
        if forward:
            gpu_op.dropout_add_layer_norm_forward(a["branch"], a["x"], a["gamma"], a["beta"], a["sum"], a["out"], kept["dropout"], EPS, stream)
        if backward:
            gpu_op.dropout_add_layer_norm_backward(a["sum"], a["gamma"], a["dout"], a["dsum"], a["dbranch"], a["dx"], a["dgamma"], a["dbeta"], kept["dropout"], EPS, stream)
    return kept["out"]


def run(state):
    if own:
        return _framework(state)
    return _plain(state["case"], state["in"])


def work(case):
    rows = case["rows"]
    forward, backward = case["pass"] != "backward", case["pass"] != "forward"
    if case["op"] == "gated":
        k, n = case["inputs"], case["outputs"]
        floats = flops = 0
        if forward:
            floats += rows * k + 2 * k * n + rows * n + (2 * rows * n if case["keep"] else 0)
            flops += 4 * rows * k * n
        if backward:
            floats += rows * n + 2 * (rows * k + 2 * k * n) + 2 * rows * n
            flops += 8 * rows * k * n
        if forward and backward:                     # inputs, weights and gates stay where they are between the two
            floats -= rows * k + 2 * k * n + 2 * rows * n
        return {"bytes": 4 * floats, "flops": flops}
    size, cols = rows * case["cols"], case["cols"]
    residual = case["op"] == "residual_norm"
    floats = 0
    if forward:
        floats += size * (4 if residual else 2) + 2 * cols
    if backward:
        floats += size * (5 if residual else 3) + 3 * cols
    if forward and backward:                         # the normalised tensor and gamma
        floats -= size + cols
    return {"bytes": 4 * floats, "flops": size * (8 * forward + 14 * backward)}


# ---- the definitions, in 64 bits --------------------------------------------------------------------------------------
def _mask_of(shape, rate, seed):
    index = np.arange(1, int(np.prod(shape)) + 1, dtype=np.uint64)
    with np.errstate(over="ignore"):
        z = index * np.uint64(0x9E3779B97F4A7C15) + np.uint64(seed) * np.uint64(0xD1342543DE82EF95)
        z ^= z >> np.uint64(30)
        z *= np.uint64(0xBF58476D1CE4E5B9)
        z ^= z >> np.uint64(27)
        z *= np.uint64(0x94D049BB133111EB)
        z ^= z >> np.uint64(31)
    keep = (z >> np.uint64(40)) >= np.ceil(np.float64(np.float32(rate)) * 2 ** 24)
    return torch.from_numpy(keep.reshape(shape)).cuda()


def exact(case, seed):
    state = prepare(case, seed)
    d = {name: tensor.double() for name, tensor in state["in"].items()}
    forward, backward = case["pass"] != "backward", case["pass"] != "forward"
    got = {}
    if case["op"] == "gated":
        n = case["outputs"]
        z = torch.mm(d["x"], d["weight"]) if forward else d["gates"]
        gate, value = z[:, :n].clone().requires_grad_(), z[:, n:].clone().requires_grad_()
        with torch.enable_grad():
            a = {"sigmoid": lambda v: 1 / (1 + torch.exp(-v)), "relu": lambda v: torch.where(v > 0, v, torch.zeros_like(v)), "tanh": torch.tanh,
                 "silu": lambda v: v / (1 + torch.exp(-v)), "gelu": lambda v: v * (1 + torch.erf(v / math.sqrt(2))) / 2}[case["activation"]](gate)
            h = a * value
            if backward:
                dgate, dvalue = torch.autograd.grad(h, (gate, value), d["dout"])
        if forward:
            got["out"] = h.detach()
            if case["keep"]:
                got["gates"] = z
        if backward:
            wg, wv = d["weight"][:, :n], d["weight"][:, n:]
            got["dx"] = torch.mm(dgate, wg.T) + torch.mm(dvalue, wv.T)
            got["dweight"] = torch.cat((torch.mm(d["x"].T, dgate), torch.mm(d["x"].T, dvalue)), 1)
        return got
    x = d["x"]
    if case["op"] == "residual_norm":
        keep = _mask_of(tuple(x.shape), case["dropout"], case["seed"])
        times = keep * (1.0 / float(np.float32(1) - np.float32(case["dropout"])))
        if forward:
            x = got["sum"] = d["x"] + d["branch"] * times
    x = x.clone().requires_grad_()
    gamma, beta = d["gamma"].requires_grad_(), d["beta"].requires_grad_()
    with torch.enable_grad():
        mean = x.sum(1, keepdim=True) / case["cols"]
        var = ((x - mean) ** 2).sum(1, keepdim=True) / case["cols"]
        y = (x - mean) / torch.sqrt(var + EPS) * gamma + beta
        if backward:
            dx, dgamma, dbeta = torch.autograd.grad(y, (x, gamma, beta), d["dout"])
    if forward:
        got["out"] = y.detach()
    if backward:
        got["dgamma"], got["dbeta"], got["dx"] = dgamma, dbeta, dx
        if case["op"] == "residual_norm":
            got["dx"] = dx + d["dsum"]
            got["dbranch"] = got["dx"] * times
    return got
