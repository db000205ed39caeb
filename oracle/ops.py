"""CPU restatement (numpy) of every operator on the training-step hot path.

TEST INFRASTRUCTURE ONLY.  Nothing in ``tinyflow_b200`` imports this package; it is the checker
the GPU kernels are compared against (tests/, ``__graft_entry__.smoke()``) and the CPU arm that
``bench.py`` times beside the GPU number.  Every function works in the dtype of its inputs, so the
same code is the fp64 parity oracle and the fp32 timed baseline.

Parity status.  The reference's own numpy branches exist only for add / mul / matmul / relu /
softmax / softmax-cross-entropy (pycode/tinyflow/autodiff.py:312-314, 385-386, 452-467, 681-686,
700-704, 753-754, 777-779); for those this module is pinned against the reference itself through
the fixtures in tests/golden/ (generated by tests/golden/make_golden.py, which imports the reference).
Convolution, pooling, batch-norm, activation-softmax, reduce and dropout are cuDNN calls in the
reference (src/gpu_op.cu:1653-4460) with print-only tests, so for those ops parity is UNPINNED
against the reference: the restatement follows the cuDNN semantics the reference configures (cited
per function) and is cross-checked against torch-CPU float64 autograd in tests/test_oracle.py.

Choices where the closed library's behaviour cannot be observed here:
  1. max-pool ties: the first maximum in row-major window order gets the gradient;
  2. a max-pool window that covers only padding outputs 0.0;
  3. softmax is computed with max subtraction (cuDNN FAST mode omits it; identical unless it overflows);
  4. dropout keep-mask is a counter-based hash of (seed, element index) — same function as the CUDA kernel;
  5. average pooling divides by the full window area, padding included.
"""
from __future__ import annotations

import numpy as np

BN_EPS = 1e-5


# ---- elementwise / fill (src/gpu_op.cu:39-45, 193-235) ---------------------------------------------
def relu(x):
    return np.maximum(x, 0)


def relu_grad(x, g):
    """x > 0 ? g : 0  (src/gpu_op.cu:230-235; the CUDA kernel, not the 0.5-at-zero numpy branch)."""
    return np.where(x > 0, g, 0).astype(g.dtype)


def sigmoid(x):
    return 1.0 / (1.0 + np.exp(-x))


# ---- broadcast / reduce (src/gpu_op.cu:47-52, 108-123, 628-884) --------------------------------------
def broadcast_tail(x, out_shape):
    """out.flat[i] = x.flat[i % x.size]."""
    n = int(np.prod(out_shape))
    return np.resize(x.reshape(-1), n).reshape(out_shape)


def broadcast_channel(x, out_shape):
    """out[n, c, ...] = x[c]."""
    shape = (1, out_shape[1]) + (1,) * (len(out_shape) - 2)
    return np.broadcast_to(x.reshape(shape), out_shape).copy()


def reduce_sum(x, in_dims, out_dims):
    """Sum over every axis whose output extent is 1 (cudnnReduceTensor ADD as configured at src/gpu_op.cu:628-810)."""
    x = x.reshape(in_dims)
    axes = tuple(i for i, (a, b) in enumerate(zip(in_dims, out_dims)) if b == 1 and a != 1)
    return x.sum(axis=axes, keepdims=True).reshape(out_dims) if axes else x.reshape(out_dims).copy()


# ---- softmax family (src/gpu_op.cu:237-301, 3238-3248, 3521) -------------------------------------------
def softmax_rows(x):
    z = x - x.max(axis=1, keepdims=True)
    e = np.exp(z)
    return e / e.sum(axis=1, keepdims=True)


def softmax_cross_entropy(logits, labels):
    """mean over rows of -sum(labels * log softmax(logits)); shape (1,) (autodiff.py:700-704)."""
    z = logits - logits.max(axis=1, keepdims=True)
    logsm = z - np.log(np.exp(z).sum(axis=1, keepdims=True))
    return np.array([np.mean(-np.sum(labels * logsm, axis=1))], dtype=logits.dtype)


def softmax_instance(x):
    """Softmax over all non-batch elements of each sample (CUDNN_SOFTMAX_MODE_INSTANCE)."""
    return softmax_rows(x.reshape(x.shape[0], -1)).reshape(x.shape)


def softmax_instance_bwd(y, dy):
    y2, d2 = y.reshape(y.shape[0], -1), dy.reshape(y.shape[0], -1)
    return (y2 * (d2 - (d2 * y2).sum(axis=1, keepdims=True))).reshape(y.shape)


def cross(x, y, b):
    """-log(x) * y * b  (src/gpu_op.cu:4538-4543)."""
    return np.log(x) * y * (-1) * b


def cross_backward(x, y, dout, b):
    """-y * b / x * dout  (src/gpu_op.cu:4568-4573)."""
    return y * (-1) * b * (1.0 / x) * dout


# ---- elementwise losses and their reductions (src/gpu_op.cu:3693-3870, 3880-4106) ------------------------
def binary_cross_entropy_terms(a, b):
    """b*log(a) + (1-b)*log(1-a) per element (matrix_cross_entropy_kernel, src/gpu_op.cu:3693-3718; no sign, no sum)."""
    return b * np.log(a) + (1 - b) * np.log(1 - a)


def l1_loss(a, b):
    """mean over rows of sum_cols |b - a|  (matrix_l1loss_kernel, src/gpu_op.cu:3719-3745)."""
    return np.array([np.abs(b - a).reshape(a.shape[0], -1).sum(axis=1).mean()])


def l2_loss(a, b):
    """half the mean over rows of sum_cols (b - a)^2  (matrix_l2loss_kernel, src/gpu_op.cu:3746-3773)."""
    return np.array([((b - a) ** 2).reshape(a.shape[0], -1).sum(axis=1).mean() / 2])


def l1_loss_grad(a, b, g):
    """sign(a - b) * g[0] / rows, with sign(0) = -1  (matrix_l1lossgradient_kernel, src/gpu_op.cu:3774-3779)."""
    return np.where((a - b) > 0, g.reshape(-1)[0] / a.shape[0], -g.reshape(-1)[0] / a.shape[0])


def l2_loss_grad(a, b, g):
    """(a - b) * g[0] / rows  (matrix_l2lossgradient_kernel, src/gpu_op.cu:3780-3785)."""
    return (a - b) * g.reshape(-1)[0] / a.shape[0]


def l1_regular(a):
    return l1_loss(np.zeros_like(a), a)


def l2_regular(a):
    return l2_loss(np.zeros_like(a), a)


def l1_regular_grad(a, g):
    return l1_loss_grad(a, np.zeros_like(a), g)


def l2_regular_grad(a, g):
    return l2_loss_grad(a, np.zeros_like(a), g)


# ---- convolution: NCHW cross-correlation, symmetric zero padding, dilation 1 -----------------------------
def conv_out_extent(n, k, pad, stride):
    return 1 + (n + 2 * pad - k) // stride


def conv_geometry(x_shape, w_shape, padding, sh, sw):
    """pad = k // 2 on both sides for SAME, 0 for VALID (src/gpu_op.cu:2081-2087)."""
    N, C, H, W = x_shape
    K, C2, R, S = w_shape
    assert C == C2
    ph, pw = (R // 2, S // 2) if padding == "SAME" else (0, 0)
    return dict(N=N, C=C, H=H, W=W, K=K, R=R, S=S, ph=ph, pw=pw, sh=sh, sw=sw,
                P=conv_out_extent(H, R, ph, sh), Q=conv_out_extent(W, S, pw, sw))


def _im2col(x, g):
    """(N, C*R*S, P*Q) view-based patch matrix of the zero-padded input."""
    xp = np.pad(x, ((0, 0), (0, 0), (g["ph"], g["ph"]), (g["pw"], g["pw"])))
    N, C = x.shape[:2]
    s = xp.strides
    win = np.lib.stride_tricks.as_strided(
        xp, shape=(N, C, g["R"], g["S"], g["P"], g["Q"]),
        strides=(s[0], s[1], s[2], s[3], s[2] * g["sh"], s[3] * g["sw"]), writeable=False)
    return win.reshape(N, C * g["R"] * g["S"], g["P"] * g["Q"])


def conv2d_fwd(x, w, g):
    """y[n,k,p,q] = sum_{c,r,s} x[n,c,p*sh+r-ph,q*sw+s-pw] * w[k,c,r,s]  (cudnnConvolutionForward, src/gpu_op.cu:2019)."""
    cols = _im2col(x, g)
    y = np.matmul(w.reshape(g["K"], -1)[None], cols)
    return y.reshape(g["N"], g["K"], g["P"], g["Q"])


def conv2d_wgrad(x, dy, g):
    """dw[k,c,r,s] = sum_{n,p,q} dy[n,k,p,q] * x[n,c,p*sh+r-ph,q*sw+s-pw]  (src/gpu_op.cu:1716)."""
    cols = _im2col(x, g)                                  # (N, CRS, PQ)
    d = dy.reshape(g["N"], g["K"], -1)                    # (N, K, PQ)
    dw = np.matmul(d, cols.transpose(0, 2, 1)).sum(axis=0)
    return dw.reshape(g["K"], g["C"], g["R"], g["S"])


def conv2d_dgrad(dy, w, g):
    """dx = transposed correlation of dy with w, stride-aware  (src/gpu_op.cu:1804)."""
    N, C, H, W = g["N"], g["C"], g["H"], g["W"]
    d = dy.reshape(N, g["K"], -1)
    cols = np.matmul(w.reshape(g["K"], -1).T[None], d)    # (N, CRS, PQ)
    cols = cols.reshape(N, C, g["R"], g["S"], g["P"], g["Q"])
    dxp = np.zeros((N, C, H + 2 * g["ph"], W + 2 * g["pw"]), dtype=dy.dtype)
    for r in range(g["R"]):
        for s in range(g["S"]):
            dxp[:, :, r:r + g["sh"] * g["P"]:g["sh"], s:s + g["sw"] * g["Q"]:g["sw"]] += cols[:, :, r, s]
    return dxp[:, :, g["ph"]:g["ph"] + H, g["pw"]:g["pw"] + W].copy()


# The three convolution passes at chosen output coordinates only: direct float64 dot products, cheap at any
# tensor size.  Same formulas as the dense functions above (tests/test_oracle.py holds them to those).
def conv2d_fwd_at(x, w, g, n, k, p, q):
    """y[n,k,p,q] for index vectors n, k, p, q (each of length T)."""
    C, R, S = g["C"], g["R"], g["S"]
    r, s = np.meshgrid(np.arange(R), np.arange(S), indexing="ij")
    i = p[:, None, None] * g["sh"] + r[None] - g["ph"]                    # (T, R, S)
    j = q[:, None, None] * g["sw"] + s[None] - g["pw"]
    ok = (i >= 0) & (i < g["H"]) & (j >= 0) & (j < g["W"])
    xs = x[n[:, None, None, None], np.arange(C)[None, :, None, None], np.clip(i, 0, g["H"] - 1)[:, None], np.clip(j, 0, g["W"] - 1)[:, None]]
    xs = np.where(ok[:, None], xs, 0).astype(np.float64)                   # (T, C, R, S)
    return np.einsum("tcrs,tcrs->t", xs, w[k].astype(np.float64))


def conv2d_dgrad_at(dy, w, g, n, c, h, wi):
    """dx[n,c,h,wi] = sum_{k,r,s} dy[n,k,p,q] * w[k,c,r,s] over the (p, q) with p*sh + r - ph = h, q*sw + s - pw = wi."""
    R, S, K = g["R"], g["S"], g["K"]
    r, s = np.meshgrid(np.arange(R), np.arange(S), indexing="ij")
    pn = h[:, None, None] + g["ph"] - r[None]                             # p * sh
    qn = wi[:, None, None] + g["pw"] - s[None]
    p, q = pn // g["sh"], qn // g["sw"]
    ok = (pn % g["sh"] == 0) & (qn % g["sw"] == 0) & (p >= 0) & (p < g["P"]) & (q >= 0) & (q < g["Q"])
    d = dy[n[:, None, None, None], np.arange(K)[None, :, None, None], np.clip(p, 0, g["P"] - 1)[:, None], np.clip(q, 0, g["Q"] - 1)[:, None]]
    d = np.where(ok[:, None], d, 0).astype(np.float64)                     # (T, K, R, S)
    wk = w[:, c].astype(np.float64).transpose(1, 0, 2, 3)                  # (T, K, R, S)
    return np.einsum("tkrs,tkrs->t", d, wk)


def conv2d_wgrad_at(x, dy, g, k, c, r, s):
    """dw[k,c,r,s] = sum_{n,p,q} dy[n,k,p,q] * x[n,c,p*sh+r-ph,q*sw+s-pw] for index vectors k, c, r, s."""
    out = np.empty(len(k), np.float64)
    pp, qq = np.arange(g["P"]), np.arange(g["Q"])
    for t in range(len(k)):
        i, j = pp * g["sh"] + r[t] - g["ph"], qq * g["sw"] + s[t] - g["pw"]
        oi, oj = (i >= 0) & (i < g["H"]), (j >= 0) & (j < g["W"])
        xs = x[:, c[t]][:, i[oi]][:, :, j[oj]].astype(np.float64)
        ds = dy[:, k[t]][:, oi][:, :, oj].astype(np.float64)
        out[t] = np.vdot(xs, ds)
    return out


# ---- pooling (cudnnPoolingForward / Backward as configured at src/gpu_op.cu:2880-3028) ---------------------
def pool_geometry(x_shape, ph, pw, sh, sw, kh, kw):
    N, C, H, W = x_shape
    return dict(N=N, C=C, H=H, W=W, ph=ph, pw=pw, sh=sh, sw=sw, kh=kh, kw=kw,
                P=1 + (H + 2 * ph - kh) // sh, Q=1 + (W + 2 * pw - kw) // sw)


def _pool_windows(x, g, fill):
    xp = np.pad(x, ((0, 0), (0, 0), (g["ph"], g["ph"]), (g["pw"], g["pw"])), constant_values=fill)
    s = xp.strides
    return np.lib.stride_tricks.as_strided(
        xp, shape=(g["N"], g["C"], g["P"], g["Q"], g["kh"], g["kw"]),
        strides=(s[0], s[1], s[2] * g["sh"], s[3] * g["sw"], s[2], s[3]), writeable=False)


def maxpool_fwd(x, g):
    """Returns (y, idx): idx is the flat h*W+w position of the first maximum in the input plane, -1 for an all-padding window."""
    win = _pool_windows(x, g, -np.inf).reshape(g["N"], g["C"], g["P"], g["Q"], -1)
    arg = win.argmax(axis=-1)                              # first maximum in row-major window order
    y = np.take_along_axis(win, arg[..., None], axis=-1)[..., 0]
    r, s = arg // g["kw"], arg % g["kw"]
    h = np.arange(g["P"])[:, None] * g["sh"] - g["ph"] + r
    w = np.arange(g["Q"])[None, :] * g["sw"] - g["pw"] + s
    idx = (h * g["W"] + w).astype(np.int32)
    empty = ~np.isfinite(y) & (y < 0)                      # window made of padding only
    idx = np.where(empty, -1, idx).astype(np.int32)
    y = np.where(empty, 0, y).astype(x.dtype)
    return y, idx


def maxpool_bwd(x, dy, g):
    _, idx = maxpool_fwd(x, g)
    dx = np.zeros((g["N"], g["C"], g["H"] * g["W"]), dtype=dy.dtype)
    flat_idx = idx.reshape(g["N"], g["C"], -1)
    d = dy.reshape(g["N"], g["C"], -1)
    valid = flat_idx >= 0
    n_i, c_i, _ = np.nonzero(valid)
    np.add.at(dx, (n_i, c_i, flat_idx[valid]), d[valid])
    return dx.reshape(g["N"], g["C"], g["H"], g["W"])


def avgpool_fwd(x, g):
    win = _pool_windows(x, g, 0.0)
    return (win.sum(axis=(-1, -2)) / (g["kh"] * g["kw"])).astype(x.dtype)


def avgpool_bwd(dy, g):
    dxp = np.zeros((g["N"], g["C"], g["H"] + 2 * g["ph"], g["W"] + 2 * g["pw"]), dtype=dy.dtype)
    share = dy / (g["kh"] * g["kw"])
    for r in range(g["kh"]):
        for s in range(g["kw"]):
            dxp[:, :, r:r + g["sh"] * g["P"]:g["sh"], s:s + g["sw"] * g["Q"]:g["sw"]] += share
    return dxp[:, :, g["ph"]:g["ph"] + g["H"], g["pw"]:g["pw"] + g["W"]].copy()


# ---- 3-D convolution (forward) and pooling: NCDHW, same conventions as the 2-D functions -------------------------------
def conv3d_fwd(x, w, pads, strides):
    """y[n,k,o,p,q] = sum_{c,t,r,s} x[n,c,o*sd+t-pd,p*sh+r-ph,q*sw+s-pw] * w[k,c,t,r,s]  (cudnnConvolutionForward on the
    Nd descriptors of src/gpu_op.cu:2431-2527)."""
    N, C, D, H, W = x.shape
    K, _, T, R, S = w.shape
    (pd, ph, pw), (sd, sh, sw) = pads, strides
    Od, P, Q = conv_out_extent(D, T, pd, sd), conv_out_extent(H, R, ph, sh), conv_out_extent(W, S, pw, sw)
    xp = np.pad(x, ((0, 0), (0, 0), (pd, pd), (ph, ph), (pw, pw)))
    y = np.zeros((N, K, Od, P, Q), dtype=x.dtype)
    for t in range(T):
        for r in range(R):
            for s in range(S):
                patch = xp[:, :, t:t + sd * Od:sd, r:r + sh * P:sh, s:s + sw * Q:sw]
                y += np.einsum("ncopq,kc->nkopq", patch, w[:, :, t, r, s])
    return y


def _pool3d_windows(x, pads, strides, window, fill):
    N, C, D, H, W = x.shape
    (pd, ph, pw), (sd, sh, sw), (kd, kh, kw) = pads, strides, window
    Od, P, Q = conv_out_extent(D, kd, pd, sd), conv_out_extent(H, kh, ph, sh), conv_out_extent(W, kw, pw, sw)
    xp = np.pad(x, ((0, 0), (0, 0), (pd, pd), (ph, ph), (pw, pw)), constant_values=fill)
    s = xp.strides
    win = np.lib.stride_tricks.as_strided(xp, shape=(N, C, Od, P, Q, kd, kh, kw),
                                          strides=(s[0], s[1], s[2] * sd, s[3] * sh, s[4] * sw, s[2], s[3], s[4]), writeable=False)
    return win, (Od, P, Q)


def pool3d_fwd(x, mode, pads, strides, window):
    """Max (padding ignored, an all-padding window gives 0) or average over the full window, padding counted."""
    if mode == "max":
        win, _ = _pool3d_windows(x, pads, strides, window, -np.inf)
        y = win.reshape(win.shape[:5] + (-1,)).max(axis=-1)
        return np.where(np.isneginf(y), 0, y).astype(x.dtype)
    win, _ = _pool3d_windows(x, pads, strides, window, 0)
    return win.reshape(win.shape[:5] + (-1,)).sum(axis=-1) / float(np.prod(window))


def pool3d_bwd(x, dy, mode, pads, strides, window):
    """Gradient of pool3d_fwd: max pooling routes dy to the first maximum of each window in (depth, row, column) order."""
    N, C, D, H, W = x.shape
    (pd, ph, pw), (sd, sh, sw), (kd, kh, kw) = pads, strides, window
    dxp = np.zeros((N, C, D + 2 * pd, H + 2 * ph, W + 2 * pw), dtype=dy.dtype)
    if mode == "max":
        win, (Od, P, Q) = _pool3d_windows(x, pads, strides, window, -np.inf)
        arg = win.reshape(win.shape[:5] + (-1,)).argmax(axis=-1)            # first maximum
        valid = ~np.isneginf(win.reshape(win.shape[:5] + (-1,)).max(axis=-1))
        t, rem = np.divmod(arg, kh * kw)
        r, s = np.divmod(rem, kw)
        n, c, o, p, q = np.meshgrid(np.arange(N), np.arange(C), np.arange(Od), np.arange(P), np.arange(Q), indexing="ij")
        np.add.at(dxp, (n[valid], c[valid], (o * sd + t)[valid], (p * sh + r)[valid], (q * sw + s)[valid]), dy[valid])
    else:
        Od, P, Q = dy.shape[2:]
        for t in range(kd):
            for r in range(kh):
                for s in range(kw):
                    dxp[:, :, t:t + sd * Od:sd, r:r + sh * P:sh, s:s + sw * Q:sw] += dy / float(kd * kh * kw)
    return dxp[:, :, pd:pd + D, ph:ph + H, pw:pw + W].copy()


# ---- batch normalisation, scale 1 / bias 0 / eps 1e-5 / batch statistics (src/gpu_op.cu:4224-4460) ----------
def _bn_axes(x, mode):
    # per-activation: statistics over the batch axis only; spatial: over batch and all spatial axes
    return (0,) if mode == "pre_activation" else (0,) + tuple(range(2, x.ndim))


def bn_fwd(x, mode):
    ax = _bn_axes(x, mode)
    mean = x.mean(axis=ax, keepdims=True)
    var = ((x - mean) ** 2).mean(axis=ax, keepdims=True)
    inv = 1.0 / np.sqrt(var + x.dtype.type(BN_EPS))
    return ((x - mean) * inv).astype(x.dtype), mean, inv


def bn_bwd(x, dy, mode):
    ax = _bn_axes(x, mode)
    _, mean, inv = bn_fwd(x, mode)
    xh = (x - mean) * inv
    return (inv * (dy - dy.mean(axis=ax, keepdims=True) - xh * (dy * xh).mean(axis=ax, keepdims=True))).astype(x.dtype)


# ---- concat along axis 1 (src/gpu_op.cu:967-1088) ---------------------------------------------------------------
def concat(a, b):
    return np.concatenate([a, b], axis=1)


def concat_split(a_shape, dout, which):
    ca = a_shape[1]
    return dout[:, :ca].copy() if which == 0 else dout[:, ca:].copy()


# ---- dropout: same counter-based mask as the CUDA kernel -----------------------------------------------------------
def dropout_uniform(seed, n):
    """u[i] in [0,1): top 24 bits of a splitmix64-style mix of (i+1) keyed by the seed."""
    with np.errstate(over="ignore"):
        i = np.arange(1, n + 1, dtype=np.uint64)
        z = i * np.uint64(0x9E3779B97F4A7C15) + np.uint64(seed) * np.uint64(0xD1342543DE82EF95)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        z = z ^ (z >> np.uint64(31))
    return (z >> np.uint64(40)).astype(np.float32) * np.float32(1.0 / 16777216.0)


def dropout(x, p, seed):
    keep = dropout_uniform(seed, x.size).reshape(x.shape) >= np.float32(p)
    scale = x.dtype.type(np.float32(1.0) / (np.float32(1.0) - np.float32(p)))
    return np.where(keep, x * scale, 0).astype(x.dtype)


# ---- optimisers (src/gpu_op.cu:4461-4507, 4600-4605) ------------------------------------------------------------------
def sgd(w, g, lr):
    return w - w.dtype.type(lr) * g


def adam(w, m, v, g, b1, b2, b1t, b2t, e, lr):
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    w = w - lr * m / (1 - b1t) / (np.sqrt(v / (1 - b2t)) + e)
    return w, m, v


# ---- layer normalisation and the gated dense layer (no counterpart in the reference) ---------------
def layer_norm(x, gamma, beta, eps):
    """(y, normalised x, 1 / spread) over the last axis."""
    mean = x.mean(axis=-1, keepdims=True)
    inv = 1 / np.sqrt(((x - mean) ** 2).mean(axis=-1, keepdims=True) + eps)
    xh = (x - mean) * inv
    return gamma * xh + beta, xh, inv


def layer_norm_backward(x, gamma, dy, eps):
    """(dx, dgamma, dbeta)"""
    _, xh, inv = layer_norm(x, gamma, 0, eps)
    g = gamma * dy
    dx = inv * (g - g.mean(axis=-1, keepdims=True) - xh * (g * xh).mean(axis=-1, keepdims=True))
    axes = tuple(range(x.ndim - 1))
    return dx, (dy * xh).sum(axis=axes), dy.sum(axis=axes)


def gate(activation, g):
    """(value, derivative) of the activation of a gated layer."""
    if activation == "relu":
        return np.where(g > 0, g, 0), np.where(g > 0, 1.0, 0.0)
    if activation == "tanh":
        return np.tanh(g), 1 / np.cosh(np.clip(g, -300, 300)) ** 2
    if activation == "gelu":
        from scipy.special import erfc
        share = 0.5 * erfc(-g / np.sqrt(2))
        return g * share, share + g * np.exp(-g * g / 2) / np.sqrt(2 * np.pi)
    from scipy.special import expit
    s, rest = expit(g), expit(-g)
    return (s, s * rest) if activation == "sigmoid" else (g * s, s * (1 + g * rest))


def gated_linear(x, weight, activation):
    """(out, both projections)"""
    z = x @ weight
    half = weight.shape[1] // 2
    return gate(activation, z[:, :half])[0] * z[:, half:], z


def gated_linear_backward(x, weight, z, dout, activation):
    """(dx, dweight)"""
    half = weight.shape[1] // 2
    value, slope = gate(activation, z[:, :half])
    dz = np.concatenate([dout * z[:, half:] * slope, dout * value], axis=1)
    return dz @ weight.T, x.T @ dz
