"""What the gated layer's calls refuse, before anything touches a device (the arrays here are only described)."""
import pytest

from tests.test_norm_refusals import MB, described, op, refused  # noqa: F401

M, K, F = 6, 10, 8
SHAPES = {"x": (M, K), "w": (K, 2 * F), "z": (M, 2 * F), "h": (M, F), "d": (M, F), "dx": (M, K), "dw": (K, 2 * F)}
USED = {"forward": ("x", "w", "z", "h"), "backward": ("x", "w", "z", "d", "dx", "dw")}
WRITTEN = {"forward": ("z", "h"), "backward": ("dx", "dw")}


def arrays(**changed):
    a = {n: described(s, (1 + i) * MB) for i, (n, s) in enumerate(SHAPES.items())}
    a.update(changed)
    return a


def call(op, which, a, activation="silu"):
    if which == "forward":
        return lambda: op.gated_linear_forward(a["x"], a["w"], a["z"], a["h"], activation, None)
    return lambda: op.gated_linear_backward(a["x"], a["w"], a["z"], a["d"], a["dx"], a["dw"], activation, None)


@pytest.mark.parametrize("which", ["forward", "backward"])
def test_refusals(op, which):
    for name in USED[which]:
        at = (1 + list(SHAPES).index(name)) * MB
        shape = SHAPES[name]
        for other, words in ((described(shape, at, kind=1), "not on the GPU"), (described(shape, at, device=1), "another GPU"), (described(shape, 0), "no memory"),
                             (described(shape, at + 2), "not aligned"), (described((shape[0] + 1, shape[1]), at), "has to be|differ"),
                             (described((shape[0] * shape[1],), at), "has to be|have to be"), (described((shape[1], shape[0]), at), "has to be|differ")):
            refused(call(op, which, arrays(**{name: other})), words)
    for out in WRITTEN[which]:
        for name in USED[which]:
            if name != out:
                refused(call(op, which, arrays(**{out: described(SHAPES[out], (1 + list(SHAPES).index(name)) * MB + 4)})), "shares memory")
    odd = {n: described((s[0], 2 * F - 1), (20 + i) * MB) for i, (n, s) in enumerate(SHAPES.items()) if s[1] == 2 * F}
    refused(call(op, which, arrays(**odd)), "odd")
    with pytest.raises(AssertionError, match="unknown option"):
        call(op, which, arrays(), "softmax")()
    from tinyflow_b200._base import _LIB, last_error
    for bad in (3, -1, 6):
        a = arrays()
        if which == "forward":
            rc = _LIB.TfGatedLinearForward(a["x"].handle, a["w"].handle, a["z"].handle, a["h"].handle, bad, None, None)
        else:
            rc = _LIB.TfGatedLinearBackward(a["x"].handle, a["w"].handle, a["z"].handle, a["d"].handle, a["dx"].handle, a["dw"].handle, bad, None, None)
        assert rc == -1 and "activation" in last_error()
