"""What the calls of rotation, normed heads and attention refuse, before anything touches a device (the arrays here are only described)."""
import ctypes

import pytest

from tests.test_norm_refusals import MB, described, op, refused  # noqa: F401

H, G, D, B, TQ, TK = 6, 2, 10, 2, 4, 7
SHAPES = {"q": (B * TQ, H * D), "k": (B * TK, G * D), "v": (B * TK, G * D), "documents": (B * TK,), "prefix": (B,), "slopes": (H,), "out": (B * TQ, H * D), "stats": (B, H, TQ, 2),
          "dout": (B * TQ, H * D), "dq": (B * TQ, H * D), "dk": (B * TK, G * D), "dv": (B * TK, G * D)}
USED = {"forward": ("q", "k", "v", "documents", "prefix", "slopes", "out", "stats"), "backward": tuple(SHAPES)}
WRITTEN = {"forward": ("out", "stats"), "backward": ("dq", "dk", "dv")}


def arrays(**changed):
    a = {n: described(s, (1 + i) * MB) for i, (n, s) in enumerate(SHAPES.items())}
    a.update(changed)
    return a


def attention(op, which, a, state=None):
    state = state or op.attention_state(TQ, H, G)
    if which == "forward":
        return lambda: op.attention_forward(a["q"], a["k"], a["v"], a["documents"], a["prefix"], a["slopes"], a["out"], a["stats"], state, None)
    return lambda: op.attention_backward(*(a[n] for n in SHAPES), state, None)


@pytest.mark.parametrize("which", ["forward", "backward"])
def test_attention_arrays(op, which):
    for name in USED[which]:
        at, shape = (1 + list(SHAPES).index(name)) * MB, SHAPES[name]
        for other, words in ((described(shape, at, kind=1), "not on the GPU"), (described(shape, at, device=1), "another GPU"), (described(shape, 0), "no memory"),
                             (described(shape, at + 2), "not aligned"), (described((shape[0] + 1,) + shape[1:], at), "size|sequences|tokens|have to")):
            refused(attention(op, which, arrays(**{name: other})), words)
    for out in WRITTEN[which]:
        for name in USED[which]:
            if name != out:
                refused(attention(op, which, arrays(**{out: described(SHAPES[out], (1 + list(SHAPES).index(name)) * MB)})), "shares memory")
    for name in ("q", "k", "v"):
        rows, cols = SHAPES[name]
        refused(attention(op, which, arrays(**{name: described((rows, cols + 1), MB * 30)})), "heads")
        refused(attention(op, which, arrays(**{name: described((rows * cols,), MB * 30)})), "matrices")
    # more queries than keys with documents
    few = {n: described((B * 3,) + SHAPES[n][1:], 30 * MB + i * MB) for i, n in enumerate(("k", "v", "documents", "dk", "dv"))}
    refused(attention(op, which, arrays(**few)), "documents")
    wide = {n: described((s[0], s[1] // D * 257), 30 * MB + i * MB) for i, (n, s) in enumerate(SHAPES.items()) if len(s) == 2}
    refused(attention(op, which, arrays(**wide)), "1 to 256")


def test_attention_states(op):
    from tinyflow_b200._base import new_cell
    for bad, words in ((dict(length=0), "at least one query"), (dict(heads=5), "do not share"), (dict(kv_heads=0), "do not share"), (dict(window=-1), "window"),
                       (dict(scale=float("nan")), "scale"), (dict(cap=-1.0), "cap"), (dict(cap=float("inf")), "cap")):
        arguments = dict(length=4, heads=6, kv_heads=2)
        arguments.update(bad)
        refused(lambda: op.attention_state(**arguments), words)
    refused(lambda: op.attention_state(4, 2, 2, state=op.rotary_state(8)), "another descriptor")
    refused(lambda: op.rotary_state(8, state=op.attention_state(4, 2, 2)), "another descriptor")
    for which in ("forward", "backward"):
        refused(attention(op, which, arrays(), state=new_cell(3)), "TfAttentionState")
        refused(attention(op, which, arrays(), state=op.rotary_state(8)), "TfAttentionState")
        refused(attention(op, which, arrays(), state=op.attention_state(3, H, G)), "sequences of 3")
        refused(attention(op, which, arrays(), state=op.attention_state(TQ, 7, 7)), "heads")


T, QH, KH, RD = 12, 3, 2, 8
HEADS = {"q": (T, QH * RD), "k": (T, KH * RD), "gq": (RD,), "gk": (RD,), "at": (T,), "yq": (T, QH * RD), "yk": (T, KH * RD), "dyq": (T, QH * RD), "dyk": (T, KH * RD),
         "dq": (T, QH * RD), "dk": (T, KH * RD), "dgq": (RD,), "dgk": (RD,)}
CALLS = {"rotate": ("q", "at", "yq"), "back": ("dyq", "at", "dq"), "norm": ("q", "k", "gq", "gk", "at", "yq", "yk"),
         "norm back": ("q", "k", "gq", "gk", "at", "dyq", "dyk", "dq", "dk", "dgq", "dgk")}
RESULTS = {"rotate": ("yq",), "back": ("dq",), "norm": ("yq", "yk"), "norm back": ("dq", "dk", "dgq", "dgk")}


def heads(op, which, state=None, length=4, start=0, eps=1e-6, **changed):
    a = {n: described(s, (1 + i) * MB) for i, (n, s) in enumerate(HEADS.items())}
    a.update(changed)
    state = state or op.rotary_state(RD)
    given = [a[n] for n in CALLS[which]]
    if which == "rotate":
        return lambda: op.rotary_forward(*given, length, start, state, None)
    if which == "back":
        return lambda: op.rotary_backward(*given, length, start, state, None)
    if which == "norm":
        return lambda: op.head_norm_rotary_forward(*given, length, start, eps, state, None)
    return lambda: op.head_norm_rotary_backward(*given, length, start, eps, state, None)


@pytest.mark.parametrize("which", list(CALLS))
def test_heads_arrays(op, which):
    from tinyflow_b200._base import new_cell
    for name in CALLS[which]:
        at, shape = (1 + list(HEADS).index(name)) * MB, HEADS[name]
        for other, words in ((described(shape, at, kind=1), "not on the GPU"), (described(shape, at, device=1), "another GPU"), (described(shape, 0), "no memory"),
                             (described(shape, at + 1), "not aligned"), (described((shape[0] + 1,) + shape[1:], at), "size|tokens")):
            refused(heads(op, which, **{name: other}), words)
    for out in RESULTS[which]:
        for name in CALLS[which]:
            if name != out:
                refused(heads(op, which, **{out: described(HEADS[out], (1 + list(HEADS).index(name)) * MB)}), "shares memory")
    first = CALLS[which][0]
    refused(heads(op, which, **{first: described((T, QH * RD + 1), 40 * MB)}), "not heads of 8")
    refused(heads(op, which, **{first: described((T * QH * RD,), 40 * MB)}), "matrix")
    refused(heads(op, which, length=0), "length")
    refused(heads(op, which, start=-1), "start")
    refused(heads(op, which, state=new_cell(3)), "TfRotaryState")
    if which.startswith("norm"):
        refused(heads(op, which, eps=-1.0), "eps")
        refused(heads(op, which, eps=float("nan")), "eps")
        refused(heads(op, which, k=None), "go together")
        refused(heads(op, which, gk=None), "go together")


def test_rotary_states(op):
    from tinyflow_b200._base import _LIB, TinyflowError, check_call, new_cell
    for arguments, words in (((0,), "1 to 256"), ((257,), "1 to 256"), ((8, 10), "do not fit")):
        refused(lambda: op.rotary_state(*arguments), words)
    f = (ctypes.c_double * 2)(1.0, float("nan"))
    with pytest.raises(TinyflowError, match="frequency 1"):
        check_call(_LIB.TfRotaryState(8, 2, 0, f, ctypes.c_float(1.0), new_cell(3)))
    with pytest.raises(TinyflowError, match="layout"):
        check_call(_LIB.TfRotaryState(8, 1, 2, f, ctypes.c_float(1.0), new_cell(3)))
    with pytest.raises(TinyflowError, match="amplitude"):
        check_call(_LIB.TfRotaryState(8, 1, 0, f, ctypes.c_float(float("inf")), new_cell(3)))
    for bad in (dict(layout="quarter"), dict(scaling="square"), dict(rotated=7), dict(scaling="parts"), dict(factor=0.0, scaling="linear")):
        with pytest.raises(AssertionError):
            op.rotary_state(8, **bad)


def test_frequencies(op):
    f, amplitude = op.rotary_frequencies(8, 10000.0)
    assert amplitude == 1.0 and f == [10000.0 ** (-2.0 * i / 8) for i in range(4)]
    assert op.rotary_frequencies(8, 10000.0, "linear", 4.0)[0] == [v / 4 for v in f]
    stretched = op.rotary_frequencies(8, 10000.0, "stretched", 4.0)[0]
    assert stretched[0] == 1.0 and abs(stretched[-1] / f[-1] - 0.25) < 1e-12
    parts, amplitude = op.rotary_frequencies(64, 10000.0, "parts", 4.0, 4096)
    plain = op.rotary_frequencies(64, 10000.0)[0]
    assert parts[0] == plain[0] and abs(parts[-1] - plain[-1] / 4) < 1e-18 and amplitude > 1
    assert all(p / 4 <= v <= p for p, v in zip(plain, parts)) and op.rotary_frequencies(0) == ([], 1.0)
