"""Numbers of the states that do not fit the library's, which would arrive as others: 2^32 + 5 as a window of 5."""
import pytest

from tests.test_norm_refusals import op  # noqa: F401


@pytest.mark.parametrize("name", ["heads", "kv_heads", "window"])
@pytest.mark.parametrize("value", [2 ** 32 + 2, 2 ** 31, -2 ** 32 + 2])
def test_attention_states(op, name, value):
    with pytest.raises(AssertionError, match="32 bits"):
        op.attention_state(**dict(dict(length=4, heads=2, kv_heads=2, window=0), **{name: value}))


def test_the_largest_window(op):
    op.attention_state(4, 2, 2, window=2 ** 31 - 1)


def test_rotary_states(op):
    with pytest.raises(AssertionError, match="32 bits"):
        op.rotary_state(2 ** 32 + 8, 8)
