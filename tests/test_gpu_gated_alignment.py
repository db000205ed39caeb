"""Gated layers whose arrays lie differently between 16-byte boundaries: every access width is chosen from the arrays that it serves.
Checks and tolerances are those of test_gpu_gated."""
import pytest

from tests import test_gpu_gated
from tests.test_gpu_norm import place
from tests.test_gpu_ops import env  # noqa: F401

pytestmark = pytest.mark.gpu
# floats behind a boundary: input, weight, gradient of the output; projections, output, output again, gradients of the input and of the weight
PLACES = [(1, 0, 0, 0, 0, 0, 0, 0), (0, 2, 0, 0, 0, 0, 0, 0), (0, 0, 3, 0, 0, 0, 0, 0), (0, 0, 0, 1, 0, 0, 0, 0), (0, 0, 0, 0, 3, 2, 0, 0), (0, 0, 0, 0, 0, 0, 1, 2), (2, 2, 2, 2, 2, 2, 2, 2), (3, 1, 2, 2, 1, 0, 3, 1)]
# one row and few against large weights, small layers, the tensor cores with whole and ragged tiles, with clusters, elementwise kernels apart
SHAPES = [(1, 1024, 1024), (1, 622, 4026), (8, 1024, 1024), (3, 700, 1002), (16, 1024, 1024), (12, 1000, 1004), (40, 96, 64), (64, 200, 132), (700, 512, 520), (777, 500, 1002), (300, 520, 500), (3000, 64, 32), (1300, 768, 1536)]


@pytest.mark.parametrize("at", PLACES)
@pytest.mark.parametrize("M,K,F", SHAPES)
def test_arrays_apart(env, monkeypatch, M, K, F, at):
    offsets = iter(at)
    monkeypatch.setattr(test_gpu_gated, "place", lambda env, value, misaligned: place(env, value, next(offsets)))
    test_gpu_gated.check(env, M, K, F, "silu", misaligned=None)


@pytest.mark.parametrize("at", PLACES)
@pytest.mark.parametrize("path", [1, 2])
def test_arrays_apart_on_each_engine(env, monkeypatch, at, path):
    offsets = iter(at)
    monkeypatch.setattr(test_gpu_gated, "place", lambda env, value, misaligned: place(env, value, next(offsets)))
    test_gpu_gated.check(env, 400, 300, 600, "gelu", misaligned=None, path=path)
