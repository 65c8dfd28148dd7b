"""Attention on every kernel and with every way of cutting the keys (test_cache_plan.py checks that these sizes reach them)."""
import numpy as np
import pytest

from cache_reference import Case
from cache_routes import ROUTES, width
from shim import q8_cache as C
from test_gpu_cache_attention import check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    with C.Ops() as o:
        yield o


@pytest.mark.parametrize("name", list(ROUTES))
def test_attention(ops, name):
    dtype, sequences, heads, kv_heads, dim, page, longest, _ = ROUTES[name]
    case = Case(np.random.default_rng(len(name)), sequences, heads, kv_heads, dim, page, longest=longest)
    assert case.width == width(sequences, page) and case.tokens == sum(n for n, _ in sequences)
    check(ops, np.random.default_rng(3), case, dtype)


def test_more_sequences_than_a_wave(ops):
    """Tiles are found over sequences, 64 at a time: 300 of them, some empty, few rows and many."""
    rng = np.random.default_rng(11)
    sequences = [(int(n), int(n) + int(t)) for n, t in zip(rng.choice([0, 1, 1, 1, 5, 40], 300), rng.integers(0, 90, 300))]
    case = Case(rng, sequences, 4, 2, 64, 16, extra_rows=2, front_rows=1)
    check(ops, rng, case, "bf16")
