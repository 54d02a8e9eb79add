"""Sizes next to the entry points' limits, which the counting behind them has to hold: refused, or planned
for as smaller ones are, before any launch (CPU)."""
import pytest

from needle_amd import _lib

P = 1 << 20      # an aligned stand-in address that is never dereferenced
MOST = (1 << 31) - 1


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_budgets_that_are_counted_past_31_bits(lib):
    """A workgroup's threads step 1,024 entries on from the last ones of a list."""
    for budget in (0x7fff0001, MOST - 1024, MOST):
        assert lib.ndl_kv_select(P, P, P, 4, 2, 16, P, 8, 8, P, 3, budget, 4, 8, None) == -2, budget
