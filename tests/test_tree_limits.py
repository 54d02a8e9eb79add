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


def test_grids_of_the_weights(lib):
    """The weights of every 256 keys of a kv head take a workgroup of 512 threads where scores are not
    kept; a grid's threads are counted in 32 bits, and a larger one loses the rest without an error."""
    def weigh(blocks_per_head, hkv):
        w = 16 * blocks_per_head
        return lib.ndl_attention_mass(P, P, P, 64 * hkv, P, 4, P, w, w, None, P, 1, 1, 1, 16 * w,
                                      hkv, hkv, 64, 16, 0, 0.1, 1.0, None, 0, None)
    for per, hkv in ((1 << 22, 2), ((1 << 22) + 1, 2), ((1 << 23) - 1, 2), (1 << 20, 8),
                     (1 << 20, 9)):
        assert weigh(per, hkv) == -2, (per, hkv)
    # one workgroup fewer goes on to the workspace, which is missing
    for per, hkv in (((1 << 22) - 1, 2), ((1 << 23) - 1, 1), ((1 << 20) - 1, 8)):
        assert weigh(per, hkv) == -3, (per, hkv)


def test_grids_of_the_selection(lib):
    """A workgroup of 1,024 threads for a kv head of a sequence."""
    def select(hkv):
        return lib.ndl_kv_select(P, P, P, 1, hkv, 16, P, 8, 8, P, 3, 32, 4, 8, None)
    assert select(1 << 22) == -2 and select(MOST) == -2
