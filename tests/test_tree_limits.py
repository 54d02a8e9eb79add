"""Sizes next to the entry points' limits, which the counting behind them has to hold: refused, or planned
for as smaller ones are, before any launch (CPU)."""
import pytest
import torch

from needle_amd import _lib, ops

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


@pytest.mark.parametrize("which", ["16-bit", "8-bit", "mass"])
def test_bounds_of_tokens_next_to_31_bits(lib, which):
    """The row blocks of max_seqlen tokens (8 sequences, group 1: 2^31 tokens by 256, more than a grid or
    31 bits of row blocks hold): refused as a large bound is, no negative number of them."""
    def call(most, keys):
        chunk = (P, P, 128, P, *((P,) if which == "8-bit" else ()), 4, P, 500, 500, P, P)
        rest = (8, 90, most, keys, 2, 2, 64, 16, 0, 0.1)
        if which == "mass":
            return lib.ndl_attention_mass(P, *chunk, *rest, 1.0, P, 1 << 50, None)
        f = lib.ndl_fp8_tree_attention if which == "8-bit" else lib.ndl_tree_attention
        return f(*chunk, P, 2, 2, *rest, P, 1 << 50, None)

    def need(most, keys):
        if which == "mass":
            return lib.ndl_attention_mass_workspace_bytes(8, 90, most, keys, 2, 2, 64, 16)
        f = (lib.ndl_fp8_tree_attention_workspace_bytes if which == "8-bit" else
             lib.ndl_tree_attention_workspace_bytes)
        return f(8, most, keys, 2, 2, 64, 16)
    for keys in (64, 8000):
        for most in (1 << 29, MOST - 256, MOST - 255, MOST):
            assert call(most, keys) == -1, (most, keys)
            assert need(most, keys) == need(1 << 29, keys) < 1 << 20


def test_the_weights_over_an_8_bit_pool():
    pool = ops.Fp8KVCache(torch.zeros(2, 3, 2, 16, 64, dtype=torch.float8_e4m3fn),
                          torch.zeros(2, 3, 2, 16, dtype=torch.uint8))
    table, lens = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(TypeError, match="16-bit"):
        ops.attention_mass(torch.zeros(1, 4, 64), pool, table, lens, torch.zeros(3, 2, 16), 0.1, 4,
                           2, 64)
