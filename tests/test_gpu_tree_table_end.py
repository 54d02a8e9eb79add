"""Trees after contexts that are longer than their block table holds: the table's last tokens are attended
whole, those past it and the nodes not, wherever the table ends in a tile of keys.  Bounds:
test_gpu_tree_attention.py's.
"""
import pytest
import torch

from test_gpu_tree_attention import Case

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("fp8", [False, True], ids=["16-bit", "8-bit"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(8, 2, 64, 16), (7, 1, 128, 16), (4, 2, 64, 32)])
@pytest.mark.parametrize("blocks", [1, 2, 3, 5])
def test_contexts_past_the_table(shape, blocks, dtype, fp8):
    """Contexts from just before the table's end (nodes fall past it, or half of them) to far past."""
    cap = blocks * shape[3]
    lens = [cap - 5, cap, cap + 1, cap + 15, cap + 16, cap + 17, cap + 31, cap + 32, cap + 52,
            cap + 64, cap + 200, cap + 2001]
    counts = [9, 3, 20, 1, 7, 2, 40, 5, 12, 1, 33, 6]
    c = Case(shape, counts, lens, dtype, seed=blocks, fp8=fp8)
    c.table = c.table[:, :blocks].contiguous()
    c.check(c.run())


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_long_table_of_an_odd_number_of_blocks(dtype):
    """In shares; over the 8-bit pool in row blocks of up to 256 columns as well."""
    for fp8, most in ((False, 9), (False, 70), (True, 9), (True, 140)):
        c = Case((8, 2, 64, 16), [most, 11], [6416 + 100, 6416 + 16], dtype, seed=4, fp8=fp8)
        c.table = c.table[:, :401].contiguous()
        assert not (fp8 and most > 16) or most * 4 * 401 * 16 * 2 * 2 >= 12 << 20
        c.check(c.run())
