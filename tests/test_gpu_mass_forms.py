"""attention_mass where a call's bounds choose between its forms: scores kept, or made again from K
because those of the bounds would take more than the workspace may.  Bounds:
test_gpu_attention_mass.py's.
"""
import math

import pytest
import torch

from needle_amd import ops
from test_gpu_attention_mass import Case

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]
KEPT = 1 << 30                 # bytes of scores that a call keeps at most


def widened(c, columns):
    """The case with invalid columns behind its table until its scores would pass KEPT."""
    per_key = 4 * columns * len(c.counts) * c.hkv
    cols = KEPT // (per_key * c.bs) + 1
    c.table = torch.cat([c.table, torch.full((len(c.counts), cols - c.table.shape[1]), -1,
                                             dtype=torch.int32)], 1)
    keys = c.table.shape[1] * c.bs
    need = ops.attention_mass_workspace_bytes(len(c.counts), int(c.cu[-1]), max(c.counts), keys,
                                              c.h, c.hkv, c.d, c.bs)
    assert need < per_key * keys
    return c


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(32, 8, 128, 16), (14, 2, 64, 64), (16, 1, 128, 32)])
def test_decode_without_kept_scores(shape, dtype):
    lens = [0, 1, 14, 31, 32, 100, 257, 300, 1900, -1]
    c = widened(Case(shape, [1] * len(lens), lens, dtype, seed=31), shape[0] // shape[1])
    c.check(c.run(decode=True))
    c.check(c.run(decode=True, decay=0.75), 0.75)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts", [[1, 1, 1], [3, 0, 8], [8, 5, 1]])
def test_short_chunks_without_kept_scores(counts, dtype):
    c = widened(Case((8, 2, 64, 16), counts, [700, 20, 33], dtype, seed=32), 4 * max(counts))
    c.check(c.run())
    c.check(c.run(max_context_len=700))        # with its scores kept


def test_just_within_the_kept_scores():
    """The largest table whose scores are kept, and one column more."""
    c = Case((8, 2, 64, 16), [1, 1], [300, 45], seed=33)
    cols = KEPT // (4 * 4 * 2 * 2 * 16)
    for w, kept in ((cols, True), (cols + 1, False)):
        need = ops.attention_mass_workspace_bytes(2, 2, 1, w * 16, 8, 2, 64)
        assert (need > KEPT) == kept
    c.table = torch.cat([c.table, torch.full((2, cols - c.table.shape[1]), -1,
                                             dtype=torch.int32)], 1)
    c.check(c.run(decode=True))

def test_rows_whose_scores_are_all_minus_infinity():
    """The softmax's sum is 0: no weight and zeros, whether scores are kept or made again, for that row
    alone."""
    for counts in ([8, 2], [40, 2]):
        c = Case((8, 2, 64, 16), counts, [0, 100], seed=34)
        # the first token's own key, the only one it attends, is -inf in a dimension where the queries
        # of kv head 1 are positive
        c.pool[0, int(c.table[0, 0]), 1, 0, 3] = -math.inf
        c.q[:, 4:, 3] = c.q[:, 4:, 3].abs() + 0.5
        out, mass = c.run()
        assert not out[0, 4:].any()
        assert out[0, :4].isfinite().all() and out[1:].isfinite().all()
        p = torch.arange(counts[0])
        got = mass.cpu()[c.table[0].long()[p // 16], :, p % 16]
        assert got.isfinite().all(), (counts, got)
        # a head's tokens give 1 each, the first one's row nothing on kv head 1
        total = got.sum(0)
        want = torch.tensor([4.0 * counts[0], 4.0 * (counts[0] - 1)])
        assert (total - want).abs().max() < 2.0 ** -12 * want.max(), total
