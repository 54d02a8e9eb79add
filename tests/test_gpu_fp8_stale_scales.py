"""Rows that no token attends may hold any bytes, in the scales as in the codes: a pool of
uninitialised memory holds 255, which is no scale."""
import pytest
import torch

from test_gpu_fp8_attention import DTYPES, Case, _unpacks, _wide
from test_gpu_fp8_decode_append import Step

pytestmark = pytest.mark.gpu


def _stale(c):
    """255 in every scale byte that no sequence attends."""
    used = torch.zeros(c.nb, c.bs, dtype=torch.bool)
    for i, (n, m) in enumerate(zip(c.lens, c.counts)):
        p = torch.arange(max(0, n + m))
        used[c.table[i][p // c.bs].long(), p % c.bs] = True
    c.scales[:, ~used[:, None].expand(-1, c.hkv, -1)] = 255
    return c


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(14, 2, 64, 16), (32, 8, 128, 16), (16, 4, 128, 64)])
def test_decode_and_chunks(shape, dtype):
    lens = [0, 1, 15, 16, 31, 32, 100, -1]
    c = _stale(Case(shape, [1] * 8, lens, dtype, seed=1))
    c.check(c.run(decode=True))
    Step(c).check()
    c = _stale(Case(shape, [1, 2, 0, 9], [37, 0, 250, 15], dtype, seed=2))
    c.check(c.run())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(14, 2, 64, 16), (16, 4, 128, 64)])
def test_shares_and_long_chunks(shape, dtype):
    c = _stale(Case(shape, [1, 1, 1], [2900, 3, 1111], dtype, seed=3))
    c.check(c.run(decode=True))
    c = _stale(Case(shape, [90, 3], [77, 9], dtype, seed=4, extra_cols=_wide(shape, [90, 3])))
    assert _unpacks(c)
    c.check(c.run())
