"""Trees over 8-bit pools whose rows are small: keys that are subnormal in float16, whole or halved, count
as they are.

Codes of 2^-3 to 2 less a bit under a scale of 2^-15 are keys of 2^-18 to 2^-14, halves of 2^-19 and more
in steps of 2^-22 and more: float16 holds them all, so that the bound is test_gpu_tree_attention.py's.
Values of those sizes are subnormal as well, but exact; outputs are off by what that bound says of
subnormal ones.  Codes below 2^-5 have halves of odd multiples of 2^-25: where keys are held in float16
each is off by 2^-24 at most, a score by scale sum_d |q_d| 2^-24, which enters a probability's
numerator and denominator.
"""
import pytest
import torch

from test_gpu_tree_attention import Case, attention_bound
from test_gpu_tree_wide_fp8 import wide

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def small(c, lowest, highest):
    """Codes of c from byte `lowest` to `highest`, both signs, under 2^-15; queries that give scores of
    about 1."""
    codes, scales = c.pool
    held = scales < 254                    # (rows that no sequence holds keep what they have)
    new = torch.randint(lowest, highest + 1, codes.shape, generator=c.gen, dtype=torch.uint8)
    new += torch.randint(0, 2, codes.shape, generator=c.gen, dtype=torch.uint8) * 128
    codes[held] = new[held]
    scales[held] = 127 - 15
    c.q = (c.q.float() * 2.0 ** 12).to(c.dtype)
    return c


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(8, 2, 64, 16), (8, 2, 128, 64)])
@pytest.mark.parametrize("many", [False, True], ids=["few-columns", "many-columns"])
def test_keys_that_float16_holds(many, shape, dtype):
    counts, lens = [24, 3, 18], [45, 300, 0]
    if many:
        c = wide(shape, counts, lens, dtype, seed=41)
    else:
        c = Case(shape, [4, 3, 2], lens, dtype, seed=41, fp8=True)
    small(c, 0x20, 0x3F)
    c.scale = 4.0
    r = c.want()
    assert 0.2 < float(r.big.mean())
    c.check(c.run())


@pytest.mark.parametrize("many", [False, True], ids=["few-columns", "many-columns"])
def test_the_smallest_float16_keys(many):
    """Codes of the lowest bits: 2^-9 to 2^-6 by 2^-15."""
    shape, counts, lens = (8, 2, 64, 16), [24, 3, 18], [45, 300, 0]
    if many:
        c = wide(shape, counts, lens, torch.float16, seed=42)
    else:
        c = Case(shape, [4, 3, 2], lens, torch.float16, seed=42, fp8=True)
    small(c, 0x00, 0x08)
    c.scale = 64.0
    r = c.want()
    off = c.scale * c.q.double().abs().sum(-1) * 2.0 ** -24         # [T, H], of a score
    bound = attention_bound(r, c.dtype, c.d) + (2 * off).expm1()[..., None] * r.weight
    assert ((c.run().cpu().double() - r.out).abs() <= bound).all()
