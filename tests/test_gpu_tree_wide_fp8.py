"""Wide trees over the 8-bit pool, whose codes are unpacked once for up to 256 columns: a call takes
these row blocks by its columns and by the scores that its bounds allow, so a wide table (of blocks that
are not valid) has small trees take them.  Bounds: test_gpu_tree_attention.py's.
"""
import pytest
import torch

from test_gpu_tree_attention import Case, attention_bound

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def wide(shape, counts, lens, dtype, whole=False, **more):
    """A case past 64 columns and 12 * 2^20 scores in all."""
    h, hkv, _, bs = shape
    cols = max(counts) * (h // hkv)
    assert cols > 64
    c = Case(shape, counts, lens, dtype, fp8=True, **more)
    w = c.table.shape[1]
    need = -(-(12 << 20) // (cols * bs * len(counts) * hkv))
    if whole:
        assert w * bs <= 1536 and need <= 1536 // bs      # row blocks are not split
    if need > w:
        c.table = torch.cat([c.table, torch.full((len(counts), need - w), -1,
                                                 dtype=torch.int32)], 1)
    assert cols * c.table.shape[1] * bs * len(counts) * hkv >= 12 << 20
    return c


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(14, 2, 64, 16), (32, 8, 128, 16), (28, 4, 128, 64),
                                   (16, 1, 128, 32), (16, 1, 64, 256)])
@pytest.mark.parametrize("counts", [[17, 2, 0, 9], [32, 33, 5, 18], [70, 1, 0, 37]])
def test_trees(shape, counts, dtype):
    c = wide(shape, counts, [37, 0, 250, 15], dtype, seed=2)
    c.check(c.run())
    c.ctx[0] = -2                     # attends nothing
    got = c.run()
    c.check(got)
    assert not got[:counts[0]].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(32, 8, 128, 16), (64, 8, 64, 64)])
@pytest.mark.parametrize("most", [16, 17, 31, 33, 65])
def test_whole_row_blocks(shape, most, dtype):
    """From half of the four-group form's columns to two row blocks of the eight-group one's; lengths
    that end anywhere in a tile."""
    if most * (shape[0] // shape[1]) <= 64:
        most += 1
    counts = [most, 3, most - 5, 1, 20 % most, most // 2, 0, most]
    counts += counts[::-1]
    lens = [0, 1, 31, 32, 33, 700, 64, 95, 96, 5, 127, 128, 300, 16, 15, 2]
    c = wide(shape, counts, lens, dtype, whole=True, seed=5)
    c.check(c.run())


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_contexts(dtype):
    """More tiles than codes are loaded ahead of, and than a window of block ids holds."""
    c = wide((28, 4, 128, 64), [36, 12], [4500, 2111], dtype, seed=3)
    c.check(c.run())
    c.check(c.run(max_context_len=5000))


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_codes_and_blocks_that_are_not_valid(dtype):
    c = wide((8, 2, 128, 16), [24, 30, 18, 4], [45, 300, 900, 40], dtype, seed=6)
    for x, (i, node) in enumerate([(0, 2), (0, 4), (1, 1), (1, 7), (2, 17)]):
        p = c.lens[i] + node
        c.pool[0][1, int(c.table[i, p // 16]), x % 2, p % 16, 5 * x] = 0x7F
    p = c.lens[1] + c.counts[1] - 1          # a leaf's key
    c.pool[0][0, int(c.table[1, p // 16]), 0, p % 16, 3] = 0x7F
    c.table[0, 1] = -1
    c.table[2, 0] = c.nb
    c.table[2, 40] = 1 << 30
    c.table[3] = -5
    r = c.want()
    assert 0.0 < r.out.isnan().float().mean() < 0.2
    got = c.run()
    c.check(got)
    assert not got[72:].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_any_mask(dtype):
    gen = torch.Generator().manual_seed(8)
    counts = [40, 7, 70]
    see = [torch.rand(n, n, generator=gen) < 0.3 for n in counts]
    see[0][3] = see[0][17] = False           # with no context: nothing to attend
    c = wide((8, 2, 64, 16), counts, [0, 21, 64], dtype, seed=9, see=see)
    got = c.run()
    c.check(got)
    assert not got[3].any() and not got[17].any()


@pytest.mark.parametrize("scale", [0.0, -0.11, 0.3])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scales(scale, dtype):
    c = wide((8, 2, 64, 16), [20, 30], [45, 1900], dtype, seed=12)
    c.scale = scale
    c.check(c.run())


def test_the_largest_float16_rows():
    """Rows of 65,504, whose code is 65,536: such a value counts as that or as 65,504, and outputs
    stay finite."""
    c = wide((8, 2, 128, 16), [20, 18], [45, 130], torch.float16, seed=4)
    codes, scales = c.pool
    for i in range(2):
        p = torch.arange(c.lens[i] + c.counts[i])
        blk = c.table[i].long()[p // 16]
        codes[1, blk, :, p % 16, 7] = 0x78           # 256 * 2^8
        scales[1, blk, :, p % 16] = 127 + 8
        codes[0, blk[5], :, 5, 9] = 0xF8             # a key of -65,536 among small ones
        scales[0, blk[5], :, 5] = 127 + 8
    c.q *= 2.0 ** -10
    got = c.run()
    r = c.want()
    assert got.isfinite().all() and (got[:, :, 7] == 65504).all()
    assert (r.out[:, :, 7] - 65536).abs().max() < 1e-6
    # Elsewhere values are up to 208 * 2^8.  A probability in float16 is off by half a step of it or by
    # 2^-25 (subnormal ones; the largest is 1 or more): attention_bound takes values up to 32 for that.
    bound = attention_bound(r, c.dtype, c.d) + r.lens[:, None, None] * 2.0 ** -25 * 208 * 256
    off = (got.cpu().double() - r.out).abs()
    off[:, :, 7] = 0.0
    assert (off <= bound).all()
