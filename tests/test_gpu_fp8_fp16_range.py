"""Attention in float16 over rows at the end of that format: the largest finite values, 63,488 to
65,504, are 65,536 as codes (256 under the scale 2^8), a number that float16 has not.

Bounds as in test_gpu_fp8_attention, with two terms of their own: a value of 65,536 that is held in
float16 is 65,504, off by 2^-11 of it, so sum_t p_t |v_t| counts once more; and a probability that is
subnormal in float16, off by 2^-25, stands before values of 65,536."""
import pytest
import torch

from needle_amd import ops
from oracle import fp8_ref
from test_gpu_fp8_attention import DEV, Case, _unpacks, _wide

pytestmark = pytest.mark.gpu


class Large(Case):
    """Rows `at` (plane, sequence, position) of every kv head hold codes up to 256 under 2^8."""

    def __init__(self, *args, at, **more):
        super().__init__(*args, dtype=torch.float16, **more)
        self.at = at
        for n, (plane, seq, pos) in enumerate(at):
            b, r = int(self.table[seq, pos // self.bs]), pos % self.bs
            row = self.codes[plane, b, :, r]
            row[:, n % 3::5] = 0x78              # 256
            row[:, n % 4::7] = 0xF8
            self.scales[plane, b, :, r] = 135

    def check(self, got):
        out, weight, big, n = self.want()
        got = got.double().cpu()
        assert out.abs().max() < 65504 and got.isfinite().all()
        u = 2.0 ** -11
        rel = 2 * (self.d + 8) * 2.0 ** -24 * big[..., None] + 2.0 ** -20 \
            + n[:, None, None] * 2.0 ** -23
        bound = u * (2 * weight + out.abs()) + rel * weight \
            + 2.0 ** -25 * (n[:, None, None] * 28 + len(self.at) * 65536)
        assert ((got - out).abs() <= bound).all()


def _case(count, d, at, seed, **more):
    shape, counts = (8, 2, d, 16), [count, max(1, count // 2)]
    return Large(shape, counts, [40, 95], seed=seed, at=at,
                 extra_cols=_wide(shape, counts) if count == 80 else 1, **more)


@pytest.mark.parametrize("count", [1, 6, 80])
@pytest.mark.parametrize("d", [64, 128])
def test_values(count, d):
    """In cached rows and in the chunk's own, the last one among them, which the causal mask keeps
    from the tokens before it."""
    c = _case(count, d, [(1, 0, 3), (1, 0, 17), (1, 0, 39 + count), (1, 1, 20),
                         (1, 1, 94 + max(1, count // 2))], 1)
    assert _unpacks(c) == (count == 80)
    c.check(c.run(decode=count == 1) if count == 1 else c.run())


@pytest.mark.parametrize("count", [1, 6, 80])
@pytest.mark.parametrize("d", [64, 128])
def test_keys(count, d):
    """Keys enter the scores at their value, on every path."""
    c = _case(count, d, [(0, 0, 3), (0, 0, 39 + count), (0, 1, 20)], 2)
    c.q = (c.q.float() * 2.0 ** -11).to(c.dtype)
    c.check(c.run(decode=count == 1) if count == 1 else c.run())


@pytest.mark.parametrize("scale", [-0.1, 0.0])
def test_keys_of_long_chunks_under_any_scale(scale):
    c = _case(80, 64, [(0, 0, 3), (0, 0, 119), (0, 1, 20)], 3)
    c.q = (c.q.float() * 2.0 ** -11).to(c.dtype)
    c.scale = scale
    assert _unpacks(c)
    c.check(c.run())


def test_shares_and_merge():
    """The parts of a split sequence, the rescaled sums among them."""
    for counts in ([1, 1, 1], [3, 1, 6]):
        c = Large((32, 8, 128, 16), counts, [2900, 3, 1111], seed=4,
                  at=[(1, 0, 0), (1, 0, 1500), (1, 0, 2900), (1, 2, 700), (1, 2, 1111)])
        assert ops.fp8_attention_workspace_bytes(3, sum(counts), max(counts), c.table.shape[1] * 16,
                                                 32, 8, 128) > 0
        c.check(c.run(decode=max(counts) == 1))


def test_rows_appended_in_float16():
    """What a float16 model writes: its largest number in the last token's values."""
    gen = torch.Generator().manual_seed(5)
    k, v = (torch.randn(9, 2, 64, generator=gen).half() for _ in range(2))
    v[8, :, 5] = 65504.0
    q = torch.randn(9, 8, 64, generator=gen).half()
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    pool = ops.fp8_kv_pool(1, 2, 16, 64, device=DEV)
    cu = torch.tensor([0, 9], dtype=torch.int32, device=DEV)
    ctx = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.kv_append_fp8(k.to(DEV), v.to(DEV), *pool, table, ctx, cu)
    got = ops.varlen_prefill_fp8(q.to(DEV), *pool, table, cu, ctx, 9, 0.125, 8, 2, 64).cpu()
    assert got.isfinite().all()
    out, weight, _, _ = fp8_ref.attention(q, pool.codes.cpu().view(torch.uint8), pool.scales.cpu(),
                                          table.cpu(), cu.cpu(), ctx.cpu(), 0.125)
    assert got[:8].abs().max() < 8 and (got[8, :, 5].double() - out[8, :, 5]).abs().max() <= \
        2.0 ** -9 * weight[8, :, 5].max()


@pytest.mark.parametrize("count", [1, 3, 80])
def test_an_output_at_the_end(count):
    """Tokens that attend nothing but values of 65,504 have that, not infinity."""
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    if count == 80:
        table = torch.zeros(1, _wide((8, 2, 64, 128), [80]), dtype=torch.int32, device=DEV)
    v = torch.full((count, 2, 64), 65504.0, dtype=torch.float16, device=DEV)
    v[:, 1, 7] = -65504.0
    q = torch.randn(count, 8, 64, generator=torch.Generator().manual_seed(6)).half().to(DEV)
    pool = ops.fp8_kv_pool(1, 2, 128, 64, device=DEV)
    cu = torch.tensor([0, count], dtype=torch.int32, device=DEV)
    ctx = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.kv_append_fp8(v.sign(), v, *pool, table, ctx, cu)
    if count == 1:
        got = ops.paged_decode_fp8(q, *pool, table, ctx, 0.125, 8, 2, 64)
    else:
        got = ops.varlen_prefill_fp8(q, *pool, table, cu, ctx, count, 0.125, 8, 2, 64)
    want = torch.full_like(got, 65504.0)
    want[:, 4:, 7] = -65504.0
    # (a sum of float16 probabilities over their fp32 sum is 1 to 2^-11: 65,504 or the next below)
    assert (got.float() - want.float()).abs().max() <= 32
