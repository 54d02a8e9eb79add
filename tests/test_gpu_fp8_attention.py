"""Attention over the 8-bit pool on the GPU against its definition in float64.

The bound of every output element, from the roundings made on the way (u: half a step of the
16-bit format, 2^-8 or 2^-11): the probabilities and the output are rounded once each, u (A + |o|)
with A = sum_t p_t |v_t|; a score is a sum of D products in fp32 with two more roundings, off by
(D + 8) 2^-24 of scale sum_d |q_d k_d|, which enters a probability's numerator and denominator;
the exponentials, the running sums and the merge add 2^-20 + n 2^-23.  float16 probabilities
below 2^-14 are subnormal, each off by 2^-25 where the largest is at least 1.
"""
import pytest
import torch

from needle_amd import ops
from oracle import fp8_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float16]


class Case:
    """Sequences of `counts` new tokens after `lens` cached ones.  Every row that no sequence
    attends holds random bytes, NaN codes among them."""

    def __init__(self, shape, counts, lens, dtype=torch.bfloat16, seed=0, extra_cols=1, wide=True):
        self.h, self.hkv, self.d, self.bs = shape
        self.dtype, self.counts, self.lens = dtype, counts, lens
        gen = self.gen = torch.Generator().manual_seed(seed)
        need = [max(1, -(-(c + n) // self.bs)) for c, n in zip(lens, counts)]
        self.nb = sum(need) + 3
        perm = torch.randperm(self.nb - 1, generator=gen)
        self.table = torch.full((len(lens), max(need) + extra_cols), self.nb - 1,
                                dtype=torch.int32)
        self.codes = torch.randint(0, 256, (2, self.nb, self.hkv, self.bs, self.d),
                                   generator=gen, dtype=torch.uint8)
        self.codes[..., ::7] = 0x7F
        self.scales = torch.randint(1, 255, self.codes.shape[:4], generator=gen,
                                    dtype=torch.uint8)
        at = 0
        for i, n in enumerate(need):
            blocks = perm[at:at + n]
            at += n
            self.table[i, :n] = blocks.to(torch.int32)
            total = max(0, lens[i] + counts[i])
            if not total:
                continue
            p = torch.arange(total)
            blk, row = blocks[p // self.bs], p % self.bs
            c = torch.randint(0, 256, (total, 2, self.hkv, self.d), generator=gen,
                              dtype=torch.uint8)
            c[(c & 127) > 117] = 0x31          # within 224, no NaN
            self.codes[:, blk, :, row] = c
            # values about 1, and rows up to 8 times smaller or larger
            self.scales[:, blk, :, row] = torch.randint(
                118, 124, (total, 2, self.hkv), generator=gen, dtype=torch.uint8)
        self.cu = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32)
        self.ctx = torch.tensor(lens, dtype=torch.int32)
        self.q = torch.randn(int(self.cu[-1]), self.h, self.d, generator=gen).to(dtype)
        self.scale = 1.0 / self.d ** 0.5

    def want(self):
        return fp8_ref.attention(self.q, self.codes, self.scales, self.table, self.cu, self.ctx,
                                 self.scale)

    def run(self, decode=False, q=None, **more):
        q = self.q.to(DEV) if q is None else q
        pool = (self.codes.to(DEV).view(torch.float8_e4m3fn), self.scales.to(DEV))
        heads = (self.scale, self.h, self.hkv, self.d)
        if decode:
            return ops.paged_decode_fp8(q, *pool, self.table.to(DEV), self.ctx.to(DEV), *heads,
                                        **more)
        return ops.varlen_prefill_fp8(q, *pool, self.table.to(DEV), self.cu.to(DEV),
                                      self.ctx.to(DEV), max(max(self.counts), 1), *heads, **more)

    def check(self, got):
        out, weight, big, n = self.want()
        got = got.double().cpu()
        rows = int(self.cu[-1])
        got, out, weight, big, n = (x[:rows] for x in (got, out, weight, big, n))
        assert torch.equal(got.isnan(), out.isnan())
        u = torch.finfo(self.dtype).eps / 2
        rel = 2 * (self.d + 8) * 2.0 ** -24 * big[..., None] + 2.0 ** -20 \
            + n[:, None, None] * 2.0 ** -23
        bound = u * (weight + out.abs()) + rel * weight
        if self.dtype == torch.float16:
            bound = bound + n[:, None, None] * 2.0 ** -25 * 32    # values are at most 28
        off = (got - out).abs().nan_to_num(0.0)
        worst = (off / bound.nan_to_num(1.0).clamp(min=1e-300)).max() if off.numel() else 0.0
        assert worst <= 1.0, float(worst)


SHAPES = [(14, 2, 64, 16), (32, 8, 128, 16), (28, 4, 128, 64), (16, 1, 128, 32), (3, 3, 64, 1024),
          (10, 2, 64, 256), (13, 1, 128, 16)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_decode(shape, dtype):
    lens = [0, 1, 14, 15, 16, 31, 32, 63, 100, 129, 257, -1, -5]
    c = Case(shape, [1] * len(lens), lens, dtype, seed=1)
    c.check(c.run(decode=True))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("counts", [[1, 2, 0, 3], [5, 1, 8, 4], [16, 3, 17, 1], [70, 0, 33]])
def test_chunks(shape, dtype, counts):
    lens = [37, 0, 250, 15][:len(counts)]
    c = Case(shape, counts, lens, dtype, seed=2)
    c.check(c.run())
    c.ctx[0] = -2                     # attends nothing
    got = c.run()
    c.check(got)
    assert not got[:counts[0]].any()


@pytest.mark.parametrize("shape", [(14, 2, 64, 16), (32, 8, 128, 16), (7, 1, 128, 64)])
@pytest.mark.parametrize("counts", [[1, 1, 1], [3, 1, 6], [40, 9, 2]])
def test_shares_and_merge(shape, counts):
    """Contexts long enough for the split into shares, of very different lengths."""
    c = Case(shape, counts, [2900, 3, 1111], seed=3)
    assert ops.fp8_attention_workspace_bytes(3, sum(counts), max(counts), c.table.shape[1] * c.bs,
                                             c.h, c.hkv, c.d, c.bs) > 0
    c.check(c.run(decode=max(counts) == 1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(8, 2, 64, 16), (16, 4, 128, 32)])
def test_row_blocks_of_one_chunk(shape, dtype):
    """Chunks of several row blocks, just short of those that are unpacked first."""
    c = Case(shape, [60, 33, 1, 17], [1500, 70, 800, 0], dtype, seed=15)
    c.check(c.run())
    c.check(c.run(max_context_len=1500))


def _wide(shape, counts):
    """Table columns from which a call of these chunks unpacks its keys first."""
    rows = max(counts) * (shape[0] // shape[1])
    assert rows >= 224
    return -(-(1 << 24) // (rows * shape[1] * len(counts) * shape[3]))


def _unpacks(c, max_context_len=None):
    keys = c.table.shape[1] * c.bs
    if max_context_len is not None:
        keys = min(keys, max_context_len + max(c.counts))
    pool = len(c.counts) * -(-keys // c.bs) * c.bs * c.hkv * c.d * 4
    return ops.fp8_attention_workspace_bytes(len(c.counts), sum(c.counts), max(c.counts), keys,
                                             c.h, c.hkv, c.d, c.bs) >= pool


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("counts,lens", [([260], [0]), ([300, 1, 90], [77, 400, 0]),
                                         ([257, 5], [1000, -3])])
def test_long_chunks(shape, dtype, counts, lens):
    """Chunks whose keys are unpacked into the workspace first, and, with a bound that says how
    few there are, the same chunks as row blocks."""
    c = Case(shape, counts, lens, dtype, seed=16, extra_cols=_wide(shape, counts))
    assert _unpacks(c)
    c.check(c.run())
    ws = ops.decode_workspace(ops.fp8_attention_workspace_bytes(
        len(lens), sum(counts), max(counts), c.table.shape[1] * c.bs, c.h, c.hkv, c.d, c.bs), DEV)
    ws.fill_(0xFF)
    c.check(c.run(workspace=ws))
    if not _unpacks(c, max(lens)):
        c.check(c.run(max_context_len=max(lens)))


def test_long_chunks_in_more_keys():
    """Prefixes of thousands of tokens, split over the workgroups of the prefill."""
    for shape, counts, lens in (((28, 4, 128, 16), [200, 64], [3100, 2500]),
                                ((14, 2, 64, 64), [300], [5000])):
        c = Case(shape, counts, lens, seed=17)
        assert _unpacks(c, max(lens))
        c.check(c.run(max_context_len=max(lens)))


def test_many_row_blocks_in_shares():
    """More than 64 row blocks: their slots are found over several steps of the scan."""
    c = Case((8, 8, 64, 16), [1] * 70, [5 + 13 * i for i in range(70)], seed=4, extra_cols=30)
    c.check(c.run(decode=True))
    c = Case((16, 2, 64, 16), [90, 200, 1], [700, 30, 1200], seed=5)
    c.check(c.run())


def test_tables_that_end_and_bad_blocks():
    """Keys past the table's columns are not attended; neither are those of an invalid block."""
    for counts in ([1, 1, 1], [4, 4, 4], [70, 20, 10], [30000, 20, 10]):
        c = Case((8, 2, 64, 16), counts, [70, 45, 0], seed=6, extra_cols=0)
        c.table = c.table[:, :3].contiguous()     # 48 keys
        assert _unpacks(c) == (counts[0] == 30000)
        c.table[1, 1] = -1
        c.table[2, 0] = c.nb                      # all that the third attends
        got = c.run(decode=counts[0] == 1)
        c.check(got)
        assert not got[int(c.cu[2]):].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count,d", [(9, 64), (80, 64), (9, 128), (80, 128)])
def test_a_nan_stays_where_it_is_attended(dtype, count, d):
    """A NaN among the chunk's own values reaches the tokens from its position on, no others."""
    shape = (8, 2, d, 16)
    c = Case(shape, [count, 4], [20, 61], dtype, seed=7,
             extra_cols=_wide(shape, [count, 4]) if count == 80 else 1)
    assert _unpacks(c) == (count == 80)
    for plane, seq, pos, d in ((1, 0, 24, 11), (1, 1, 64, 63), (0, 1, 63, 5), (1, 0, 28, 0)):
        b = int(c.table[seq, pos // 16])
        c.codes[plane, b, 1, pos % 16, d] = 0x7F if d % 2 else 0xFF
    got = c.run()
    c.check(got)
    assert got[:4].isfinite().all() and got[4, 4:, 11].isnan().all()


def test_scores_of_any_size():
    """Large scores (one key takes all), a raised maximum late in the row, and scale 0 and
    below."""
    for scale, n in ((40.0, 3), (0.0, 3), (-0.3, 3), (1e-6, 3), (40.0, 66), (0.0, 66), (-0.3, 66)):
        shape = (8, 2, 128, 16)
        c = Case(shape, [n, 1], [700, 90], seed=8,
                 extra_cols=_wide(shape, [n, 1]) if n == 66 else 1)
        c.scale = scale
        if scale == 40.0:
            c.q = (c.q.float() * 0.02).to(c.dtype)
        c.check(c.run())
    c = Case((8, 2, 128, 16), [1], [1500], seed=9)
    # keys that grow along the context: the maximum is raised again and again
    for p in range(1501):
        b = int(c.table[0, p // 16])
        c.codes[0, b, :, p % 16] = 0x38
        c.scales[0, b, :, p % 16] = 90 + p // 50
    c.q = c.q.abs()
    c.check(c.run(decode=True))


@pytest.mark.parametrize("counts", [[3, 5, 1], [60, 5, 1]])
def test_strided_queries_and_padding_rows(counts):
    shape = (14, 2, 64, 16)
    c = Case(shape, counts, [40, 0, 17], seed=10,
             extra_cols=_wide(shape, counts) if max(counts) == 60 else 1)
    n = int(c.cu[-1])
    wide = torch.full((n + 4, 18 * 64), float("nan"), dtype=c.dtype, device=DEV)
    q = wide[:, 64:64 + 14 * 64].view(n + 4, 14, 64)
    q[:n] = c.q.to(DEV)
    out = torch.full((n + 4, 14, 64), 5.0, dtype=c.dtype, device=DEV)
    got = c.run(q=q, out=out)
    assert got is out
    c.check(got)
    assert (out[n:] == 5.0).all()     # rows behind the last sequence


def test_same_inputs_same_bits_and_a_workspace_of_ones_own():
    c = Case((32, 8, 128, 16), [1] * 5, [3000, 17, 900, 1, 450], seed=11)
    need = ops.fp8_attention_workspace_bytes(5, 5, 1, c.table.shape[1] * 16, 32, 8, 128)
    ws = ops.decode_workspace(need, DEV)
    first = c.run(decode=True)
    for _ in range(3):
        ws.fill_(0xFF)                # NaN where something is read that was not written
        assert torch.equal(c.run(decode=True, workspace=ws).view(torch.int16),
                           first.view(torch.int16))


@pytest.mark.parametrize("count", [1, 6, 50])
def test_captured_and_replayed(count):
    shape = (14, 2, 64, 16)
    c = Case(shape, [count] * 3, [1900, 40, 333], seed=12,
             extra_cols=_wide(shape, [count] * 3) if count == 50 else 1)
    q, pool = c.q.to(DEV), (c.codes.to(DEV), c.scales.to(DEV))
    t, cu, ctx = c.table.to(DEV), c.cu.to(DEV), c.ctx.to(DEV)

    def step():
        if count == 1:
            return ops.paged_decode_fp8(q, *pool, t, ctx, c.scale, 14, 2, 64)
        return ops.varlen_prefill_fp8(q, *pool, t, cu, ctx, count, c.scale, 14, 2, 64)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        q.normal_()
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_on_another_stream():
    c = Case((32, 8, 128, 16), [1, 1], [1500, 77], seed=13)
    base = c.run(decode=True)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = c.run(decode=True)
    s.synchronize()
    assert torch.equal(got, base)


def test_refusals():
    c = Case((8, 2, 64, 16), [2, 2], [5, 6], seed=14)
    with pytest.raises(TypeError, match="q must be bfloat16 or float16"):
        c.run(q=c.q.float().to(DEV))
    with pytest.raises(ValueError, match="head counts"):
        ops.paged_decode_fp8(c.q[:2].to(DEV), c.codes.to(DEV), c.scales.to(DEV), c.table.to(DEV),
                             c.ctx.to(DEV), 1.0, 8, 4, 64)
    with pytest.raises(ValueError, match="batch mismatch"):
        c.run(decode=True)
    with pytest.raises(ValueError, match="1 to 16 times"):
        ops.paged_decode_fp8(torch.zeros(2, 34, 64, dtype=c.dtype, device=DEV), c.codes.to(DEV),
                             c.scales.to(DEV), c.table.to(DEV), c.ctx.to(DEV), 1.0, 34, 2, 64)
    with pytest.raises(ValueError, match="max_seqlen"):
        ops.varlen_prefill_fp8(c.q.to(DEV), c.codes.to(DEV), c.scales.to(DEV), c.table.to(DEV),
                               c.cu.to(DEV), c.ctx.to(DEV), 0, 1.0, 8, 2, 64)
    with pytest.raises(ValueError, match="out must be"):
        c.run(out=torch.empty(4, 8, 64, device=DEV))
    assert c.run(q=c.q[:0].to(DEV)).shape == (0, 8, 64)
