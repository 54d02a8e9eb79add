"""Masks of drafted trees and attention under them on the GPU, over pools in 16 and 8 bits, against
the definition in float64.

The bound of every output element, from the roundings made on the way (u: half a step of the
16-bit format, 2^-8 or 2^-11): the probabilities and the output are rounded once each, u (A + |o|)
with A = sum_t p_t |v_t|; a score is a sum of D products in fp32 with two more roundings, off by
(D + 8) 2^-24 of scale sum_d |q_d k_d|, which enters a probability's numerator and denominator;
the exponentials, the running sums and the merge add 2^-20 + n 2^-23.  float16 probabilities
below 2^-14 are subnormal, each off by 2^-25 where the largest is at least 1 (times the largest
value, 32 at most here); so are outputs below 2^-14, by 2^-25.
"""
import math

import pytest
import torch

from needle_amd import ops
from oracle import tree_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float16]


def random_tree(n, gen):
    """Parents of n nodes: mostly few branches, now and then a second root."""
    p = [-1][:n]
    for t in range(1, n):
        x = int(torch.randint(max(0, t - 6), t, (1,), generator=gen))
        p.append(-1 if torch.rand(1, generator=gen) < 0.05 else x)
    return p


def attention_bound(r, dtype, d):
    u = torch.finfo(dtype).eps / 2
    rel = 2 * (d + 8) * 2.0 ** -24 * r.big[..., None] + 2.0 ** -20 \
        + r.lens[:, None, None] * 2.0 ** -23
    bound = u * (r.weight + r.out.abs()) + rel * r.weight
    if dtype == torch.float16:
        bound = bound + r.lens[:, None, None] * 2.0 ** -25 * 32 + 2.0 ** -25
    return bound


def check(got, r, dtype, d, rows):
    got, want = got.double().cpu()[:rows], r.out[:rows]
    bound = attention_bound(r, dtype, d)[:rows]
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()],
                                                                  want[want.isinf()])
    fine = want.isfinite()
    off = (got - want).abs()[fine]
    worst = (off / bound[fine].clamp(min=1e-300)).max() if off.numel() else 0.0
    assert worst <= 1.0, float(worst)


class Case:
    """Trees of `counts` nodes after `lens` cached tokens.  Rows that no sequence holds are NaN."""

    def __init__(self, shape, counts, lens, dtype=torch.bfloat16, seed=0, fp8=False, extra_cols=1,
                 see=None):
        self.h, self.hkv, self.d, self.bs = shape
        self.dtype, self.counts, self.lens = dtype, counts, lens
        gen = self.gen = torch.Generator().manual_seed(seed)
        need = [max(1, -(-(max(c, 0) + n) // self.bs)) for c, n in zip(lens, counts)]
        self.nb = sum(need) + 3
        perm = torch.randperm(self.nb - 1, generator=gen)
        self.table = torch.full((len(lens), max(need) + extra_cols), self.nb - 1,
                                dtype=torch.int32)
        shape5 = (2, self.nb, self.hkv, self.bs, self.d)
        if fp8:
            codes = torch.full(shape5, 0x7F, dtype=torch.uint8)
            scales = torch.full(shape5[:4], 254, dtype=torch.uint8)
            self.pool = (codes, scales)
        else:
            self.pool = torch.full(shape5, math.nan, dtype=dtype)
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
            if fp8:
                c = torch.randint(0, 256, (total, 2, self.hkv, self.d), generator=gen,
                                  dtype=torch.uint8)
                c[(c & 127) > 117] = 0x31          # within 224, no NaN
                codes[:, blk, :, row] = c
                scales[:, blk, :, row] = torch.randint(118, 124, (total, 2, self.hkv),
                                                       generator=gen, dtype=torch.uint8)
            else:
                x = torch.randn(total, 2, self.hkv, self.d, generator=gen).clamp(-8, 8)
                self.pool[:, blk, :, row] = x.to(dtype)
        self.cu = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32)
        self.ctx = torch.tensor(lens, dtype=torch.int32)
        self.q = torch.randn(int(self.cu[-1]), self.h, self.d, generator=gen).to(dtype)
        self.scale = 1.0 / self.d ** 0.5
        self.parents = [random_tree(n, gen) for n in counts]
        self.see = [tree_ref.sees(p) for p in self.parents] if see is None else see
        self.words = max(1, (max(counts) + 63) // 64)
        self.mask = torch.cat([tree_ref.mask_words(s, self.words) for s in self.see])

    def want(self):
        return tree_ref.attention(self.q, self.pool, self.table, self.cu, self.ctx, self.scale,
                                  lambda i: self.see[i])

    def device_pool(self):
        if torch.is_tensor(self.pool):
            return self.pool.to(DEV)
        return ops.Fp8KVCache(self.pool[0].to(DEV).view(torch.float8_e4m3fn),
                              self.pool[1].to(DEV))

    def run(self, q=None, mask=None, max_seqlen=None, **more):
        return ops.tree_attention(self.q.to(DEV) if q is None else q, self.device_pool(),
                                  self.table.to(DEV), self.cu.to(DEV), self.ctx.to(DEV),
                                  self.mask.to(DEV) if mask is None else mask,
                                  max_seqlen or max(max(self.counts), 1), self.scale, self.h,
                                  self.hkv, self.d, **more)

    def check(self, got):
        check(got, self.want(), self.dtype, self.d, int(self.cu[-1]))


# ---------------------------------------------------------------- masks

@pytest.mark.parametrize("counts", [[1], [5, 1, 0, 64], [65, 130, 3], [256, 257], [700]])
def test_masks(counts):
    gen = torch.Generator().manual_seed(3)
    trees = [random_tree(n, gen) for n in counts]
    chain = list(range(-1, counts[-1] - 1))
    for last in (trees[-1], chain):
        trees[-1] = last
        cu = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32)
        parents = torch.tensor(sum(trees, []), dtype=torch.int32)
        mask, depth = ops.tree_mask(parents.to(DEV), cu.to(DEV), max(counts))
        words = (max(counts) + 63) // 64
        see = [tree_ref.sees(p) for p in trees]
        assert torch.equal(mask.cpu(), torch.cat([tree_ref.mask_words(s, words) for s in see]))
        assert depth.cpu().tolist() == [int(x) - 1 for s in see for x in s.sum(1)]


def test_masks_of_bad_parents():
    """The node itself, a later one, a number out of range: no parent."""
    parents = [0, 1, 0, 5, 2, -7, 3, 1 << 30, -(1 << 31), 8]
    cu = torch.tensor([0, len(parents)], dtype=torch.int32)
    mask, depth = ops.tree_mask(torch.tensor(parents, dtype=torch.int32).to(DEV), cu.to(DEV), 10)
    see = tree_ref.sees(parents)
    assert torch.equal(mask.cpu(), tree_ref.mask_words(see, 1))
    assert depth.tolist() == (see.sum(1) - 1).tolist() == [0, 0, 1, 0, 2, 0, 1, 0, 0, 1]


def test_masks_of_a_tree_past_what_is_held():
    n = 9000
    gen = torch.Generator().manual_seed(5)
    parents = [-1] + [int(torch.randint(t // 2, t, (1,), generator=gen)) for t in range(1, n)]
    cu = torch.tensor([0, n], dtype=torch.int32)
    mask, depth = ops.tree_mask(torch.tensor(parents, dtype=torch.int32).to(DEV), cu.to(DEV), n)
    mask, depth = mask.cpu(), depth.tolist()
    for t in (0, 1, 63, 64, 4095, 4096, 5000, n - 1):
        at, nodes = t, []
        while at is not None:
            nodes.append(at)
            at = tree_ref.parent_of(parents, at)
        see = torch.zeros(1, n, dtype=torch.bool)
        see[0, nodes] = True
        assert torch.equal(mask[t:t + 1], tree_ref.mask_words(see, mask.shape[1]))
        assert depth[t] == len(nodes) - 1


def test_masks_within_the_bound_of_a_call():
    """Words for fewer nodes than a sequence has: the first nodes' bits; rows outside stay."""
    gen = torch.Generator().manual_seed(6)
    tree = random_tree(100, gen)
    parents = torch.tensor([7, 7] + tree + [7], dtype=torch.int32).to(DEV)
    cu = torch.tensor([2, 102], dtype=torch.int32).to(DEV)
    mask, depth = ops.tree_mask(parents, cu, 64)
    assert torch.equal(mask[2:102].cpu(), tree_ref.mask_words(tree_ref.sees(tree), 1))


# ---------------------------------------------------------------- attention

SHAPES = [(14, 2, 64, 16), (32, 8, 128, 16), (28, 4, 128, 64), (16, 1, 128, 32), (3, 3, 64, 1024),
          (10, 2, 64, 256), (13, 1, 128, 16)]
POOLS = [False, True]


@pytest.mark.parametrize("fp8", POOLS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("counts", [[1, 2, 0, 3], [5, 1, 8, 4], [16, 3, 32, 1], [70, 0, 33]])
def test_trees(shape, dtype, counts, fp8):
    lens = [37, 0, 250, 15][:len(counts)]
    c = Case(shape, counts, lens, dtype, seed=2, fp8=fp8)
    c.check(c.run())
    c.ctx[0] = -2                     # attends nothing
    got = c.run()
    c.check(got)
    assert not got[:counts[0]].any()


@pytest.mark.parametrize("fp8", POOLS)
@pytest.mark.parametrize("shape", [(14, 2, 64, 16), (32, 8, 128, 16), (7, 1, 128, 64)])
@pytest.mark.parametrize("counts", [[1, 1, 1], [3, 1, 6], [17, 9, 2], [64, 30, 1], [140, 2, 50]])
def test_shares_and_merge(shape, counts, fp8):
    """Contexts long enough for the split into shares, of very different lengths."""
    c = Case(shape, counts, [2900, 3, 1111], seed=3, fp8=fp8)
    assert ops.tree_attention_workspace_bytes(3, max(counts), c.table.shape[1] * c.bs, c.h, c.hkv,
                                              c.d, c.bs, fp8) > 0
    c.check(c.run())
    c.check(c.run(max_context_len=2900))


@pytest.mark.parametrize("fp8", POOLS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_any_mask(dtype, fp8):
    """Masks that are no tree: later nodes, not the token itself, nothing at all; bits of nodes that
    the sequence has not."""
    gen = torch.Generator().manual_seed(8)
    counts, lens = [40, 7, 70], [0, 21, 64]
    see = [torch.rand(n, n, generator=gen) < 0.3 for n in counts]
    see[0][3] = see[0][17] = False           # with no context: nothing to attend
    see[1][2] = False                        # the context alone
    c = Case((8, 2, 64, 16), counts, lens, dtype, seed=9, fp8=fp8, see=see)
    got = c.run()
    c.check(got)
    assert not got[3].any() and not got[17].any() and got[42].any()
    mask = c.mask.clone()
    mask[40:47] |= -(1 << 7)                 # sequence 1 has seven nodes
    assert torch.equal(c.run(mask=mask.to(DEV)), got)
    wide = torch.cat([c.mask, torch.full((117, 3), -1, dtype=torch.int64)], 1).to(DEV)
    assert torch.equal(c.run(mask=wide), got)
    strided = wide[:, :2]
    assert strided.stride(0) == 5 and torch.equal(c.run(mask=strided), got)
    # fewer words than nodes: those past them are not seen
    for i, s in enumerate(c.see):
        s[:, 64:] = False
    narrow = c.mask[:, :1].contiguous().to(DEV)
    c.check(c.run(mask=narrow))


def test_a_chain_is_a_causal_chunk():
    counts, lens = [9, 1, 33], [100, 0, 700]
    for fp8 in POOLS:
        see = [torch.ones(n, n, dtype=torch.bool).tril() for n in counts]
        c = Case((32, 8, 128, 16), counts, lens, seed=4, fp8=fp8, see=see)
        got = c.run()
        c.check(got)
        args = (c.table.to(DEV), c.cu.to(DEV), c.ctx.to(DEV), 33, c.scale, 32, 8, 128)
        pool = c.device_pool()
        if fp8:
            want = ops.varlen_prefill_fp8(c.q.to(DEV), *pool, *args)
        else:
            want = ops.varlen_prefill(c.q.to(DEV), pool, *args, max_context_len=700)
        bound = 2 * attention_bound(c.want(), c.dtype, 128)
        assert ((got.double() - want.double()).abs().cpu() <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts", [[6, 12], [50, 20], [140, 3]])
def test_values_that_are_not_finite(dtype, counts):
    """Infinities and NaN in the nodes' V reach the tokens that attend them and no others; in K
    they make NaN of those."""
    for d in (64, 128):
        c = Case((8, 2, d, 16), counts, [45, 300], dtype, seed=6)
        bad = [(0, 2, math.inf), (0, 2, -math.inf), (0, 4, math.nan), (1, 1, -math.inf),
               (1, 2, math.inf), (0, 3, math.inf)]
        for x, (i, node, value) in enumerate(bad):
            p = c.lens[i] + node
            blk = int(c.table[i, p // 16])
            c.pool[1, blk, x % 2, p % 16, 5 * x % d] = value
        # one column with both infinities in two nodes
        for node, value in ((1, math.inf), (5, -math.inf)):
            p = c.lens[0] + node
            c.pool[1, int(c.table[0, p // 16]), 1, p % 16, 33] = value
        p = c.lens[1] + counts[1] - 1        # a leaf's key
        c.pool[0, int(c.table[1, p // 16]), 0, p % 16, 3] = math.nan
        r = c.want()
        assert r.out.isnan().any() and (r.out == math.inf).any() and (r.out == -math.inf).any()
        assert r.out.isfinite().float().mean() > 0.8
        c.check(c.run())


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_codes_of_nodes(dtype):
    """The 8-bit pool has NaN alone."""
    c = Case((8, 2, 128, 16), [6, 12], [45, 300], dtype, seed=6, fp8=True)
    for x, (i, node) in enumerate([(0, 2), (0, 4), (1, 1), (1, 7)]):
        p = c.lens[i] + node
        c.pool[0][1, int(c.table[i, p // 16]), x % 2, p % 16, 5 * x] = 0x7F
    r = c.want()
    assert 0.0 < r.out.isnan().float().mean() < 0.05
    c.check(c.run())


@pytest.mark.parametrize("fp8", POOLS)
def test_blocks_that_are_not_valid(fp8):
    c = Case((8, 2, 64, 16), [6, 20, 3], [45, 1900, 40], seed=7, fp8=fp8)
    c.table[0, 1] = -1
    c.table[1, 0] = c.nb
    c.table[1, 77] = 1 << 30
    c.table[2] = -5
    got = c.run()
    c.check(got)
    assert not got[26:].any()


@pytest.mark.parametrize("fp8", POOLS)
def test_trees_past_the_table(fp8):
    """Positions past the table's width are not attended."""
    c = Case((8, 2, 64, 16), [30, 12], [40, 5], seed=7, fp8=fp8, extra_cols=0)
    c.table = c.table[:, :4].contiguous()
    c.check(c.run())


@pytest.mark.parametrize("fp8", POOLS)
def test_strides_and_outputs(fp8):
    """q as a view of a fused projection; tokens before and behind the sequences."""
    c = Case((14, 2, 64, 16), [7, 3], [33, 0], seed=11, fp8=fp8)
    want = c.run()
    wide = torch.randn(10, 18 * 64, generator=c.gen).to(c.dtype)
    wide[:, :14 * 64] = c.q.view(10, -1)
    assert torch.equal(c.run(q=wide.to(DEV)[:, :14 * 64].view(10, 14, 64)), want)
    out = torch.full((15, 14, 64), 7.0, dtype=c.dtype, device=DEV)
    c.cu += 2
    c.q = torch.cat([c.q[:2], c.q, c.q[:3]])
    mask = torch.cat([c.mask[:2], c.mask, c.mask[:3]])
    got = c.run(mask=mask.to(DEV), out=out)
    assert got.data_ptr() == out.data_ptr()
    assert torch.equal(got[2:12], want) and (got[:2] == 7).all() and (got[12:] == 7).all()


@pytest.mark.parametrize("scale", [0.0, -0.11])
@pytest.mark.parametrize("fp8", POOLS)
def test_scales_of_zero_and_less(scale, fp8):
    c = Case((8, 2, 64, 16), [6, 20], [45, 1900], seed=12, fp8=fp8)
    c.scale = scale
    c.check(c.run())


def test_workspace_reuse_and_large_scores():
    """A given workspace; scores of a few hundred, whose maximum rises on the way."""
    c = Case((8, 2, 128, 16), [9, 20], [1800, 3000], torch.float16, seed=13)
    c.q *= 12
    need = ops.tree_attention_workspace_bytes(2, 20, c.table.shape[1] * 16, 8, 2, 128)
    assert need > 0
    ws = torch.full((need,), 0xFF, dtype=torch.uint8, device=DEV)
    got = c.run(workspace=ws)
    c.check(got)
    ws.fill_(0x7F)
    assert torch.equal(c.run(workspace=ws), got)


def test_many_sequences():
    gen = torch.Generator().manual_seed(1)
    n = 300
    counts = torch.randint(0, 6, (n,), generator=gen).tolist()
    lens = torch.randint(0, 90, (n,), generator=gen).tolist()
    lens[7], lens[200] = 2500, 1700
    c = Case((4, 1, 64, 16), counts, lens, seed=14)
    c.check(c.run())
    c.check(c.run(max_context_len=2500))


def test_empty_calls():
    c = Case((8, 2, 64, 16), [3], [4])
    assert c.run(q=torch.empty(0, 8, 64, dtype=c.dtype, device=DEV),
                 mask=torch.empty(0, 1, dtype=torch.int64, device=DEV)).shape == (0, 8, 64)
    mask, depth = ops.tree_mask(torch.empty(0, dtype=torch.int32, device=DEV),
                                torch.zeros(3, dtype=torch.int32, device=DEV), 4)
    assert mask.shape == (0, 1) and depth.shape == (0,)


def test_refusals():
    c = Case((8, 2, 64, 16), [3, 2], [4, 0])
    with pytest.raises(TypeError):
        c.run(mask=c.mask.int().to(DEV))
    with pytest.raises(ValueError):
        c.run(mask=c.mask[:4].to(DEV))
    with pytest.raises(ValueError):
        c.run(mask=c.mask[:, :0].to(DEV))
    with pytest.raises(ValueError):
        c.run(mask=c.mask)
    with pytest.raises(TypeError):
        c.run(q=c.q.float().to(DEV))
    with pytest.raises(TypeError):
        c.run(q=c.q.half().to(DEV))
    with pytest.raises(ValueError):
        c.run(max_seqlen=-1)
    with pytest.raises(ValueError):
        c.run(out=torch.empty(5, 8, 32, dtype=c.dtype, device=DEV))
    with pytest.raises(TypeError):
        ops.tree_mask(torch.zeros(3, dtype=torch.int64, device=DEV), c.cu.to(DEV), 3)
    with pytest.raises(ValueError):
        ops.tree_mask(torch.zeros(3, dtype=torch.int32), c.cu, 3)
    with pytest.raises(ValueError):
        ops.tree_mask(torch.zeros(3, dtype=torch.int32, device=DEV), c.cu.to(DEV), 0)
