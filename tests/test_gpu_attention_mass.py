"""Attention that adds up its weights, on the GPU against the definition in float64.

Outputs: the bound of test_gpu_tree_attention.py.  A weight p is exp(s - lse): s, made once for lse and
once for p, is a sum of D products in fp32 with two more roundings, off by (D + 8) 2^-24 of
scale sum_d |q_d k_d|; the exponentials and the denominator's sums and merge add 2^-20 + n 2^-23
(n keys), the denominator's logarithm 2^-23 of its size, which the exponential turns into as much of
p; 2^-20 covers it up to |lse| = 8, past it |lse| 2^-22.  A sum of m weights and decay times what was
there add (m + 2) 2^-24 of it.
"""
import math

import pytest
import torch

from needle_amd import ops
from oracle import tree_ref
from test_gpu_tree_attention import Case as TreeCase
from test_gpu_tree_attention import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float16]


class Case(TreeCase):
    """The chunks of a causal attention; the weights so far are random, NaN where nothing is cached."""

    def __init__(self, shape, counts, lens, dtype=torch.bfloat16, seed=0, **more):
        see = [torch.ones(n, n, dtype=torch.bool).tril() for n in counts]
        super().__init__(shape, counts, lens, dtype, seed, see=see, **more)
        self.before = torch.full((self.nb, self.hkv, self.bs), math.nan)
        for i, n in enumerate(lens):
            p = torch.arange(max(n, 0))
            at = self.table[i].long()[(p // self.bs).clamp(max=self.table.shape[1] - 1)]
            self.before[at, :, p % self.bs] = torch.rand(len(p), self.hkv, generator=self.gen) * 3

    def run(self, decode=False, q=None, mass=None, **more):
        mass = self.before.to(DEV) if mass is None else mass
        if not decode:
            more = dict(cu_seqlens=self.cu.to(DEV), max_seqlen=max(max(self.counts), 1)) | more
        out = ops.attention_mass(self.q.to(DEV) if q is None else q, self.pool.to(DEV),
                                 self.table.to(DEV), self.ctx.to(DEV), mass, self.scale, self.h,
                                 self.hkv, self.d, **more)
        return out, mass

    def check(self, got, decay=1.0):
        out, mass = got
        r = tree_ref.attention(self.q, self.pool, self.table, self.cu, self.ctx, self.scale)
        check(out, r, self.dtype, self.d, int(self.cu[-1]))
        want = tree_ref.mass(r, self.before, self.cu, self.ctx, self.h, decay)
        got = mass.cpu().double()
        assert torch.equal(got.isnan(), want.isnan())
        bound = torch.zeros_like(want)
        for i, (pos, blk, row) in r.at.items():
            p = r.probs[i]
            a, n = int(self.cu[i]), p.shape[0]
            big, keys = r.big[a:a + n, :, None], r.lens[a:a + n, None, None]
            rel = 2 * (self.d + 8) * 2.0 ** -24 * big + 2.0 ** -20 + keys * 2.0 ** -23 \
                + big * 2.0 ** -22
            b = (p * rel).view(n, self.hkv, -1, p.shape[2]).sum((0, 2))
            b = b + (n * self.h // self.hkv + 2) * 2.0 ** -24 \
                * want[blk, :, row].T.nan_to_num(0.0) + 1e-37
            for x in range(len(pos)):
                bound[blk[x], :, row[x]] = b[:, x]
        off = (got - want).abs().nan_to_num(0.0)
        worst = (off / bound.clamp(min=1e-300)).nan_to_num(0.0).max()
        assert worst <= 1.0, float(worst)


SHAPES = [(14, 2, 64, 16), (32, 8, 128, 16), (28, 4, 128, 64), (16, 1, 128, 32), (3, 3, 64, 1024),
          (10, 2, 64, 256), (13, 1, 128, 16)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_decode(shape, dtype):
    lens = [0, 1, 14, 15, 16, 31, 32, 63, 100, 129, 257, -1, -5]
    c = Case(shape, [1] * len(lens), lens, dtype, seed=1)
    c.check(c.run(decode=True))
    c.check(c.run(decode=True, decay=0.75), 0.75)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("counts", [[1, 2, 0, 3], [5, 1, 8, 4], [16, 3, 32, 1], [150, 0, 33]])
def test_chunks(shape, dtype, counts):
    lens = [37, 0, 250, 15][:len(counts)]
    c = Case(shape, counts, lens, dtype, seed=2)
    c.check(c.run())
    c.ctx[0] = -2                     # attends nothing: its weights stay as they are
    c.check(c.run())


@pytest.mark.parametrize("shape", [(14, 2, 64, 16), (32, 8, 128, 16), (7, 1, 128, 64)])
@pytest.mark.parametrize("counts", [[1, 1, 1], [3, 1, 6], [40, 30, 1]])
def test_shares_and_merge(shape, counts):
    c = Case(shape, counts, [2900, 3, 1111], seed=3)
    c.check(c.run(decode=max(counts) == 1))
    c.check(c.run(max_context_len=2900))


def test_a_decay_of_zero_forgets():
    for counts in ([1, 1], [70, 2]):
        c = Case((8, 2, 128, 16), counts, [300, 45], seed=4)
        c.before[:] = math.nan
        c.check(c.run(decay=0.0), 0.0)


def test_many_steps_add_up():
    """A prompt's chunk and decode steps one after the other, against one chunk over all: every
    token's weights summed, from its own step on."""
    c = Case((8, 2, 64, 16), [120], [0], seed=5)
    total, _ = c.run()[1], None
    mass = c.before.to(DEV).zero_()
    at = 0
    for n in (60, 1, 1, 30, 1, 27):
        cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
        ops.attention_mass(c.q[at:at + n].to(DEV), c.pool.to(DEV), c.table.to(DEV),
                           torch.tensor([at], dtype=torch.int32, device=DEV), mass, c.scale, 8, 2,
                           64, cu_seqlens=cu, max_seqlen=n)
        at += n
    p = torch.arange(120)
    blk = c.table[0].long()[p // 16]
    a, b = (x.cpu()[blk, :, p % 16] for x in (mass, total))
    assert torch.allclose(a, b, rtol=1e-4, atol=1e-6) and abs(float(a.sum()) - 120 * 8) < 1e-2


def test_a_window_is_the_last_tokens_of_a_prompt():
    c = Case((28, 4, 128, 16), [32, 32], [400, 1700], seed=6)
    c.check(c.run())
    c.check(c.run(max_context_len=1700))


def test_blocks_that_are_not_valid_and_tables_too_short():
    for counts in ([1, 1, 1], [40, 2, 9]):
        c = Case((8, 2, 64, 16), counts, [45, 1900, 40], seed=7)
        c.table[0, 1], c.table[1, 0], c.table[1, 77], c.table[2] = -1, c.nb, 1 << 30, -5
        c.check(c.run())
        c = Case((8, 2, 64, 16), counts, [45, 90, 40], seed=8, extra_cols=0)
        c.table = c.table[:, :3].contiguous()
        c.check(c.run())


def test_values_that_are_not_finite():
    for counts in ([1, 1], [50, 3]):
        c = Case((8, 2, 64, 16), counts, [45, 300], seed=9)
        p = 45 + counts[0] - 1
        c.pool[1, int(c.table[0, p // 16]), 0, p % 16, 5] = math.inf
        c.pool[0, int(c.table[1, 3]), 1, 7, 9] = math.nan        # a cached key: its kv head's rows
        c.check(c.run())


def test_strides_outputs_and_rows_outside():
    c = Case((14, 2, 64, 16), [7, 3], [33, 0], seed=11)
    want, mass = c.run()
    wide = torch.randn(13, 18 * 64, generator=c.gen).to(c.dtype)
    wide[2:12, :14 * 64] = c.q.view(10, -1)
    out = torch.full((13, 14, 64), 7.0, dtype=c.dtype, device=DEV)
    c.cu += 2
    got, mass2 = c.run(q=wide.to(DEV)[:, :14 * 64].view(13, 14, 64), out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got[2:12], want)
    assert (got[:2] == 7).all() and (got[12:] == 7).all()
    assert torch.equal(mass.view(torch.int32), mass2.view(torch.int32))


@pytest.mark.parametrize("scale", [0.0, -0.11])
def test_scales_of_zero_and_less(scale):
    for counts in ([1, 1], [60, 3]):
        c = Case((8, 2, 64, 16), counts, [45, 1900], seed=12)
        c.scale = scale
        c.check(c.run())


def test_workspace_large_scores_and_the_same_again():
    for counts in ([1, 1], [40, 9]):
        c = Case((8, 2, 128, 16), counts, [1800, 3000], torch.float16, seed=13)
        c.q *= 12
        need = ops.attention_mass_workspace_bytes(2, sum(counts), max(counts),
                                                  c.table.shape[1] * 16, 8, 2, 128)
        ws = torch.full((need,), 0xFF, dtype=torch.uint8, device=DEV)
        got = c.run(workspace=ws)
        c.check(got)
        ws.fill_(0x7F)
        again = c.run(workspace=ws)
        assert torch.equal(got[0], again[0])
        assert torch.equal(got[1].view(torch.int32), again[1].view(torch.int32))


def test_captured_into_a_graph():
    c = Case((32, 8, 128, 16), [1] * 4, [700, 60, 2000, 0], seed=14)
    dev = dict(q=c.q.to(DEV), mass=c.before.to(DEV))
    args = (c.pool.to(DEV), c.table.to(DEV), c.ctx.to(DEV))

    def step():
        return ops.attention_mass(dev["q"], *args, dev["mass"], c.scale, 32, 8, 128)
    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for seed in (1, 2, 3):
        new = torch.randn(c.q.shape, generator=torch.Generator().manual_seed(seed)).to(c.dtype)
        dev["q"].copy_(new)
        dev["mass"].copy_(c.before)
        g.replay()
        got = (out.clone(), dev["mass"].clone())
        dev["mass"].copy_(c.before)
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want)
        assert torch.equal(got[1].view(torch.int32), dev["mass"].view(torch.int32))


def test_refusals():
    c = Case((8, 2, 64, 16), [1, 1], [4, 0])
    m = c.before.to(DEV)
    for bad in (dict(mass=m.half()), dict(q=c.q.float().to(DEV))):
        with pytest.raises(TypeError):
            c.run(decode=True, **bad)
    for bad in (dict(mass=m[:2]), dict(mass=c.before), dict(mass=m.transpose(1, 2)),
                dict(max_seqlen=2), dict(q=c.q[:1].to(DEV)), dict(max_context_len=-1)):
        with pytest.raises(ValueError):
            c.run(decode=True, **bad)
    with pytest.raises(ValueError):
        c.run(max_seqlen=0)
    assert c.run(cu_seqlens=torch.zeros(3, dtype=torch.int32, device=DEV),
                 q=torch.empty(0, 8, 64, dtype=c.dtype, device=DEV))[0].shape == (0, 8, 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts", [[1, 1, 1], [2, 1, 2], [30, 4, 9]])
def test_contexts_past_the_bound_of_a_call(counts, dtype):
    """Keys past max_context_len + max_seqlen get no weight, and nothing is written past the
    workspace."""
    c = Case((32, 8, 128, 16), counts, [700, 20, 1900], dtype, seed=21)
    bound, most = 100, max(counts)
    need = ops.attention_mass_workspace_bytes(3, sum(counts), most, bound + most, c.h, c.hkv, c.d,
                                              c.bs)
    ws = torch.full((need + (4 << 20),), 0xA5, dtype=torch.uint8, device=DEV)
    out, mass = c.run(max_context_len=bound, workspace=ws)
    assert (ws[need:] == 0xA5).all()
    r = tree_ref.attention(c.q, c.pool, c.table, c.cu, c.ctx, c.scale)
    check(out, r, c.dtype, c.d, int(c.cu[-1]))
    want = tree_ref.mass(r, c.before, c.cu, c.ctx, c.h)
    mass = mass.cpu()
    for i, n in enumerate(c.lens):
        p = torch.arange(n + counts[i])
        blk = c.table[i].long()[p // 16]
        inside = p < bound + most
        got, old = mass[blk, :, p % 16], c.before[blk, :, p % 16]
        same = (got == old) | (got.isnan() & old.isnan())
        assert same[~inside].all()
        torch.testing.assert_close(got[inside].double(), want[blk, :, p % 16][inside],
                                   rtol=2.0 ** -10, atol=1e-6)
