"""Rows of a cache that stay: which (kv_select) and moved together (kv_compact), against the
definitions, exactly."""
import math

import pytest
import torch

from needle_amd import ops
from oracle import tree_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


class Cache:
    """Sequences of `lens` rows in blocks of bs; `spare` blocks that no sequence holds."""

    def __init__(self, lens, hkv=2, bs=16, seed=0, spare=0, extra_cols=1):
        self.gen = torch.Generator().manual_seed(seed)
        need = [max(1, -(-n // bs)) for n in lens]
        self.nb, self.hkv, self.bs, self.lens = sum(need) + 2 + spare, hkv, bs, lens
        perm = torch.randperm(self.nb - 1, generator=self.gen).tolist()
        self.table = torch.full((len(lens), max(need) + extra_cols), self.nb - 1,
                                dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = i32(perm[at:at + n])
            at += n
        self.free = perm[at:at + spare]

    def pool(self, dtype, d=64):
        shape = (2, self.nb, self.hkv, self.bs, d)
        if dtype == "fp8":
            return (torch.randint(0, 256, shape, generator=self.gen, dtype=torch.uint8),
                    torch.randint(0, 256, shape[:4], generator=self.gen, dtype=torch.uint8))
        return torch.randn(shape, generator=self.gen).to(dtype)

    def mass(self):
        return torch.rand((self.nb, self.hkv, self.bs), generator=self.gen)


def on_device(pool):
    if torch.is_tensor(pool):
        return pool.to(DEV)
    return ops.Fp8KVCache(pool[0].to(DEV).view(torch.float8_e4m3fn), pool[1].to(DEV))


def raw(x):
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def check_compact(c, pools, keep, counts, first=None, cu=None, dst=None, mass=None, table=None):
    table = c.table if table is None else table
    dev = [on_device(p) for p in pools]
    m = None if mass is None else mass.to(DEV)

    def put(x):
        return None if x is None else x.to(DEV)
    ops.kv_compact(dev, table.to(DEV), keep.to(DEV), counts.to(DEV), first=put(first),
                   cu_seqlens=put(cu), dst_table=put(dst), mass=m)
    parts = [(x, 1) for p in pools for x in ((p,) if torch.is_tensor(p) else p)]
    if mass is not None:
        parts.append((mass, 0))
    tree_ref.compact(parts, table, keep, counts, first, cu, dst)
    got = [x for p in dev for x in ((p,) if torch.is_tensor(p) else p)] + ([m] if m is not None
                                                                           else [])
    for x, (y, _) in zip(got, parts):
        assert torch.equal(raw(x).cpu().view(torch.uint8), y.view(torch.uint8))


def ascending(n, k, gen):
    return torch.randperm(n, generator=gen)[:k].sort().values.to(torch.int32)


DTYPES = [torch.bfloat16, torch.float16, torch.float32, "fp8"]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bs", [16, 64])
def test_paths_of_trees(dtype, d, bs):
    """Lists shared by the kv heads and layers, behind the cached tokens, in place."""
    ctx, nodes = [5, 0, 100, 63, 16], [20, 7, 64, 1, 130]
    c = Cache([a + b for a, b in zip(ctx, nodes)], hkv=3, bs=bs, seed=1)
    cu = i32([0] + torch.tensor(nodes).cumsum(0).tolist())
    keep = torch.full((sum(nodes),), -1, dtype=torch.int32)
    counts = [6, 7, 30, 1, 130]
    for i, (n, k) in enumerate(zip(nodes, counts)):
        keep[int(cu[i]):int(cu[i]) + k] = ascending(n, k, c.gen)
    check_compact(c, [c.pool(dtype, d) for _ in range(4)], keep, i32(counts), first=i32(ctx), cu=cu)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("most", [30, 64, 65, 300, 2000])
def test_lists_of_heads_in_place(dtype, most):
    """Each kv head's own list; overlapping sources and places; the weights move too."""
    lens = [most + 50, most, 3 * most, 17]
    c = Cache(lens, hkv=2, bs=32, seed=most)
    counts = [most, most, most, 17]
    keep = torch.full((4, 2, most), -1, dtype=torch.int32)
    for i in range(4):
        for h in range(2):
            keep[i, h, :counts[i]] = ascending(lens[i], counts[i], c.gen)
    check_compact(c, [c.pool(dtype)], keep, i32(counts), mass=c.mass())
    counts = [most // 2, 0, 3, 5]
    check_compact(c, [c.pool(dtype)], keep, i32(counts))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("most", [1, 40, 500])
def test_lists_of_heads_into_other_blocks(dtype, most):
    lens = [most + 50, most, 2 * most + 3]
    c = Cache(lens, hkv=4, bs=16, seed=5, spare=3 * (most // 16 + 1))
    cols = most // 16 + 1
    dst = i32(c.free).view(3, cols)
    keep = torch.full((3, 4, most), -1, dtype=torch.int32)
    for i in range(3):
        for h in range(4):          # any order here
            keep[i, h] = torch.randperm(lens[i], generator=c.gen)[:most].to(torch.int32)
    check_compact(c, [c.pool(dtype, 128) for _ in range(2)], keep, i32([most, most, most]),
                  dst=dst, mass=c.mass())


def test_entries_that_move_nothing():
    """Negative entries, positions past the tables, invalid blocks, negative starts, counts past the
    list."""
    c = Cache([60, 60, 60, 60], hkv=2, bs=16, seed=3, extra_cols=0)
    c.table[1, 1] = -1
    c.table[2, 3] = c.nb
    c.table[2, 0] = 1 << 30
    keep = torch.full((4, 2, 12), -1, dtype=torch.int32)
    keep[:, :, :8] = i32([0, 3, -5, 17, 20, 50, 63, 1 << 20])
    for first in (None, i32([0, 2, 5, -1]), i32([55, 60, 1 << 30, 3])):
        check_compact(c, [c.pool(torch.bfloat16)], keep, i32([8, 8, 8, 99]), first=first,
                      mass=c.mass())


def test_blocks_of_any_size_and_rows_of_any_width():
    c = Cache([100, 31], hkv=1, bs=24, seed=4)
    keep = torch.stack([ascending(100, 20, c.gen), ascending(31, 20, c.gen)]).view(2, 1, 20)
    check_compact(c, [c.pool(torch.float16, 24)], keep.contiguous(), i32([20, 20]))
    with pytest.raises(ValueError):
        ops.kv_compact([c.pool(torch.float16, 20).to(DEV)], c.table.to(DEV),
                       keep.contiguous().to(DEV), i32([1, 1]).to(DEV))


def test_many_layers_and_a_pool_past_4_gib():
    c = Cache([40], hkv=8, bs=16, seed=6)
    keep = ascending(30, 9, c.gen)
    check_compact(c, [c.pool(torch.bfloat16, 128) for _ in range(128)], keep, i32([9]),
                  first=i32([8]), cu=i32([0, 9]))
    # blocks whose rows lie past 2^32 bytes of a plane
    nb, hkv, bs, d = 140000, 8, 16, 128
    pool = torch.empty((2, nb, hkv, bs, d), dtype=torch.bfloat16, device=DEV)
    table = i32([[nb - 1, 7, nb - 5]]).to(DEV)
    rows = torch.randn(2, 3, hkv, bs, d, device=DEV).to(torch.bfloat16)
    pool[:, table[0].long()] = rows
    keep = i32([3, 20, 40, 47]).to(DEV)
    ops.kv_compact([pool], table, keep, i32([4]).to(DEV), cu_seqlens=i32([0, 4]).to(DEV))
    want = rows.transpose(2, 3).reshape(2, 48, hkv, d).clone()
    want[:, :4] = want[:, [3, 20, 40, 47]]
    got = pool[:, table[0].long()].transpose(2, 3).reshape(2, 48, hkv, d)
    assert torch.equal(got, want)


# ---------------------------------------------------------------- selection

def check_select(mass, table, lens, budget, sinks=0, recent=0):
    keep, kept = ops.kv_select(mass.to(DEV), table.to(DEV), lens.to(DEV), budget, sinks=sinks,
                               recent=recent)
    want = tree_ref.select(mass, table, lens, budget, sinks, recent)
    assert torch.equal(kept.cpu(), want[1])
    assert torch.equal(keep.cpu(), want[0])


@pytest.mark.parametrize("bs", [16, 24, 256])
@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (7, 0, 0), (64, 4, 16), (100, 0, 100),
                                                 (100, 60, 40), (333, 1, 0), (1000, 4, 300)])
def test_select(bs, budget, sinks, recent):
    lens = [0, 1, budget - 1, budget, budget + 1, 2 * budget + 5, 1500]
    c = Cache(lens, hkv=3, bs=bs, seed=budget)
    check_select(c.mass(), c.table, i32(lens), budget, sinks, recent)


@pytest.mark.parametrize("kind", ["zeros", "few values", "signs", "not finite", "close", "powers"])
def test_weights_of_all_kinds(kind):
    lens = [3000, 700, 65, 2049]
    c = Cache(lens, hkv=2, bs=16, seed=9)
    m = c.mass()
    if kind == "zeros":
        m[:] = 0.0
        m[m.flatten()[:1].new_ones(m.shape, dtype=torch.bool)
          & (torch.rand(m.shape, generator=c.gen) < 0.02)] = 0.5
        m[torch.rand(m.shape, generator=c.gen) < 0.3] = -0.0
    elif kind == "few values":
        m = torch.randint(0, 3, m.shape, generator=c.gen).float()
    elif kind == "signs":
        m = m - 0.5
    elif kind == "not finite":
        r = torch.rand(m.shape, generator=c.gen)
        m[r < 0.01], m[(r > 0.5) & (r < 0.51)], m[r > 0.98] = math.nan, math.inf, -math.inf
    elif kind == "close":
        m = (torch.randint(0, 1 << 12, m.shape, generator=c.gen) + (127 << 23)).int().view(
            torch.float32)
    else:
        m = torch.randn(m.shape, generator=c.gen).mul(20).exp2()
    check_select(m, c.table, i32(lens), 600)
    check_select(m, c.table, i32(lens), 64, 3, 10)


def test_tables_with_invalid_blocks_and_lengths_past_them():
    c = Cache([200, 200, 200], hkv=2, bs=16, seed=10, extra_cols=0)
    c.table[0, 3], c.table[1, 0], c.table[1, 5] = -1, c.nb, 1 << 30
    c.table[2] = -7
    check_select(c.mass(), c.table, i32([200, 200, 200]), 50, 2, 5)
    check_select(c.mass(), c.table, i32([-3, 1 << 30, 208]), 190)


def test_select_more_tokens_than_are_held():
    lens = [40000, 38912, 38912 + 70]
    c = Cache(lens, hkv=1, bs=64, seed=12)
    m = (c.mass() * 1000).round()
    check_select(m, c.table, i32(lens), 5000, 4, 60)


def test_select_then_compact():
    """A cache cut to its budget: every kv head attends what it kept."""
    lens, budget = [300, 90, 1000], 128
    c = Cache(lens, hkv=2, bs=16, seed=13)
    pool, mass = c.pool(torch.bfloat16), c.mass()
    d = [x.to(DEV) for x in (pool, mass, c.table, i32(lens))]
    keep, kept = ops.kv_select(d[1], d[2], d[3], budget, sinks=4, recent=32)
    ops.kv_compact([d[0]], d[2], keep, kept, mass=d[1])
    want = tree_ref.select(mass, c.table, i32(lens), budget, 4, 32)
    tree_ref.compact([(pool, 1), (mass, 0)], c.table, want[0], want[1])
    assert torch.equal(d[0].cpu(), pool) and torch.equal(d[1].cpu(), mass)
    # in place a second time, all that is left stays where it is
    ops.kv_compact([d[0]], d[2], *ops.kv_select(d[1], d[2], kept, budget), mass=d[1])
    assert torch.equal(d[0].cpu(), pool) and torch.equal(d[1].cpu(), mass)


def test_captured_into_a_graph():
    lens, budget = [300, 200], 100
    c = Cache(lens, hkv=2, bs=16, seed=14)
    pool, mass = c.pool(torch.bfloat16).to(DEV), c.mass().to(DEV)
    table, n = c.table.to(DEV), i32(lens).to(DEV)

    def step():
        keep, kept = ops.kv_select(mass, table, n, budget, sinks=1, recent=7)
        ops.kv_compact([pool], table, keep, kept, mass=mass)
        return keep, kept
    before = pool.clone()
    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for seed in (1, 2, 3):
        new = torch.rand(mass.shape, generator=torch.Generator().manual_seed(seed)).to(DEV)
        pool.copy_(before)
        mass.copy_(new)
        g.replay()
        got = [x.clone() for x in (pool, mass, *out)]
        pool.copy_(before)
        mass.copy_(new)
        want = (pool, mass, *step())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got[2:], want[2:]))
        assert torch.equal(got[0], pool) and torch.equal(got[1], mass)


def test_refusals():
    c = Cache([40, 40], hkv=2, bs=16, seed=15)
    pool, mass, table = c.pool(torch.bfloat16).to(DEV), c.mass().to(DEV), c.table.to(DEV)
    keep, n = torch.zeros((2, 2, 5), dtype=torch.int32, device=DEV), i32([5, 5]).to(DEV)
    fp8 = on_device(c.pool("fp8"))
    for bad in (dict(pools=[pool, fp8]), dict(pools=[pool, pool.half()]), dict(keep=keep.long()),
                dict(counts=n.long()), dict(mass=mass.double()), dict(pools=[pool.double()])):
        a = dict(pools=[pool], keep=keep, counts=n, mass=mass)
        a.update(bad)
        with pytest.raises(TypeError):
            ops.kv_compact(a["pools"], table, a["keep"], a["counts"], mass=a["mass"])
    for bad in (dict(pools=[]), dict(pools=[pool, pool]),
                dict(pools=[pool, pool[:, :4].contiguous()]),
                dict(keep=keep[:, :1]), dict(keep=keep[..., ::2]), dict(counts=n[:1]),
                dict(mass=mass[:3]), dict(pools=[pool.cpu()]), dict(keep=keep.cpu()),
                dict(first=n[:1]), dict(cu=n), dict(dst=table[:1]), dict(pools=[pool] * 129)):
        a = dict(pools=[pool], keep=keep, counts=n, mass=mass, first=None, cu=None, dst=None)
        a.update(bad)
        with pytest.raises(ValueError):
            ops.kv_compact(a["pools"], table, a["keep"], a["counts"], mass=a["mass"],
                           first=a["first"], cu_seqlens=a["cu"], dst_table=a["dst"])
    for bad in (dict(budget=0), dict(budget=8, sinks=5, recent=4), dict(budget=8, sinks=-1),
                dict(budget=8, recent=-1)):
        with pytest.raises(ValueError):
            ops.kv_select(mass, table, n, **bad)
    with pytest.raises(TypeError):
        ops.kv_select(mass.half(), table, n, 4)
    with pytest.raises(ValueError):
        ops.kv_select(mass, table, n[:1], 4)
    with pytest.raises(ValueError):
        ops.kv_select(mass[0], table, n, 4)
    assert ops.kv_select(mass, table[:0], n[:0], 4)[0].shape == (0, 2, 4)
    ops.kv_compact([pool], table, keep[..., :0], n)
