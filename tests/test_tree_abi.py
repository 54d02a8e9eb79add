"""What the entry points of drafted trees and of caches that keep some rows refuse before any launch,
their oracle against known values, and what tree_attention's direct loads rely on in its generated
code (CPU)."""
import math
import os
import re
import shutil
import subprocess

import pytest
import torch

from needle_amd import _lib
from oracle import fp8_ref, tree_ref

P = 1 << 20      # an aligned stand-in address that is never dereferenced
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_mask_refusals(lib):
    def mask(out=P, stride=2, words=2, depth=P, parents=P, cu=P, n=3, t=9, most=5):
        return lib.ndl_tree_mask(out, stride, words, depth, parents, cu, n, t, most, None)
    for bad in (dict(out=None), dict(out=P + 4), dict(depth=None), dict(parents=None),
                dict(cu=None), dict(words=0), dict(stride=1), dict(n=-1), dict(t=-1),
                dict(most=-1)):
        assert mask(**bad) == -1, bad
    assert mask(n=65536) == -2
    assert mask(n=0) == 0 and mask(t=0) == 0 and mask(most=0) == 0


@pytest.mark.parametrize("fp8", [False, True], ids=["16-bit", "8-bit"])
def test_attention_refusals(lib, fp8):
    def attend(out=P, q=P, qs=512, pool=P, scales=P, nb=4, table=P, stride=500, w=500, cu=P,
               ctx=P, mask=P, ms=2, words=2, n=3, t=9, most=3, keys=8000, h=8, hkv=2, d=64,
               bs=16, dtype=0, ws=P, size=0):
        store = (pool, scales) if fp8 else (pool,)
        f = lib.ndl_fp8_tree_attention if fp8 else lib.ndl_tree_attention
        return f(out, q, qs, *store, nb, table, stride, w, cu, ctx, mask, ms, words, n, t, most,
                 keys, h, hkv, d, bs, dtype, 0.1, ws, size, None)
    for bad in (dict(dtype=2), dict(d=96), dict(bs=12), dict(h=9), dict(h=34), dict(hkv=0),
                dict(nb=1 << 40), dict(w=1 << 30, stride=1 << 30)):
        assert attend(**bad) == -2, bad
    for bad in (dict(out=None), dict(q=None), dict(pool=None), dict(pool=P + 8), dict(table=None),
                dict(ctx=None), dict(qs=500), dict(qs=516), dict(q=P + 8), dict(most=0),
                dict(keys=0), dict(cu=None), dict(cu=None, t=3, most=1), dict(mask=None),
                dict(mask=P + 4), dict(words=0), dict(ms=1), dict(stride=3), dict(nb=0)):
        assert attend(**bad) == -1, bad
    query = (lib.ndl_fp8_tree_attention_workspace_bytes if fp8 else
             lib.ndl_tree_attention_workspace_bytes)
    need = query(3, 3, 8000, 8, 2, 64, 16)
    assert need > 0
    assert attend(size=need - 1) == -3 and attend(ws=None, size=need) == -3
    assert attend(ws=P + 16, size=need) == -3
    assert attend(n=0) == 0 and attend(t=0) == 0
    assert query(3, 3, 64, 8, 2, 64, 16) == 0          # short tables need none
    for bad in ((3, 3, 8000, 9, 2, 64, 16), (0, 3, 8000, 8, 2, 64, 16),
                (3, 0, 8000, 8, 2, 64, 16), (3, 3, 8000, 8, 2, 80, 16),
                (3, 3, 8000, 8, 2, 64, 17), (3, 3, 0, 8, 2, 64, 16)):
        assert query(*bad) == 0, bad


def test_mass_refusals(lib):
    def weigh(out=P, mass=P, q=P, qs=512, pool=P, nb=4, table=P, stride=500, w=500, cu=P, ctx=P,
              n=3, t=9, most=3, keys=8000, h=8, hkv=2, d=64, bs=16, dtype=0, ws=P, size=0):
        return lib.ndl_attention_mass(out, mass, q, qs, pool, nb, table, stride, w, cu, ctx, n, t,
                                      most, keys, h, hkv, d, bs, dtype, 0.1, 1.0, ws, size, None)
    for bad in (dict(dtype=2), dict(d=96), dict(bs=12), dict(h=9), dict(h=34), dict(hkv=0),
                dict(nb=1 << 40), dict(w=1 << 30, stride=1 << 30), dict(n=65536, t=70000)):
        assert weigh(**bad) == -2, bad
    for bad in (dict(out=None), dict(mass=None), dict(mass=P + 2), dict(q=None), dict(pool=None),
                dict(table=None), dict(ctx=None), dict(qs=500), dict(q=P + 8), dict(most=0),
                dict(keys=0), dict(cu=None), dict(cu=None, t=3), dict(stride=3), dict(nb=0)):
        assert weigh(**bad) == -1, bad
    query = lib.ndl_attention_mass_workspace_bytes
    need = query(3, 9, 3, 8000, 8, 2, 64, 16)
    assert need > 0 and weigh(size=need - 1) == -3 and weigh(ws=P + 16, size=need) == -3
    assert query(3, 9, 3, 64, 8, 2, 64, 16) > 0        # short ones keep their denominators
    assert weigh(n=0) == 0 and weigh(t=0) == 0
    for bad in ((3, 9, 3, 8000, 9, 2, 64, 16), (0, 9, 3, 8000, 8, 2, 64, 16),
                (3, 0, 3, 8000, 8, 2, 64, 16), (3, 9, 3, 8000, 8, 2, 80, 16)):
        assert query(*bad) == 0, bad


def test_verify_refusals(lib):
    def verify(tokens=P, acc=P, path=P, logits=P, stride=100, dtype=0, ids=P, parents=P, cu=P,
               u=P, temp=None, rows=4, n=2, vocab=100, ws=P, size=0):
        return lib.ndl_verify_tree(tokens, acc, path, logits, stride, dtype, ids, 1, parents, cu,
                                   u, temp, rows, n, vocab, ws, size, None)
    assert verify(dtype=7) == -2 and verify(rows=70000) == -2 and verify(n=70000) == -2
    for bad in (dict(tokens=None), dict(acc=None), dict(path=None), dict(logits=None),
                dict(ids=None), dict(parents=None), dict(cu=None), dict(u=None), dict(stride=99),
                dict(logits=P + 1), dict(dtype=2, logits=P + 2), dict(u=P + 2), dict(rows=0),
                dict(rows=-1), dict(vocab=0)):
        assert verify(**bad) == -1, bad
    need = lib.ndl_verify_tree_workspace_bytes(4, 2, 100)
    assert need > 0 and verify(size=need - 1) == -3 and verify(ws=P + 4, size=need) == -3
    assert verify(n=0) == 0


def test_select_refusals(lib):
    def select(keep=P, kept=P, mass=P, nb=4, hkv=2, bs=16, table=P, stride=8, w=8, lens=P, n=3,
               budget=32, sinks=4, recent=8):
        return lib.ndl_kv_select(keep, kept, mass, nb, hkv, bs, table, stride, w, lens, n, budget,
                                 sinks, recent, None)
    for bad in (dict(keep=None), dict(kept=None), dict(mass=None), dict(mass=P + 2),
                dict(table=None), dict(lens=None), dict(nb=0), dict(hkv=0), dict(bs=0), dict(w=0),
                dict(stride=7), dict(n=-1), dict(budget=0), dict(sinks=-1), dict(recent=-1),
                dict(sinks=16, recent=17)):
        assert select(**bad) == -1, bad
    assert select(n=65536) == -2 and select(w=1 << 28, stride=1 << 28) == -2
    assert select(w=(1 << 27) - 8, stride=1 << 27) == -2     # positions are counted on in 32 bits
    assert select(n=0) == 0


def test_compact_refusals(lib):
    import ctypes
    here = (ctypes.c_void_p * 129)(*[P + 4096 * i for i in range(129)])
    twice = (ctypes.c_void_p * 2)(P, P)
    odd = (ctypes.c_void_p * 2)(P, P + 8)
    none = (ctypes.c_void_p * 2)(P, None)

    def move(pools=here, scales=None, layers=2, mass=None, nb=4, hkv=2, bs=16, row=256, table=P,
             stride=8, w=8, to=None, ts=0, tw=0, keep=P, width=4, cu=None, rows=0, first=None,
             counts=P, n=3):
        return lib.ndl_kv_compact(pools, scales, layers, mass, nb, hkv, bs, row, table, stride, w,
                                  to, ts, tw, keep, width, cu, rows, first, counts, n, None)
    for bad in (dict(pools=None), dict(pools=odd), dict(pools=none), dict(pools=twice),
                dict(scales=none),
                dict(table=None), dict(keep=None), dict(counts=None), dict(mass=P + 2),
                dict(layers=-1), dict(n=-1), dict(nb=0), dict(hkv=0), dict(bs=0), dict(row=0),
                dict(row=24), dict(w=0), dict(stride=7), dict(to=P), dict(to=P, ts=3, tw=4),
                dict(width=-1), dict(rows=-1)):
        assert move(**bad) == -1, bad
    for bad in (dict(layers=129), dict(w=1 << 28, stride=1 << 28),
                dict(to=P, ts=1 << 28, tw=1 << 28), dict(nb=1 << 28), dict(row=1 << 20)):
        assert move(**bad) == -2, bad
    assert move(n=0) == 0 and move(width=0) == 0 and move(layers=0) == 0
    assert move(cu=P, rows=0) == 0


def test_oracle_trees():
    #      0
    #    1   2
    #   3 4   5     6 follows the context alone
    parents = torch.tensor([-1, 0, 0, 1, 1, 2, 6])
    see = tree_ref.sees(parents)
    assert [row.nonzero()[:, 0].tolist() for row in see] == [
        [0], [0, 1], [0, 2], [0, 1, 3], [0, 1, 4], [0, 2, 5], [6]]
    assert tree_ref.mask_words(see, 1)[:, 0].tolist() == [1, 3, 5, 11, 19, 37, 64]
    far = torch.zeros(1, 128, dtype=torch.bool)
    far[0, 63] = far[0, 64] = True
    assert tree_ref.mask_words(far, 2).tolist() == [[-2 ** 63, 1]]


def test_oracle_attention_is_the_chunks_without_a_tree():
    g = torch.Generator().manual_seed(3)
    pool = torch.randn(2, 5, 2, 16, 64, generator=g).to(torch.bfloat16)
    q = torch.randn(4, 4, 64, generator=g).to(torch.bfloat16)
    table = torch.tensor([[3, 1, 4]])
    r = tree_ref.attention(q, pool, table, [0, 4], [20], 0.125)
    k, v = (pool[x][table[0].long()].permute(1, 0, 2, 3).reshape(2, 48, 64).double()
            for x in (0, 1))
    for t in range(4):
        for h in range(4):
            p = torch.softmax(k[h // 2, :21 + t] @ q[t, h].double() * 0.125, 0)
            torch.testing.assert_close(r.out[t, h], p @ v[h // 2, :21 + t])
    got = tree_ref.mass(r, torch.ones(5, 2, 16), [0, 4], [20], 4, decay=0.5)
    assert math.isclose(float(got.sum()), 4 * 4 + 0.5 * 20 * 2 + (5 * 16 - 24) * 2)
    chain = tree_ref.attention(q, pool, table, [0, 4], [20], 0.125,
                               lambda i: tree_ref.sees(torch.arange(4) - 1))
    assert torch.equal(chain.out, r.out)


def test_oracle_verify():
    logits = torch.log(torch.tensor([[0.5, 0.25, 0.125, 0.125]])).repeat(4, 1)
    ids, parents = torch.tensor([0, 1, 2, 3]), torch.tensor([-1, 0, 0, 1])

    def verify(*u):
        return tree_ref.verify(logits, ids, parents, [0, 4], torch.tensor(u))
    # the root's children are tokens 1 and 2: below 0.25 the first, below 0.375 the second
    tokens, accepted, path = verify(0.2, 0.9, 0.9, 0.0)
    assert (tokens, accepted, path) == ([1, 0, -1, -1], [1], [0, 1, -1, -1])
    tokens, accepted, path = verify(0.3, 0.9, 0.9, 0.99)
    assert (tokens, accepted, path) == ([2, 3, -1, -1], [1], [0, 2, -1, -1])
    # none taken: tokens 0 and 3 are left, with 4 / 5 and 1 / 5 of what is left
    assert verify(0.4, 0.9, 0.9, 0.79)[0][:2] == [0, -1]
    assert verify(0.4, 0.9, 0.9, 0.81)[0][:2] == [3, -1]
    # a chain gives what verification of drafts gives
    g = torch.Generator().manual_seed(5)
    for _ in range(20):
        x = torch.randn(6, 5, generator=g)
        ids, u = torch.randint(0, 5, (6,), generator=g), torch.rand(6, generator=g)
        want = fp8_ref.verify(x, ids, [0, 4, 6], u, torch.tensor([1.0, 0.5]))
        got = tree_ref.verify(x, ids, torch.tensor([-1, 0, 1, 2, -1, 0]), [0, 4, 6], u,
                              torch.tensor([1.0, 0.5]))
        assert got[:2] == want


def test_oracle_rows_that_stay():
    mass = torch.tensor([5.0, 1, 4, 4, math.nan, 0, 9, 2]).view(2, 1, 4)
    keep, kept = tree_ref.select(mass, torch.tensor([[1, 0], [7, 0]]), [8, 8], 4, 1, 1)
    # rows 4 .. 7, 0 .. 3 of the pool: NaN first, then 9, 5, 4, 4, 2, 1, 0
    assert keep.tolist() == [[[0, 2, 4, 7]], [[0, 4, 6, 7]]] and kept.tolist() == [4, 4]
    x = torch.arange(8.0).view(2, 1, 4)
    tree_ref.compact([(x, 0)], torch.tensor([[1, 0]]), keep[:1], kept)
    assert x.flatten().tolist() == [0, 1, 2, 3, 4, 6, 0, 3]


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not installed")
def test_tree_attention_uses_m0_only_for_direct_lds_loads(tmp_path):
    # the loads are inline asm that writes M0, which the compiler cannot be told of
    asm = tmp_path / "tree_attention.s"
    subprocess.check_call([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang",
                           "-target-feature", "-Xclang", "-packed-fp32-ops",
                           "-I" + os.path.join(ROOT, "include"), "-S", "--cuda-device-only",
                           os.path.join(ROOT, "needle_amd", "csrc", "tree_attention.hip"), "-o",
                           str(asm)], stderr=subprocess.DEVNULL)
    body = [l.strip() for l in asm.read_text().splitlines()]
    body = [l for l in body if l and not l.startswith((";", "."))]
    uses = [i for i, l in enumerate(body) if re.search(r"\bm0\b", l)]
    assert uses, "expected the direct-load M0 writes"
    for i in uses:
        assert re.match(r"s_mov_b32 m0, (s\d+|vcc_lo|vcc_hi)$", body[i]), body[i]
        assert body[i + 1] == "s_nop 0" and \
            re.match(r"global_load_lds_dword(x4)? ", body[i + 2]), body[i:i + 3]
