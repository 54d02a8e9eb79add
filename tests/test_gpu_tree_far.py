"""Drafted trees and caches that keep some rows in pools whose planes pass 4 GiB, and from several
threads at once: the same to the bit as in a small pool, one call after the other."""
import threading

import pytest
import torch

from needle_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
H, HKV, D, BS = 32, 8, 128, 16
SCALE = D ** -0.5


class Work:
    """Trees after contexts, in a pool whose blocks are `blocks`."""

    def __init__(self, seed, dtype=torch.bfloat16):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.counts = [5, 2000, 333], [40, 7, 24]
        self.cols = (max(self.lens) + max(self.counts)) // BS + 1
        self.nb = 3 * self.cols
        t = sum(self.counts)
        self.small = torch.randn(2, self.nb, HKV, BS, D, generator=g).to(DEV, dtype)
        self.q = torch.randn(t, H, D, generator=g).to(DEV, dtype)
        self.table = torch.randperm(self.nb, generator=g).int().view(3, -1).to(DEV)
        self.parents = torch.tensor(sum(([-1] + [x // 2 for x in range(n - 1)]
                                         for n in self.counts), [])).int().to(DEV)
        self.cu = torch.tensor([0] + self.counts).cumsum(0).int().to(DEV)
        self.ctx = torch.tensor(self.lens, dtype=torch.int32, device=DEV)
        self.weights = torch.rand(self.nb, HKV, BS, generator=g).to(DEV)
        self.path = torch.tensor(sum(([0, 2, 5] + [-1] * (n - 3) for n in self.counts),
                                     [])).int().to(DEV)

    def run(self, pool, table, weights, fp8=False):
        """Results, and the pool's and the weights' blocks after them, in the table's order."""
        bound = dict(max_context_len=max(self.lens))
        most = max(self.counts)
        mask, depth = ops.tree_mask(self.parents, self.cu, most)
        outs = [mask, depth, ops.tree_attention(self.q, pool, table, self.cu, self.ctx, mask, most,
                                                SCALE, H, HKV, D, **bound)]
        if not fp8:
            outs.append(ops.attention_mass(self.q, pool, table, self.ctx, weights, SCALE, H, HKV, D,
                                           cu_seqlens=self.cu, max_seqlen=most, **bound))
            outs.append(ops.attention_mass(self.q[:3], pool, table, self.ctx, weights, SCALE, H,
                                           HKV, D, decay=0.5, **bound))
        counts = torch.full((3,), 3, dtype=torch.int32, device=DEV)
        ops.kv_compact([pool], table, self.path, counts, first=self.ctx, cu_seqlens=self.cu)
        keep, kept = ops.kv_select(weights, table, self.ctx, 100, sinks=2, recent=9)
        ops.kv_compact([pool], table, keep, kept, mass=weights)
        order = table.flatten().long()
        for x in (pool if fp8 else (pool,)):
            outs.append(x.view(torch.uint8).index_select(1, order))
        return outs + [keep, kept, weights.index_select(0, order)]


@pytest.mark.parametrize("fp8", [False, True], ids=["16-bit", "8-bit"])
def test_planes_past_4_gib(fp8):
    w = Work(1)
    row = HKV * BS * D * (1 if fp8 else 2)
    far = (1 << 32) // row + 2 * w.nb
    if fp8:
        small, big = ops.fp8_kv_pool(w.nb, HKV, BS, D, device=DEV), None
        ops.kv_append_fp8(*(w.small[x].permute(0, 2, 1, 3).reshape(-1, HKV, D) for x in (0, 1)),
                          small.codes, small.scales,
                          torch.arange(w.nb, dtype=torch.int32, device=DEV)[None],
                          torch.zeros(1, dtype=torch.int32, device=DEV),
                          torch.tensor([0, w.nb * BS], dtype=torch.int32, device=DEV))
        big = type(small)(torch.empty(2, far, HKV, BS, D, dtype=small.codes.dtype, device=DEV),
                          torch.empty(2, far, HKV, BS, dtype=small.scales.dtype, device=DEV))
        for x, y in zip(big, small):
            x.view(torch.uint8)[:, far - w.nb:] = y.view(torch.uint8)
    else:
        small = w.small.clone()
        big = torch.empty(2, far, HKV, BS, D, dtype=small.dtype, device=DEV)
        big[:, far - w.nb:] = small
    weights = torch.empty(far, HKV, BS, device=DEV)
    weights[far - w.nb:] = w.weights
    want = w.run(small, w.table, w.weights.clone(), fp8)
    got = w.run(big, w.table + (far - w.nb), weights, fp8)
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_threads_on_their_own_streams():
    works = [Work(s) for s in range(4)]
    want = [w.run(w.small.clone(), w.table, w.weights.clone()) for w in works]
    pools = [w.small.clone() for w in works]
    masses = [w.weights.clone() for w in works]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []
    ready = threading.Barrier(4)

    def go(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                ready.wait()
                for _ in range(5):
                    pools[i].copy_(works[i].small)
                    masses[i].copy_(works[i].weights)
                    got[i] = works[i].run(pools[i], works[i].table, masses[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:           # noqa: BLE001 (reported below)
            errors.append(e)
    threads = [threading.Thread(target=go, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for g, w in zip(got, want):
        for x, y in zip(g, w):
            assert torch.equal(x, y)
