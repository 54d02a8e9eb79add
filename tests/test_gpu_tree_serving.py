"""The operators of drafted trees, and those of caches that keep some rows, run together as serving
runs them, on the GPU.

Trees: every step appends the nodes of a tree to the pools of two layers, masks and attends them,
verifies them by the layers' outputs and moves the accepted path's rows together.  Each step's outputs
are within attention's bound (test_gpu_tree_attention.py) of the definition in float64, its verdict is
the definition's for the logits that it got, and at the end the pools hold, to the byte, what
appending the accepted tokens one by one gives.

Bounded caches: decoding adds up weights, and what is past the budget goes.  Every head's rows are
those of the tokens that the definition picks by the weights, to the byte.
"""
import pytest
import torch

from needle_amd import ops
from oracle import tree_ref
from test_gpu_tree_attention import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
H, HKV, D, VOCAB, LAYERS = 8, 2, 64, 24, 2
SCALE = D ** -0.5


class Model:
    """Queries, keys and values that are the token's own, in every layer; the logits are of the sum
    of the layers' outputs."""

    def __init__(self, dtype, seed):
        g = torch.Generator().manual_seed(seed)
        self.q, self.k, self.v = (
            torch.randn(LAYERS, VOCAB, h, D, generator=g).to(DEV, dtype) for h in (H, HKV, HKV))
        self.head = torch.randn(H * D, VOCAB, generator=g).to(DEV) / 8
        f = torch.outer(torch.arange(4096.0), 1e4 ** (-torch.arange(0, D, 2) / D))
        self.cos, self.sin = (torch.cat((x, x), 1).to(DEV, dtype) for x in (f.cos(), f.sin()))


class Serving:
    def __init__(self, dtype, fp8, bs, lens, seed):
        self.m, self.dtype, self.fp8, self.bs = Model(dtype, seed), dtype, fp8, bs
        self.g = torch.Generator().manual_seed(seed + 1)
        self.n, self.w = len(lens), 512 // bs
        nb = self.n * self.w + 3
        self.table = torch.randperm(nb, generator=self.g)[:self.n * self.w].int().view(self.n, -1)
        self.dtable = self.table.to(DEV)
        self.pools = [self.pool(nb) for _ in range(LAYERS)]
        self.nb = nb
        self.tokens = [torch.randint(0, VOCAB, (n,), generator=self.g).tolist() for n in lens]
        self.fill(self.pools, [t[:-1] for t in self.tokens])    # the newest is not cached yet

    def pool(self, nb):
        if self.fp8:
            return ops.fp8_kv_pool(nb, HKV, self.bs, D, device=DEV)
        return torch.zeros(2, nb, HKV, self.bs, D, dtype=self.dtype, device=DEV)

    def append(self, layer, pool, ids, positions, ctx, cu):
        """q, rotated, of the packed tokens; their K and V go behind ctx."""
        m = self.m
        q, k, v = (x[layer].index_select(0, ids) for x in (m.q, m.k, m.v))
        cos, sin = m.cos.index_select(0, positions), m.sin.index_select(0, positions)
        if self.fp8:
            return ops.kv_append_fp8(k, v, pool.codes, pool.scales, self.dtable, ctx, cu, q=q,
                                     cos=cos, sin=sin)
        return ops.rope_kv_append(q, k, v, cos, sin, pool, self.dtable, ctx, cu)

    def fill(self, pools, tokens):
        ids = torch.tensor(sum(tokens, [])).to(DEV)
        pos = torch.tensor(sum(([*range(len(t))] for t in tokens), [])).to(DEV)
        cu = torch.tensor([0] + [len(t) for t in tokens]).cumsum(0).int().to(DEV)
        ctx = torch.zeros(self.n, dtype=torch.int32, device=DEV)
        for layer, pool in enumerate(pools):
            self.append(layer, pool, ids, pos, ctx, cu)


class Trees(Serving):
    NODES = 14          # of every tree: its root, three children, and so on

    def __init__(self, *a):
        super().__init__(*a)
        n, t = self.n, self.n * self.NODES
        self.cu = (torch.arange(n + 1) * self.NODES).int().to(DEV)
        self.ids = torch.zeros(t, dtype=torch.int64, device=DEV)
        self.parents = torch.zeros(t, dtype=torch.int32, device=DEV)
        self.u = torch.zeros(t, device=DEV)
        self.ctx = torch.tensor([len(x) - 1 for x in self.tokens], dtype=torch.int32, device=DEV)
        self.temp = torch.tensor([1.0, 0.0, 2.0, 1.0][:n], device=DEV)
        self.seq = torch.arange(n, device=DEV).repeat_interleave(self.NODES)

    def draw(self):
        """The next trees: the first children of a node have different tokens."""
        parents = [-1, 0, 0, 0]
        while len(parents) < self.NODES:
            parents.append(int(torch.randint(0, len(parents), (1,), generator=self.g)))
        ids = torch.randint(0, VOCAB, (self.n, self.NODES), generator=self.g)
        for i, t in enumerate(self.tokens):
            ids[i, 0] = t[-1]
            ids[i, 1:4] = torch.randperm(VOCAB, generator=self.g)[:3]
        self.ids.copy_(ids.flatten())
        self.parents.copy_(torch.tensor(parents * self.n))
        self.u.copy_(torch.rand(self.n * self.NODES, generator=self.g))

    def step(self):
        mask, depth = ops.tree_mask(self.parents, self.cu, self.NODES)
        pos = (self.ctx.index_select(0, self.seq) + depth).long()
        self.q, self.out = [], []
        for layer, pool in enumerate(self.pools):
            q = self.append(layer, pool, self.ids, pos, self.ctx, self.cu)
            out = ops.tree_attention(q, pool, self.dtable, self.cu, self.ctx, mask, self.NODES,
                                     SCALE, H, HKV, D, max_context_len=500)
            self.q.append(q)
            self.out.append(out)
        x = sum(o.float() for o in self.out).view(len(self.ids), H * D)
        self.logits = (x[:, :, None] * self.m.head[None]).sum(1)      # (no library product)
        self.verdict = ops.verify_tree(self.logits, self.ids, self.parents, self.cu, self.u,
                                       temperature=self.temp)
        _, accepted, path = self.verdict
        ops.kv_compact(self.pools, self.dtable, path, accepted + 1, first=self.ctx,
                       cu_seqlens=self.cu)

    def check_step(self, before):
        cu, ids, parents, ctx = (x.cpu() for x in (self.cu, self.ids, self.parents, self.ctx))

        def see(i):
            return tree_ref.sees(parents[cu[i]:cu[i + 1]])
        for layer in range(LAYERS):
            pool = before[layer]
            r = tree_ref.attention(self.q[layer].cpu(), pool, self.table, cu, ctx, SCALE, see)
            check(self.out[layer], r, self.dtype, D, len(ids))
        tokens, accepted, path = (x.tolist() for x in self.verdict)
        assert (tokens, accepted, path) == tree_ref.verify(
            self.logits.cpu(), ids, parents, cu, self.u.cpu(), self.temp.cpu())
        for i, k in enumerate(accepted):
            self.tokens[i] += tokens[int(cu[i]):int(cu[i]) + k + 1]
        self.ctx += torch.tensor(accepted, device=DEV, dtype=torch.int32) + 1
        return sum(accepted)


def on_cpu(pool):
    return pool.cpu() if torch.is_tensor(pool) else (pool.codes.cpu(), pool.scales.cpu())


@pytest.mark.parametrize("how", ["eager", "stream", "graph"])
@pytest.mark.parametrize("dtype,fp8,bs", [(torch.bfloat16, False, 16), (torch.float16, False, 64),
                                          (torch.bfloat16, True, 32), (torch.float16, True, 16)],
                         ids=["bf16", "fp16", "bf16-8bit", "fp16-8bit"])
def test_decoding_with_trees(dtype, fp8, bs, how):
    s = Trees(dtype, fp8, bs, [1, 37, 130, 300], 7)
    graph, stream = None, torch.cuda.current_stream()
    if how != "eager":
        stream = torch.cuda.Stream()
    taken = 0
    for turn in range(6):
        s.draw()
        stream.wait_stream(torch.cuda.current_stream())
        # the rows that verification moves are compared as the attention saw them: a second run of
        # the same step on the moved rows would see others
        with torch.cuda.stream(stream):
            if how == "graph" and turn == 1:
                kept = [p.clone() if torch.is_tensor(p) else type(p)(*(x.clone() for x in p))
                        for p in s.pools]
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    s.step()
                for p, k in zip(s.pools, kept):                # capture ran nothing
                    for x, y in zip([p] if torch.is_tensor(p) else p,
                                    [k] if torch.is_tensor(k) else k):
                        assert torch.equal(x, y)
            if graph is None:
                s.step()
            else:
                graph.replay()
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        # what the attention saw: the nodes in their order
        seen = [p.clone() if torch.is_tensor(p) else type(p)(*(x.clone() for x in p))
                for p in s.pools]
        depth = ops.tree_mask(s.parents, s.cu, s.NODES)[1]
        pos = (s.ctx.index_select(0, s.seq) + depth).long()
        for layer, pool in enumerate(seen):
            s.append(layer, pool, s.ids, pos, s.ctx, s.cu)
        taken += s.check_step([on_cpu(p) for p in seen])
    assert taken > 0
    # as if the tokens had come one by one
    alone = [s.pool(s.nb) for _ in range(LAYERS)]
    s.fill(alone, [t[:-1] for t in s.tokens])
    for got, want in zip(s.pools, alone):
        for x, y in zip(*((on_cpu(p),) if torch.is_tensor(p) else on_cpu(p)
                          for p in (got, want))):
            for i, t in enumerate(s.tokens):
                p = torch.arange(len(t) - 1)
                blk = s.table[i].long()[p // bs]
                assert torch.equal(x[:, blk, :, p % bs], y[:, blk, :, p % bs])


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
@pytest.mark.parametrize("dtype,bs", [(torch.bfloat16, 16), (torch.float16, 32)])
def test_decoding_in_a_bounded_cache(dtype, bs, graph):
    """Prompts are cut to the budget by their last tokens' weights; then every step that finds a cache
    of budget + spare rows cuts it again."""
    budget, spare, sinks, recent, window = 48, 4, 2, 8, 5
    s = Serving(dtype, False, bs, [20, 90, 150], 11)
    mass = ops.kv_mass_pool(s.nb, HKV, bs, device=DEV)
    lens = torch.tensor([len(t) - 1 for t in s.tokens], dtype=torch.int32, device=DEV)
    where = lens.clone()                                     # the newest token's position
    # the tokens of every (sequence, kv head), by position: what a row of the caches is of
    rows = [[list(range(len(t) - 1)) for _ in range(HKV)] for t in s.tokens]

    # the prompts' last tokens, by their queries in the first layer
    last = torch.tensor(sum((t[-1 - window:-1] for t in s.tokens), [])).to(DEV)
    cu = (torch.arange(s.n + 1) * window).int().to(DEV)
    pos = torch.cat([torch.arange(len(t) - 1 - window, len(t) - 1) for t in s.tokens]).to(DEV)
    scratch = s.pool(s.nb)
    q = s.append(0, scratch, last, pos, lens - window, cu)
    out = ops.attention_mass(q, s.pools[0], s.dtable, lens - window, mass, SCALE, H, HKV, D,
                             cu_seqlens=cu, max_seqlen=window)
    r = tree_ref.attention(q.cpu(), s.pools[0].cpu(), s.table, cu.cpu(), (lens - window).cpu(),
                           SCALE)
    check(out, r, dtype, D, len(last))

    def cut():
        """Rows of all caches above the budget; eager or replayed alike."""
        keep, kept = ops.kv_select(mass, s.dtable, lens, budget, sinks=sinks, recent=recent)
        ops.kv_compact(s.pools, s.dtable, keep, kept, mass=mass)
        lens.copy_(kept)
        return keep, kept

    def check_cut(weights, lens_before, keep, kept):
        want, count = tree_ref.select(weights, s.table, lens_before, budget, sinks, recent)
        assert torch.equal(keep.cpu(), want) and torch.equal(kept.cpu(), count)
        moved = mass.cpu()
        for i in range(s.n):
            for h in range(HKV):
                at = want[i, h, :int(count[i])].long()
                p = torch.arange(len(at))
                blk, src = s.table[i].long()[p // bs], s.table[i].long()[at // bs]
                assert torch.equal(moved[blk, h, p % bs], weights[src, h, at % bs])
                rows[i][h] = [rows[i][h][x] for x in at.tolist()]

    def check_rows():
        for layer, pool in enumerate(s.pools):
            pool = pool.cpu()
            for i, t in enumerate(s.tokens):
                # every token's row, appended alone
                ids = torch.tensor(t, device=DEV)
                one = torch.zeros(2, len(t), HKV, 16, D, dtype=dtype, device=DEV)
                table = torch.arange(len(t), dtype=torch.int32, device=DEV)[:, None]
                m, at = s.m, torch.arange(len(t), device=DEV)
                ops.rope_kv_append(None, m.k[layer][ids], m.v[layer][ids], m.cos[at], m.sin[at],
                                   one, table, torch.zeros_like(table[:, 0]),
                                   torch.arange(len(t) + 1, dtype=torch.int32, device=DEV))
                one = one.cpu()
                for h in range(HKV):
                    p = torch.arange(len(rows[i][h]))
                    blk = s.table[i].long()[p // bs]
                    assert torch.equal(pool[:, blk, h, p % bs], one[:, rows[i][h], h, 0])

    weights, before = mass.cpu(), lens.cpu()
    keep, kept = cut()
    check_cut(weights, before, keep, kept)
    check_rows()

    ids = torch.zeros(s.n, dtype=torch.int64, device=DEV)

    def step():
        outs = []
        for layer, pool in enumerate(s.pools):
            q = s.append(layer, pool, ids, where.long(), lens, None)
            if layer == 0:
                outs.append((q, ops.attention_mass(q, pool, s.dtable, lens, mass, SCALE, H, HKV,
                                                   D, decay=0.875)))
            else:
                outs.append((q, ops.paged_decode(q, pool, s.dtable, lens, SCALE, H, HKV, D)))
        return outs
    replay = None
    for turn in range(3 * spare):
        ids.copy_(torch.tensor([t[-1] for t in s.tokens]))
        weights, before = mass.cpu(), lens.cpu()
        if not graph or turn == 0:
            outs = step()
        else:
            if replay is None:
                replay = torch.cuda.CUDAGraph()
                with torch.cuda.graph(replay):
                    outs = step()
            replay.replay()
        torch.cuda.synchronize()
        cu1 = torch.arange(s.n + 1)
        for layer, (q, out) in enumerate(outs):
            r = tree_ref.attention(q.cpu(), s.pools[layer].cpu(), s.table, cu1, before, SCALE)
            if layer == 0:
                check(out, r, dtype, D, s.n)
                want = tree_ref.mass(r, weights, cu1, before, H, 0.875)
                # (test_gpu_attention_mass.py has its bound: here, of scores up to 50 in size,
                # 2 * 72 * 50 * 2^-24 + 2^-18)
                torch.testing.assert_close(mass.cpu().double(), want, rtol=2.0 ** -11, atol=1e-6)
            else:
                # (weights and output rounded to 8 bits and more, of values up to 4)
                torch.testing.assert_close(out.cpu().double(), r.out, rtol=2.0 ** -6, atol=2.0 ** -6)
        for i in range(s.n):
            for h in range(HKV):
                rows[i][h].append(len(s.tokens[i]) - 1)
            s.tokens[i].append(int(torch.randint(0, VOCAB, (1,), generator=s.g)))
        lens += 1
        where += 1
        if turn % spare == spare - 1:
            weights, before = mass.cpu(), lens.cpu()
            check_cut(weights, before, *cut())
            check_rows()
    assert int(lens.max()) == budget
