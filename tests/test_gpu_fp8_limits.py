"""The 8-bit pool's operators and the draft verification where their indexes end: pools past 2^32
bytes, more sequences, row blocks and drafts than one step of a scan takes, the longest blocks and
tables, several streams and graphs at once."""
import pytest
import torch

from needle_amd import _lib, ops
from oracle import fp8_ref
from test_gpu_fp8_attention import Case, _wide
from test_gpu_verify import _case as verify_case, _check as verify_check, _run as verify_run

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("counts", [[1, 1], [3, 20], [120, 7]])
def test_pools_past_four_gigabytes(counts):
    """The same blocks at the far end of a pool of 2^32 bytes and more."""
    shape = (8, 2, 128, 16)
    c = Case(shape, counts, [700, 45], seed=1,
             extra_cols=_wide(shape, counts) if max(counts) == 120 else 1)
    nb = (1 << 32) // (2 * 2 * 16 * 128) + 1000
    codes = torch.full((2, nb, 2, 16, 128), 0x7F, dtype=torch.uint8, device=DEV)
    scales = torch.zeros(2, nb, 2, 16, dtype=torch.uint8, device=DEV)
    codes[:, -c.nb:], scales[:, -c.nb:] = c.codes.to(DEV), c.scales.to(DEV)
    table, cu, ctx = (c.table + (nb - c.nb)).to(DEV), c.cu.to(DEV), c.ctx.to(DEV)
    heads = (c.scale, c.h, c.hkv, c.d)
    if max(counts) == 1:
        got = ops.paged_decode_fp8(c.q.to(DEV), codes, scales, table, ctx, *heads)
    else:
        got = ops.varlen_prefill_fp8(c.q.to(DEV), codes, scales, table, cu, ctx, max(counts),
                                     *heads)
    c.check(got)
    # read back what is attended, write it again, and nothing else changes
    total = [n + m for n, m in zip(c.lens, counts)]
    rcu = torch.tensor([0, total[0], sum(total)], dtype=torch.int32, device=DEV)
    zero = torch.zeros(2, dtype=torch.int32, device=DEV)
    k, v = ops.kv_read_fp8(codes, scales, table, zero, rcu, sum(total))
    vals = fp8_ref.values(c.codes, c.scales)
    for i in range(2):
        p = torch.arange(total[i])
        want = vals[:, c.table[i][p // 16].long(), :, p % 16]       # [tokens, 2, Hkv, D]
        rows = slice(int(rcu[i]), int(rcu[i + 1]))
        assert torch.equal(k[rows].cpu().double(), want[:, 0])
        assert torch.equal(v[rows].cpu().double(), want[:, 1])
    # (the scale of what is written again is the smallest power: not the bytes, the values)
    sample = slice(nb - c.nb, nb)
    rest = codes[:, :1000].clone()
    ops.kv_append_fp8(k, v, codes, scales, table, zero, rcu)
    k2, v2 = ops.kv_read_fp8(codes, scales, table, zero, rcu, sum(total))
    assert torch.equal(k2, k) and torch.equal(v2, v)
    assert torch.equal(codes[:, :1000], rest)
    used = torch.zeros(c.nb, 16, dtype=torch.bool)
    for i in range(2):
        p = torch.arange(total[i])
        used[c.table[i][p // 16].long(), p % 16] = True
    free = ~used[None, :, None, :].expand(2, -1, 2, -1)
    assert torch.equal(codes[:, sample].cpu()[free], c.codes[free])
    assert torch.equal(scales[:, sample].cpu()[free], c.scales[free])


@pytest.mark.parametrize("n", [64, 65, 128, 300])
def test_many_sequences(n):
    """Decode, append and read of more sequences than a wave's lanes, or than four steps of the
    scan over row blocks; some empty."""
    c = Case((4, 2, 64, 16), [1] * n, [(37 * i) % 200 - 1 for i in range(n)], seed=n,
             extra_cols=60)
    c.check(c.run(decode=True))
    counts = [(i * 7) % 5 for i in range(n)]
    c = Case((4, 2, 64, 16), counts, [(41 * i) % 150 for i in range(n)], seed=n + 1)
    c.check(c.run())
    pool = c.codes.to(DEV), c.scales.to(DEV)
    k, v = ops.kv_read_fp8(*pool, c.table.to(DEV), c.ctx.to(DEV), c.cu.to(DEV), int(c.cu[-1]))
    vals = fp8_ref.values(c.codes, c.scales)
    for i in range(n):
        for t in range(counts[i]):
            blk, row = fp8_ref.slot(c.table[i], c.lens[i] + t, 16, c.nb)
            at = int(c.cu[i]) + t
            assert torch.equal(k[at].cpu().double(), vals[0, blk, :, row])
            assert torch.equal(v[at].cpu().double(), vals[1, blk, :, row])
    rows = int(c.cu[-1])
    nk = torch.randn(rows, 2, 64, generator=c.gen).bfloat16()
    codes, scales = c.codes.clone(), c.scales.clone()
    fp8_ref.append(nk, nk.flip(0), codes, scales, c.table, c.cu, c.ctx)
    ops.kv_append_fp8(nk.to(DEV), nk.flip(0).to(DEV), *pool, c.table.to(DEV), c.ctx.to(DEV),
                      c.cu.to(DEV))
    assert torch.equal(pool[0].cpu(), codes) and torch.equal(pool[1].cpu(), scales)


@pytest.mark.parametrize("n", [64, 65, 300])
@pytest.mark.parametrize("count", [1, 3, 40])
def test_many_row_blocks_in_shares(n, count):
    """Tables of 1,700 keys and more are cut into shares: row blocks of nothing, of one tile and of
    many, more of them than a wave's lanes or four steps of the scan."""
    counts = [1] * n if count == 1 else [(i * 7) % count for i in range(n)]
    if count == 40:
        counts = counts[:65]
    lens = [(37 * i) % 400 - 1 for i in range(len(counts))]
    lens[len(counts) // 2] = 1700
    c = Case((4, 2, 64, 16), counts, lens, seed=n, extra_cols=10)
    keys = c.table.shape[1] * 16
    assert ops.fp8_attention_workspace_bytes(len(counts), int(c.cu[-1]), max(counts), keys, 4, 2,
                                             64) > 0
    c.check(c.run(decode=count == 1))


def test_one_long_context():
    """One sequence over all workgroups, in blocks of 1,024 tokens."""
    c = Case((4, 1, 64, 1024), [1], [70001], seed=3)
    c.check(c.run(decode=True))
    c = Case((4, 1, 64, 1024), [5], [40000], seed=4)
    c.check(c.run())


@pytest.mark.parametrize("probs", [True, False])
def test_many_drafts(probs):
    """Sequences of more rows than are decided on at a time, all accepted or rejected late."""
    case = verify_case([64, 65, 66, 130, 1, 200], 77, torch.float32, 5, probs)
    logits, ids, cu, u, t, draft = case
    verify_check(case)
    u = u * 1e-6                                # nearly everything is accepted
    u[-1], u[int(cu[1]) - 1] = 0.3, 0.9
    if probs:
        verify_check((logits, ids, cu, u, t, draft))
    # points at the likeliest tokens, temperature 0: accepted but where one is replaced
    ids[1:] = logits.argmax(-1)[:-1]
    ids[int(cu[3]) + 100] = (ids[int(cu[3]) + 100] + 1) % 77
    cold = torch.zeros(6)
    tokens, accepted = verify_run(logits, ids, cu, u, cold, None)
    assert accepted.tolist() == [63, 64, 65, 99, 0, 199]
    assert (tokens.tolist(), accepted.tolist()) == fp8_ref.verify(logits, ids, cu, u, cold, None)


def test_the_largest_vocabulary():
    verify_check(verify_case([3, 2], 1 << 18, torch.bfloat16, 6))
    logits = torch.zeros(2, (1 << 18) + 1, dtype=torch.bfloat16, device=DEV)
    ids = torch.zeros(2, dtype=torch.long, device=DEV)
    cu = torch.tensor([0, 2], dtype=torch.int32, device=DEV)
    with pytest.raises(_lib.NeedleAmdError):
        ops.verify_drafts(logits, ids, cu, torch.zeros(2, device=DEV))


def test_slices_that_end_unevenly():
    """Vocabularies about the borders of a load, a step and a slice, rows at any alignment."""
    for vocab in (8, 9, 2047, 2048, 2049, 2055, 6143, 6145, 12289):
        for dtype in (torch.bfloat16, torch.float32):
            logits, ids, cu, u, t, draft = verify_case([3, 1, 4], vocab, dtype, vocab)
            tokens, accepted = fp8_ref.verify(logits, ids, cu, u, t, draft)
            for off in (0, 1, 3):
                wide = torch.zeros(len(ids), vocab + 5, dtype=dtype, device=DEV)
                wide[:, off:off + vocab] = logits.to(DEV)
                d = torch.zeros(draft.shape[0], vocab + 3, device=DEV)
                d[:, off:off + vocab] = draft.to(DEV)
                got = ops.verify_drafts(wide[:, off:off + vocab], ids.to(DEV), cu.to(DEV),
                                        u.to(DEV), draft_probs=d[:, off:off + vocab])
                assert (got[0].tolist(), got[1].tolist()) == (tokens, accepted), (vocab, off)


def test_streams_and_graphs_at_once():
    """The operators on two streams, and two captured graphs replayed beside each other."""
    cases = [Case((8, 2, 64, 16), [2, 5], [900, 70 + i], seed=20 + i, extra_cols=80)
             for i in range(2)]
    checks = [tuple(x.to(DEV) for x in verify_case([4, 3], 5000, torch.bfloat16, 30 + i, True,
                                                   [1.0])) for i in range(2)]
    inputs = [[x.to(DEV) for x in (c.q, c.codes, c.scales, c.table, c.cu, c.ctx)] for c in cases]

    def step(i):
        q, codes, scales, table, cu, ctx = inputs[i]
        out = ops.varlen_prefill_fp8(q, codes, scales, table, cu, ctx, 5, 0.125, 8, 2, 64)
        logits, ids, vcu, u, t, draft = checks[i]
        return (out, *ops.verify_drafts(logits, ids, vcu, u, temperature=t, draft_probs=draft))

    want = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(step(i))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(i))
        graphs.append(g)
    for _ in range(5):
        for a in outs:
            for x in a:
                x.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
