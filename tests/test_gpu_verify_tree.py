"""Verification of drafted trees on the GPU against the definition in float64, token for token."""
import math

import pytest
import torch

from needle_amd import ops
from oracle import fp8_ref, tree_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _case(counts, vocab, dtype, seed, temps=None, likely=0.8, chain=False):
    """Trees whose nodes are often the likeliest tokens where they hang, some of them twice."""
    gen = torch.Generator().manual_seed(seed)
    n, total = len(counts), sum(counts)
    cu = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32)
    logits = (torch.randn(total, vocab, generator=gen) * 2.5).to(dtype)
    best = logits.float().topk(min(4, vocab), -1).indices
    ids = torch.randint(0, vocab, (total,), generator=gen)
    parents = torch.full((total,), -1, dtype=torch.int32)
    for i in range(n):
        a, m = int(cu[i]), counts[i]
        kids = {}
        for t in range(1, m):
            p = t - 1 if chain else int(torch.randint(max(0, t // 2 - 2), t, (1,), generator=gen))
            parents[a + t] = p
            k = kids[p] = kids.get(p, -1) + 1
            if torch.rand(1, generator=gen) < likely:
                ids[a + t] = best[a + p, k % best.shape[1]]
    u = torch.rand(total, generator=gen)
    t = None if temps is None else torch.tensor((temps * n)[:n])
    return logits, ids, parents, cu, u, t


def _run(logits, ids, parents, cu, u, t):
    got = ops.verify_tree(logits.to(DEV), ids.to(DEV), parents.to(DEV), cu.to(DEV), u.to(DEV),
                          temperature=None if t is None else t.to(DEV))
    return [x.cpu() for x in got]


def _check(case):
    tokens, accepted, path = _run(*case)
    want = tree_ref.verify(*case)
    assert accepted.tolist() == want[1]
    assert path.tolist() == want[2]
    assert tokens.tolist() == want[0]
    assert tokens.dtype == case[1].dtype and accepted.dtype == path.dtype == torch.int32


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 7, 1000, 4099, 32000, 50257])
def test_against_the_definition(vocab, dtype):
    _check(_case([5, 1, 30, 8, 2, 64], vocab, dtype, 1 + vocab))
    _check(_case([14, 70], vocab, dtype, 2 + vocab, [0.7, 1.3]))


def test_temperatures():
    temps = [0.0, 1.0, 0.3, 2.0, -1.0, math.nan, math.inf, 1e-30, 1e-42]
    _check(_case([13, 12, 25, 1, 4, 2, 33, 14, 3], 5000, torch.bfloat16, 7, temps))


def test_a_large_vocabulary_and_batch():
    _check(_case([1, 26, 12, 40] * 5, 151936, torch.bfloat16, 8, [0.9, 0.0, 1.2]))


def test_paths_are_long():
    """Sharp distributions: most drafts are taken, past the first 64 nodes too."""
    case = _case([60, 200, 333], 3000, torch.float32, 3, [0.15, 0.2, 0.1], likely=1.0)
    want = tree_ref.verify(*case)
    assert min(want[1]) >= 3 and max(want[1]) >= 10 and max(want[2]) >= 64
    _check(case)


def test_a_chain_is_verify_drafts():
    case = _case([7, 1, 30, 4], 9000, torch.bfloat16, 5, [0.4, 1.0, 0.2, 0.0], likely=0.95,
                 chain=True)
    logits, ids, parents, cu, u, t = case
    tokens, accepted, path = _run(*case)
    want = ops.verify_drafts(logits.to(DEV), ids.to(DEV), cu.to(DEV), u.to(DEV),
                             temperature=t.to(DEV))
    assert torch.equal(tokens, want[0].cpu()) and torch.equal(accepted, want[1].cpu())
    for i, k in enumerate(accepted.tolist()):
        a, b = int(cu[i]), int(cu[i + 1])
        assert path[a:b].tolist() == list(range(k + 1)) + [-1] * (b - a - k - 1)


def test_siblings_with_one_token_and_tokens_outside():
    logits, ids, parents, cu, u, t = _case([9], 500, torch.float32, 11)
    parents[:] = torch.tensor([-1, 0, 0, 0, 0, 0, 1, 3, 5], dtype=torch.int32)
    logits[0] = -2.0
    logits[0, 7], logits[0, 9] = 4.0, 3.9
    ids[1:6] = torch.tensor([7, 7, 9, -3, 500])
    for first in (0.1, 0.3, 0.42, 0.6, 0.75, 0.99):
        u[0] = first
        for last in (0.0, 0.5, 0.999):
            u[8] = last
            _check((logits, ids, parents, cu, u, t))


def test_children_with_all_the_weight():
    """Nothing is left for another token: the row's argmax."""
    logits, ids, parents, cu, u, t = _case([4], 300, torch.float32, 12)
    parents[:] = torch.tensor([-1, 0, 0, 1], dtype=torch.int32)
    logits[0] = -math.inf
    logits[0, 17], logits[0, 4] = 1.0, 1.0
    ids[1:3] = torch.tensor([17, 4])
    u[0] = 1.0                               # outside [0, 1): no child is taken
    _check((logits, ids, parents, cu, u, t))
    assert _run(logits, ids, parents, cu, u, t)[0][0] == 4


def test_parents_that_are_not_valid():
    logits, ids, parents, cu, u, t = _case([12, 8], 400, torch.bfloat16, 13, [0.2])
    parents[[2, 3, 5, 7, 14]] = torch.tensor([2, 9, 1 << 30, -5, 7], dtype=torch.int32)
    _check((logits, ids, parents, cu, u, t))


def test_masked_rows_and_values_that_are_not_finite():
    case = _case([14] * 6, 3001, torch.float32, 10)
    logits, ids, parents, cu, u, t = case
    inf = math.inf
    logits[0, 5:] = -inf                      # most of a row masked
    logits[14] = -inf                         # all of it
    logits[28, 100] = math.nan
    logits[28, 2000] = inf
    logits[42, 7], logits[42, 90] = inf, inf
    logits[56, :] = -3.4e38                   # the type's lowest value as a mask
    logits[56, 11] = 0.0
    logits[70, ::2] = -inf
    ids[15], ids[29], ids[43], ids[57] = 0, 100, 7, 11
    _check(case)


def test_int32_ids_strided_logits_and_rows_outside():
    logits, ids, parents, cu, u, t = _case([16, 5], 4100, torch.float16, 9)
    want = tree_ref.verify(logits, ids, parents, cu, u)
    wide = torch.zeros(24, 4203, dtype=torch.float16)
    wide[2:23, 3:4103] = logits

    def pad(x):
        return torch.cat([x[:2], x, x[:1]]).to(DEV)
    tokens, accepted, path = ops.verify_tree(wide.to(DEV)[:, 3:4103], pad(ids.int()),
                                             pad(parents), (cu + 2).to(DEV), pad(u))
    assert tokens[2:23].tolist() == want[0] and tokens.dtype == torch.int32
    assert accepted.tolist() == want[1] and path[2:23].tolist() == want[2]


def test_more_nodes_than_a_tree_has():
    """Rows past the 1,024th are no part of the tree; sequences without rows."""
    n = 1100
    gen = torch.Generator().manual_seed(2)
    logits = torch.full((n + 3, 50), -30.0)
    ids = torch.randint(0, 50, (n + 3,), generator=gen)
    parents = torch.tensor(list(range(-1, n - 1)) + [-1, 0, 0], dtype=torch.int32)
    logits[torch.arange(n + 2), ids[1:]] = 30.0          # each row's next is certain
    cu = torch.tensor([0, n, n, n + 3], dtype=torch.int32)
    u = torch.full((n + 3,), 0.5)
    tokens, accepted, path = _run(logits, ids, parents, cu, u, None)
    assert accepted.tolist()[:2] == [1023, 0]
    assert path[:1024].tolist() == list(range(1024)) and (path[1024:n] == -1).all()
    assert tokens[:1023].tolist() == ids[1:1024].tolist() and (tokens[1024:n] == -1).all()
    assert int(tokens[1023]) == int(logits[1023].argmax())


def test_the_tokens_are_distributed_as_the_target():
    """A sequence's first token over many draws: each as often as its probability, within five
    standard deviations."""
    n, v = 6000, 12
    gen = torch.Generator().manual_seed(21)
    row = torch.randn(v, generator=gen)
    logits = row.repeat(3 * n, 1)
    ids = torch.tensor([0, 3, 8]).repeat(n)
    parents = torch.tensor([-1, 0, 0], dtype=torch.int32).repeat(n)
    cu = torch.arange(0, 3 * n + 1, 3, dtype=torch.int32)
    u = torch.rand(3 * n, generator=gen)
    tokens, accepted, path = _run(logits, ids, parents, cu, u, None)
    count = torch.bincount(tokens.view(n, 3)[:, 0], minlength=v).double()
    p = torch.softmax(row.double(), 0)
    assert ((count - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt()).all()
    assert 0 < accepted.sum() < n


def test_captured_into_a_graph():
    case = _case([20, 33], 8000, torch.bfloat16, 15, [0.5])
    dev = [x.to(DEV) for x in case]
    ops.verify_tree(*dev[:5], temperature=dev[5])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.verify_tree(*dev[:5], temperature=dev[5])
    for seed in (1, 2, 3):
        dev[4].copy_(torch.rand(53, generator=torch.Generator().manual_seed(seed)))
        g.replay()
        want = ops.verify_tree(*dev[:5], temperature=dev[5])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals():
    dev = [x.to(DEV) for x in _case([5, 3], 100, torch.float32, 1, [1.0])]
    logits, ids, parents, cu, u, t = dev
    for bad in (dict(ids=ids.float()), dict(parents=parents.long()), dict(u=u.double()),
                dict(logits=logits.double()), dict(t=t.half())):
        a = dict(logits=logits, ids=ids, parents=parents, u=u, t=t)
        a.update(bad)
        with pytest.raises(TypeError):
            ops.verify_tree(a["logits"], a["ids"], a["parents"], cu, a["u"], temperature=a["t"])
    for bad in (dict(ids=ids[:7]), dict(parents=parents[:7]), dict(u=u[:7]), dict(t=t[:1]),
                dict(logits=logits[0]), dict(logits=logits.t()), dict(parents=parents.cpu()),
                dict(cu=torch.arange(20, dtype=torch.int32, device=DEV))):
        a = dict(logits=logits, ids=ids, parents=parents, u=u, t=t, cu=cu)
        a.update(bad)
        with pytest.raises(ValueError):
            ops.verify_tree(a["logits"], a["ids"], a["parents"], a["cu"], a["u"],
                            temperature=a["t"])
    assert all(x.numel() == 0 for x in ops.verify_tree(
        torch.empty(0, 10, device=DEV), ids[:0], parents[:0],
        torch.zeros(1, dtype=torch.int32, device=DEV), u[:0]))
