"""Draft verification on the GPU against the definition in float64, token for token."""
import math

import pytest
import torch

from needle_amd import ops
from oracle import fp8_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _case(counts, vocab, dtype, seed, probs=True, temps=None):
    gen = torch.Generator().manual_seed(seed)
    n, total = len(counts), sum(counts)
    cu = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32)
    logits = (torch.randn(total, vocab, generator=gen) * 2.0).to(dtype)
    ids = torch.randint(0, vocab, (total,), generator=gen)
    draft = None
    rows = [r for i in range(n) for r in range(int(cu[i]), int(cu[i + 1]) - 1)]
    if rows:
        near = logits[rows].float() + torch.randn(len(rows), vocab, generator=gen) * 0.5
        d = torch.softmax(near, -1)
        x = torch.multinomial(d, 1, generator=gen)[:, 0]
        if not probs:     # points: often the likeliest token
            x = torch.where(torch.rand(len(rows), generator=gen) < 0.7, logits[rows].float()
                            .argmax(-1), x)
        ids[torch.tensor(rows) + 1] = x
        if probs:
            draft = d
    elif probs:
        draft = torch.empty(0, vocab)
    u = torch.rand(total, generator=gen)
    t = None if temps is None else torch.tensor((temps * n)[:n])
    return logits, ids, cu, u, t, draft


def _run(logits, ids, cu, u, t, draft):
    tokens, accepted = ops.verify_drafts(
        logits.to(DEV), ids.to(DEV), cu.to(DEV), u.to(DEV),
        temperature=None if t is None else t.to(DEV),
        draft_probs=None if draft is None else draft.to(DEV))
    return tokens.cpu(), accepted.cpu()


def _check(case):
    tokens, accepted = _run(*case)
    logits, ids, cu, u, t, draft = case
    want = fp8_ref.verify(logits, ids, cu, u, t, draft)
    assert accepted.tolist() == want[1]
    assert tokens.tolist() == want[0]
    assert tokens.dtype == ids.dtype and accepted.dtype == torch.int32


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("vocab", [1, 7, 1000, 4099, 32000, 50257])
def test_against_the_definition(vocab, probs, dtype):
    _check(_case([5, 1, 3, 8, 2, 1], vocab, dtype, 1 + vocab, probs))
    _check(_case([4, 2], vocab, dtype, 2 + vocab, probs, [0.7, 1.3]))


@pytest.mark.parametrize("probs", [True, False])
def test_temperatures(probs):
    temps = [0.0, 1.0, 0.3, 2.0, -1.0, math.nan, math.inf, 1e-30, 1e-42]
    _check(_case([3, 2, 5, 1, 4, 2, 3, 4, 3], 5000, torch.bfloat16, 7, probs, temps))


def test_a_large_vocabulary_and_batch():
    _check(_case([1, 6, 2, 9] * 10, 151936, torch.bfloat16, 8, True, [0.9, 0.0, 1.2]))


def test_int32_ids_strided_logits_and_one_sequence():
    logits, ids, cu, u, t, draft = _case([6], 4100, torch.float16, 9)
    wide = torch.zeros(6, 4203, dtype=torch.float16)
    wide[:, 3:4103] = logits
    want = fp8_ref.verify(logits, ids, cu, u, None, draft)
    tokens, accepted = ops.verify_drafts(wide.to(DEV)[:, 3:4103], ids.int().to(DEV), cu.to(DEV),
                                         u.to(DEV), draft_probs=draft.to(DEV))
    assert tokens.tolist() == want[0] and tokens.dtype == torch.int32
    assert accepted.tolist() == want[1]


@pytest.mark.parametrize("probs", [True, False])
def test_masked_rows_and_values_that_are_not_finite(probs):
    logits, ids, cu, u, t, draft = _case([4] * 8, 3001, torch.float32, 10, probs)
    inf = math.inf
    logits[0, 5:] = -inf                      # most of a row masked
    logits[4] = -inf                          # all of it
    logits[9, 100] = math.nan
    logits[9, 2000] = inf
    logits[13, 7], logits[13, 90] = inf, inf
    logits[16, :] = -3.4e38                   # the type's lowest value as a mask
    logits[16, 11] = 0.0
    logits[20, ::2] = -inf
    ids[5], ids[10], ids[14], ids[17] = 0, 100, 90, 11
    _check((logits, ids, cu, u, t, draft))


def test_uniforms_at_the_ends():
    for value in (0.0, 1.0, 0.99999994, -0.5, 2.0, math.nan):
        logits, ids, cu, u, t, draft = _case([3, 1, 4], 999, torch.bfloat16, 11)
        logits[:, 700:] = -math.inf           # the last tokens have no weight
        u[:] = value
        _check((logits, ids, cu, u, t, draft))


def test_a_draft_distribution_that_leaves_nothing():
    """q = p: a draft is accepted unless u = 1 rejects it, and then p itself is drawn from; q of
    NaN and below 0 counts as 0; tokens outside the vocabulary are rejected."""
    logits, ids, cu, u, t, _ = _case([2, 2, 2, 3], 64, torch.float32, 12)
    logits[:, 32:] = -math.inf
    draft = torch.softmax(logits.double(), -1).float()[[0, 2, 4, 6, 7]]
    draft[0] = 2.0                            # covers p everywhere
    draft[1, :8], draft[1, 8:16] = math.nan, -1.0
    ids[3] = 40
    ids[5], ids[7] = -1, 64
    u[0] = 0.9
    _check((logits, ids, cu, u, t, draft))
    # without distributions: a rejected draft that is all the row has
    logits[0] = -math.inf
    logits[0, 3], ids[1], u[0] = 0.0, 3, 1.0
    _check((logits, ids, cu, u, t, None))


def test_tokens_are_distributed_as_the_target():
    """Over many sequences of one drafted token, the first token's frequencies are p's: each is a
    binomial, and none of 12 is further off than 5 standard deviations."""
    n, v = 20000, 12
    gen = torch.Generator().manual_seed(13)
    row = torch.randn(v, generator=gen)
    q = torch.softmax(torch.randn(v, generator=gen), -1)
    logits = row.repeat(2 * n, 1)
    ids = torch.zeros(2 * n, dtype=torch.long)
    ids[1::2] = torch.multinomial(q, n, replacement=True, generator=gen)
    cu = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32)
    u = torch.rand(2 * n, generator=gen)
    p = torch.softmax(row.double(), -1)
    tokens = []
    for a in range(0, n, 10000):              # at most 65,535 rows a call
        s = slice(2 * a, 2 * a + 20000)
        got, _ = ops.verify_drafts(logits[s].to(DEV), ids[s].to(DEV), cu[:10001].to(DEV),
                                   u[s].to(DEV), draft_probs=q.repeat(10000, 1).to(DEV))
        tokens.append(got.cpu()[::2])
    count = torch.bincount(torch.cat(tokens), minlength=v).double()
    assert ((count - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt()).all()


def test_captured_and_replayed():
    logits, ids, cu, u, t, draft = (x.to(DEV) for x in _case([4, 1, 6], 20001, torch.bfloat16, 14,
                                                             True, [1.0, 0.0, 0.8]))

    def step():
        return ops.verify_drafts(logits, ids, cu, u, temperature=t, draft_probs=draft)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(5):
        u.uniform_()
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_refusals():
    logits, ids, cu, u, t, draft = (x.to(DEV) for x in _case([3, 2], 100, torch.bfloat16, 15,
                                                             True, [1.0]))
    ops_ = ops.verify_drafts
    with pytest.raises(ValueError, match="GPU tensor"):
        ops_(logits.cpu(), ids, cu, u)
    with pytest.raises(TypeError, match="unsupported dtype"):
        ops_(logits.double(), ids, cu, u)
    with pytest.raises(ValueError, match="rows must be contiguous"):
        ops_(logits[:, ::2], ids, cu, u)
    with pytest.raises(TypeError, match="int32 or int64"):
        ops_(logits, ids.float(), cu, u)
    with pytest.raises(ValueError, match="ids must be"):
        ops_(logits, ids[:4], cu, u)
    with pytest.raises(TypeError, match="cu_seqlens"):
        ops_(logits, ids, cu.long(), u)
    with pytest.raises(TypeError, match="uniforms must be float32"):
        ops_(logits, ids, cu, u.double())
    with pytest.raises(ValueError, match="temperature"):
        ops_(logits, ids, cu, u, temperature=t[:1])
    with pytest.raises(ValueError, match="draft_probs"):
        ops_(logits, ids, cu, u, draft_probs=draft[:2])
    with pytest.raises(ValueError, match="every sequence has a row"):
        ops_(logits[:1], ids[:1], cu, u[:1])
    got = ops_(logits[:0], ids[:0], cu[:1], u[:0])
    assert got[0].shape == (0,) and got[1].shape == (0,)
