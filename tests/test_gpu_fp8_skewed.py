"""Attention over the 8-bit pool in shares whose ends move by more than a row block's empty slots
(long sequences), with short sequences before, between and after the long ones: what a batch holds
into which new sequences are taken while others run on.  Against the definition in float64, bounds as
in test_gpu_fp8_attention."""
import pytest
import torch

from needle_amd import ops
from test_gpu_fp8_attention import Case
from test_gpu_fp8_decode_append import Step

pytestmark = pytest.mark.gpu

FRONT = [20]
FRONTS = [0, 1, 100, 31]


def _lens(n, tokens, short, where):
    lens = [tokens - 7 * (i % 5) for i in range(n)]
    at = {"front": 0, "middle": n // 2, "end": n}[where]
    return lens[:at] + short + lens[at:]


def _moves_ends(c):
    """Whether the call is cut into shares whose ends move by more than the empty slots (1 before a
    row block of 16 columns, 4 before one of 32): by an eighth of a share's slots.  The number of
    shares is read from the workspace's size: (shares + row blocks) parts per kv head."""
    counts, group = c.counts, c.h // c.hkv
    size = ops.fp8_attention_workspace_bytes(len(counts), sum(counts), max(counts),
                                             c.table.shape[1] * c.bs, c.h, c.hkv, c.d, c.bs)
    nt = 1 if max(counts) * group <= 16 else 2
    toks, pad = 16 * nt // group, 1 if nt == 1 else 4
    per_seq = -(-max(counts) // toks)
    shares = size // (8 + 4 * c.d) // (c.hkv * toks * group) - len(counts) * per_seq
    slots = sum(-(-(n + min(toks * (e + 1), m)) // 32) + pad for n, m in zip(c.lens, counts)
                for e in range(-(-m // toks)) if n >= 0)
    return shares > 0 and slots // shares // 8 > pad


@pytest.mark.parametrize("where,short", [("front", FRONT), ("front", FRONTS), ("middle", FRONTS),
                                         ("end", FRONTS)])
@pytest.mark.parametrize("shape,n,dtype", [((32, 8, 128, 16), 40, torch.bfloat16),
                                           ((16, 8, 64, 64), 48, torch.float16)])
def test_decode(shape, n, dtype, where, short):
    lens = _lens(n, 2000, short, where)
    c = Case(shape, [1] * len(lens), lens, dtype, seed=1)
    assert _moves_ends(c)
    c.check(c.run(decode=True))


@pytest.mark.parametrize("shape,n", [((32, 8, 128, 16), 40), ((16, 8, 64, 64), 48)])
@pytest.mark.parametrize("short", [FRONT, FRONTS + [-1]])
def test_a_decode_step_in_one_call(shape, n, short):
    lens = _lens(n, 2000, short, "front")
    c = Case(shape, [1] * len(lens), lens, seed=2)
    assert _moves_ends(c)
    Step(c).check()


@pytest.mark.parametrize("where,short", [("front", FRONT), ("front", FRONTS), ("middle", FRONTS)])
@pytest.mark.parametrize("count,dtype", [(8, torch.bfloat16), (5, torch.float16)])
def test_drafts(count, dtype, where, short):
    lens = _lens(64, 1800, short, where)
    c = Case((32, 8, 128, 16), [count] * len(lens), lens, dtype, seed=3)
    assert _moves_ends(c)
    c.check(c.run())


def test_sequences_without_tokens_between():
    lens = _lens(48, 2000, [700, 5, 3], "front")
    counts = [0, 3, 0] + [(i * 3) % 5 for i in range(48)]
    c = Case((32, 8, 128, 16), counts, lens, seed=4)
    assert _moves_ends(c)
    c.check(c.run())
