"""Draft verification where cu_seqlens does not give every sequence its row: a draft whose row of
draft_probs is not there cannot be judged, and is not accepted."""
import torch

import pytest

from needle_amd import _lib, ops
from oracle import fp8_ref
from test_gpu_verify import DEV, _case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_drafts_without_a_row_are_rejected(dtype):
    """An empty sequence first: the second one's first draft would be judged by row -1, its second
    by row 0."""
    vocab = 3001
    logits, ids, _, u, _, draft = _case([3], vocab, dtype, 1)
    cu = torch.tensor([0, 0, 3], dtype=torch.int32)
    u[:2] = 1e-6                              # what could be accepted would be
    tokens, accepted = ops.verify_drafts(logits.to(DEV), ids.to(DEV), cu.to(DEV), u.to(DEV),
                                         draft_probs=draft[:1].to(DEV))
    # rejected, and nothing to take off the target's own distribution
    none = ids.clone()
    none[1] = -1
    want = fp8_ref.verify(logits, none, [0, 3], u, None, torch.zeros(2, vocab))
    assert accepted.tolist() == [0, 0] and want[1] == [0]
    assert tokens.tolist() == want[0]


def test_drafts_without_any_row_are_rejected():
    """As many rows as sequences: draft_probs is empty, and not the same as none given."""
    vocab = 999
    logits, ids, _, u, _, _ = _case([3], vocab, torch.bfloat16, 3)
    cu = torch.tensor([0, 0, 0, 3], dtype=torch.int32)
    u[:2] = 1e-6
    none = ids.clone()
    none[1] = -1
    want = fp8_ref.verify(logits, none, [0, 3], u, None, torch.zeros(2, vocab))
    args = [x.to(DEV) for x in (logits, ids, cu, u)]
    for empty in (torch.empty(0, vocab, device=DEV), torch.empty(5, vocab, device=DEV)[:0]):
        for native in (_lib.NATIVE, None):
            with pytest.MonkeyPatch.context() as m:
                m.setattr(_lib, "NATIVE", native)
                tokens, accepted = ops.verify_drafts(*args, draft_probs=empty)
            assert accepted.tolist() == [0, 0, 0] and tokens.tolist() == want[0]


def test_sequences_without_rows_between():
    """Without draft distributions an empty sequence has nothing, and changes nothing."""
    logits, ids, cu, u, _, _ = _case([4, 2, 3], 999, torch.bfloat16, 2, False)
    want = fp8_ref.verify(logits, ids, cu, u, None, None)
    cu = torch.tensor([0, 0, 4, 4, 4, 6, 9], dtype=torch.int32)
    tokens, accepted = ops.verify_drafts(logits.to(DEV), ids.to(DEV), cu.to(DEV), u.to(DEV))
    assert tokens.tolist() == want[0]
    assert accepted.tolist() == [0, want[1][0], 0, 0, *want[1][1:]]
