"""Long chunks over the 8-bit pool whose keys, by the call's bounds, do not fit the workspace's 16-bit
pool at once: the sequences go through it a group at a time.  Against the definition in float64,
bounds as in test_gpu_fp8_attention."""
import pytest
import torch

from needle_amd import _lib, ops
from test_gpu_fp8_attention import DEV, DTYPES, Case

pytestmark = pytest.mark.gpu

SHAPE = (8, 2, 64, 16)


def _case(held, counts, lens, **more):
    """A table so wide that `held` sequences of its keys fit."""
    row = 2 * 64 * 4 * 16                        # bytes of a column in 16 bits
    cols = _lib.NDL_FP8_UNPACK_BYTES // (held * row) - 8
    need = max(max(1, -(-(n + m) // 16)) for n, m in zip(lens, counts))
    c = Case(SHAPE, counts, lens, extra_cols=cols - need, **more)
    size = ops.fp8_attention_workspace_bytes(len(lens), sum(counts), max(counts), cols * 16, *SHAPE)
    assert c.table.shape[1] == cols and held * cols * row <= size < (held + 1) * cols * row
    assert held < len(lens)
    return c


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("held", [1, 2])
def test_groups(held, dtype):
    c = _case(held, [120, 5, 0, 90, 77], [300, 40, 9, 0, -3], dtype=dtype, seed=1)
    # a NaN among the values of the second group's chunk
    pos = 60
    c.codes[1, int(c.table[3, pos // 16]), 1, pos % 16, 11] = 0x7F
    got = c.run()
    c.check(got)
    assert got[125:185].isfinite().all() and got[185:215, 4:, 11].isnan().all()
    # a bound that says how few keys there are: one group
    c.check(c.run(max_context_len=300))


def test_every_row_of_a_group_is_its_own():
    """More sequences than a group holds twice over, rows behind the last one left as they were."""
    counts = [60, 1, 33, 64, 7, 20, 58]
    c = _case(3, counts, [17, 500, 0, 31, 90, 2, 250], seed=2)
    n = int(c.cu[-1])
    q = torch.full((n + 3, 8, 64), float("nan"), dtype=c.dtype, device=DEV)
    q[:n] = c.q.to(DEV)
    out = torch.full_like(q, 5.0)
    c.check(c.run(q=q, out=out))
    assert (out[n:] == 5.0).all()


def test_captured_and_replayed():
    c = _case(2, [70, 60, 65], [200, 40, 333], seed=3)
    q, pool = c.q.to(DEV), (c.codes.to(DEV), c.scales.to(DEV))
    t, cu, ctx = c.table.to(DEV), c.cu.to(DEV), c.ctx.to(DEV)

    def step():
        return ops.varlen_prefill_fp8(q, *pool, t, cu, ctx, 70, c.scale, 8, 2, 64)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        q.normal_()
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
