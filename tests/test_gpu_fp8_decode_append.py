"""The 8-bit decode step in one call (append, rotation and attention) against the append followed
by the attention: the same pool bytes and the same output, bit for bit."""
import pytest
import torch

from needle_amd import _lib, ops
from test_gpu_fp8_attention import DTYPES, SHAPES, Case

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Step:
    """A decode step: q, k and v views of one projection's rows, cos and sin of a wider table."""

    def __init__(self, case, rope=True, seed=0):
        c = self.case = case
        gen = torch.Generator().manual_seed(seed)
        n, h, hkv, d = len(c.lens), c.h, c.hkv, c.d
        rows = torch.randn(n, (h + 2 * hkv) * d, generator=gen)
        rows *= 2.0 ** torch.randint(-3, 4, (n, 1), generator=gen)
        rows = rows.to(c.dtype).to(DEV)
        self.q, self.k, self.v = (x.view(n, -1, d) for x in
                                  rows.split([h * d, hkv * d, hkv * d], dim=-1))
        cs = torch.randn(n, 2 * d, generator=gen).to(c.dtype).to(DEV)
        self.rope = dict(cos=cs[:, :d], sin=cs[:, d:]) if rope else {}
        self.table, self.ctx = c.table.to(DEV), c.ctx.to(DEV)
        self.heads = (c.scale, h, hkv, d)

    def pool(self):
        return self.case.codes.to(DEV).view(torch.float8_e4m3fn), self.case.scales.to(DEV)

    def together(self, pool, **more):
        return ops.paged_decode_fp8(self.q, *pool, self.table, self.ctx, *self.heads,
                                    new_k=self.k, new_v=self.v, **self.rope, **more)

    def apart(self, pool):
        q = self.q
        if self.rope:
            q = ops.kv_append_fp8(self.k, self.v, *pool, self.table, self.ctx, q=q, **self.rope)
        else:
            ops.kv_append_fp8(self.k, self.v, *pool, self.table, self.ctx)
        return ops.paged_decode_fp8(q, *pool, self.table, self.ctx, *self.heads)

    def check(self):
        a, b = self.pool(), self.pool()
        want, got = self.apart(a), self.together(b)
        for x, y in zip(a, b):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


LENS = [0, 1, 14, 15, 16, 17, 31, 32, 33, 63, 100, 129, 257, -1, -5]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("rope", [True, False])
def test_whole_row_blocks(shape, dtype, rope):
    Step(Case(shape, [1] * len(LENS), LENS, dtype, seed=1), rope).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(14, 2, 64, 16), (32, 8, 128, 16), (7, 1, 128, 64),
                                   (4, 4, 64, 1024)])
def test_shares(shape, dtype):
    """Tables wide enough for shares; contexts that end anywhere in them."""
    for lens in ([2900, 3, 1111, 0, -2], [1700 + 33 * i for i in range(9)], LENS + [5000]):
        Step(Case(shape, [1] * len(lens), lens, dtype, seed=2, extra_cols=2)).check()
    lens = [(53 * i) % 300 for i in range(130)] + [2000]
    Step(Case(shape, [1] * len(lens), lens, dtype, seed=3)).check()


@pytest.mark.parametrize("lens", [[48, 47, 63, 100, 5], [2048, 2047, 2500, 64, 2063]])
def test_tables_that_end_and_bad_blocks(lens):
    """At and past the table's end the last column is written again, at the position's row of it;
    an invalid block is not written."""
    for bs in (16, 64):
        c = Case((8, 2, 64, bs), [1] * 5, lens, seed=4, extra_cols=0)
        cols = 48 // bs if lens[0] == 48 and bs == 16 else 2048 // bs if lens[0] == 2048 else 1
        c.table = c.table[:, :cols].contiguous()
        Step(c).check()
        c.table[1, -1] = -1
        c.table[3, 0] = c.nb
        c.table[4] = 1 << 30
        Step(c).check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_are_not_finite(dtype):
    c = Case((4, 2, 64, 16), [1] * 4, [3, 40, 17, 90], dtype, seed=5)
    s = Step(c, rope=False)
    s.k[0, 0, 5], s.v[1, 1, 63], s.v[2, 0, 0] = float("inf"), float("nan"), float("-inf")
    s.k[3], s.v[3] = 0.0, 0.0
    a, b = s.pool(), s.pool()
    want, got = s.apart(a), s.together(b)
    assert torch.equal(got.isnan(), want.isnan()) and got.isnan().any()
    assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
    for x, y in zip(a, b):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_workspace_output_and_the_python_path(monkeypatch):
    for lens in ([40, 7], [3000, 7]):
        s = Step(Case((14, 2, 64, 16), [1, 1], lens, seed=6))
        want = s.apart(s.pool())
        need = ops.fp8_attention_workspace_bytes(2, 2, 1, s.table.shape[1] * 16, 14, 2, 64)
        ws = ops.decode_workspace(need, DEV)
        ws.fill_(0xFF)
        out = torch.empty_like(want)
        assert s.together(s.pool(), out=out, workspace=ws) is out and torch.equal(out, want)
        assert _lib.NATIVE is not None
        pool = s.pool()
        assert _lib.NATIVE.fp8_attention(
            s.q, *pool, s.table, None, s.ctx, 1, 0, *s.heads, s.k, s.v, s.rope["cos"],
            s.rope["sin"]) is not None
        monkeypatch.setattr(_lib, "NATIVE", None)
        assert torch.equal(s.together(s.pool()), want)
        monkeypatch.undo()


@pytest.mark.parametrize("lens", [[40, 7, 300], [3000, 7, 1200]])
def test_captured_and_replayed(lens):
    s = Step(Case((32, 8, 128, 16), [1] * 3, lens, seed=7))
    a, b = s.pool(), s.pool()
    s.apart(a)
    s.together(b)         # (appends too: both pools have had the first step)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = s.together(b)
    for r in range(4):
        s.q.normal_()
        s.k.normal_()
        s.v.normal_()
        s.ctx += 1
        want = s.apart(a)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), r
    for x, y in zip(a, b):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_refusals():
    s = Step(Case((8, 2, 64, 16), [1, 1], [5, 6], seed=8))
    pool = s.pool()
    args = (s.q, *pool, s.table, s.ctx, *s.heads)
    cos, sin = s.rope["cos"], s.rope["sin"]
    bad = [(ValueError, "go together", dict(new_k=s.k)),
           (ValueError, "cos / sin need", dict(cos=cos, sin=sin)),
           (ValueError, "cos and sin go", dict(new_k=s.k, new_v=s.v, cos=cos)),
           (TypeError, "new_v dtype", dict(new_k=s.k, new_v=s.v.half())),
           (ValueError, "one row per", dict(new_k=s.k[:1], new_v=s.v)),
           (ValueError, "new_k must be", dict(new_k=s.k[..., :32], new_v=s.v)),
           (TypeError, "cos dtype", dict(new_k=s.k, new_v=s.v, cos=cos.half(), sin=sin)),
           (ValueError, "sin must be", dict(new_k=s.k, new_v=s.v, cos=cos, sin=sin[:1])),
           (ValueError, "on cuda", dict(new_k=s.k, new_v=s.v.cpu()))]
    for kind, text, more in bad:
        with pytest.raises(kind, match=text):
            ops.paged_decode_fp8(*args, **more)
    for x, y in zip(pool, s.pool()):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    empty = ops.paged_decode_fp8(s.q[:0], *pool, s.table[:0], s.ctx[:0], *s.heads, new_k=s.k[:0],
                                 new_v=s.v[:0])
    assert empty.shape == (0, 8, 64)
