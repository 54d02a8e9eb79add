"""The 8-bit pool's append and read-back on the GPU against the definition, bit for bit."""
import pytest
import torch

from needle_amd import ops
from oracle import fp8_ref, paged_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float16]
# heads, kv heads, head_dim, block size
SHAPES = [(14, 2, 64, 16), (32, 8, 128, 16), (28, 4, 128, 64), (3, 3, 64, 1024), (16, 1, 128, 32)]


def _rows(n, h, d, dtype, gen):
    """Rows of very different sizes, zeros, subnormals and the format's ends among them."""
    x = torch.randn(n, h, d, generator=gen, dtype=torch.float32)
    span = 2 if dtype == torch.float16 else 30
    x *= 2.0 ** torch.randint(-span, span + 1, (n, h, 1), generator=gen).float()
    if n > 2:
        x[0] = 0.0
        x[1, 0] *= 2.0 ** (-22 if dtype == torch.float16 else -120)
        x[2, 0, 5] = torch.finfo(dtype).max
    # the border of the scale: 448 and 449 times a power of two
    x[n - 1, 0, :2] = torch.tensor([448.0, 3.0])
    if h > 1:
        x[n - 1, 1, :2] = torch.tensor([450.0, -3.0])
        x[n - 1, 1, 2:] = x[n - 1, 1, 2:].clamp(-300, 300)
    return x.to(dtype)


def _quantised(rows):
    codes, scales = zip(*(fp8_ref.quantise_row(r.double().tolist())
                          for r in rows.reshape(-1, rows.shape[-1])))
    return (torch.tensor(codes, dtype=torch.uint8).view(rows.shape),
            torch.tensor(scales, dtype=torch.uint8).view(rows.shape[:-1]))


def _pool(nb, hkv, bs, d, gen):
    """A pool of random bytes: a stray write shows."""
    return ops.Fp8KVCache(
        torch.randint(0, 256, (2, nb, hkv, bs, d), generator=gen, dtype=torch.uint8),
        torch.randint(1, 255, (2, nb, hkv, bs), generator=gen, dtype=torch.uint8))


def _expect(pool, rows_k, rows_v, table, lens, cu):
    codes, scales = pool.codes.clone(), pool.scales.clone()
    nb, bs = codes.shape[1], codes.shape[3]
    (kc, ks), (vc, vs) = _quantised(rows_k), _quantised(rows_v)
    for i in range(table.shape[0]):
        for t in range(int(cu[i]), int(cu[i + 1])):
            at = fp8_ref.slot(table[i], int(lens[i]) + t - int(cu[i]), bs, nb)
            if at is not None:
                codes[0, at[0], :, at[1]], scales[0, at[0], :, at[1]] = kc[t], ks[t]
                codes[1, at[0], :, at[1]], scales[1, at[0], :, at[1]] = vc[t], vs[t]
    return codes, scales


def _case(shape, counts, lens, seed, extra_cols=0):
    h, hkv, d, bs = shape
    gen = torch.Generator().manual_seed(seed)
    need = [-(-max(c + n, 1) // bs) for c, n in zip(lens, counts)]
    nb = sum(need) + 2
    perm = torch.randperm(nb - 1, generator=gen).tolist()
    table = torch.full((len(lens), max(need) + extra_cols), nb - 1, dtype=torch.int32)
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(perm[:n], dtype=torch.int32)
        perm = perm[n:]
    cu = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32)
    return gen, _pool(nb, hkv, bs, d, gen), table, torch.tensor(lens, dtype=torch.int32), cu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_append_is_the_definition_and_reads_back(shape, dtype):
    h, hkv, d, bs = shape
    counts, lens = [1, 7, 0, 18, 3], [0, 15, 4, bs - 2, -1]   # a negative position is dropped
    gen, pool, table, ctx, cu = _case(shape, counts, lens, 1)
    total = int(cu[-1])
    k, v = _rows(total, hkv, d, dtype, gen), _rows(total, hkv, d, dtype, gen)
    want = _expect(pool, k, v, table, ctx, cu)
    g = ops.Fp8KVCache(pool.codes.to(DEV), pool.scales.to(DEV))
    ops.kv_append_fp8(k.to(DEV), v.to(DEV), *g, table.to(DEV), ctx.to(DEV), cu.to(DEV))
    assert torch.equal(g.scales.cpu(), want[1])
    assert torch.equal(g.codes.cpu(), want[0])
    # read back: the chunk and two tokens before it; past cu_seqlens nothing is written
    first = (ctx - 2).to(DEV)
    n = [c + 2 for c in counts]
    rcu = torch.tensor([0] + list(torch.tensor(n).cumsum(0)), dtype=torch.int32)
    rk, rv = ops.kv_read_fp8(g.codes.view(torch.float8_e4m3fn), g.scales, table.to(DEV), first,
                             rcu.to(DEV), sum(n), dtype=dtype)
    vals = fp8_ref.values(*want)
    for i in range(len(lens)):
        for t in range(n[i]):
            at = fp8_ref.slot(table[i], lens[i] - 2 + t, bs, pool.codes.shape[1])
            x = vals[:, at[0], :, at[1]] if at is not None else torch.zeros(2, hkv, d)
            for p, got in ((0, rk), (1, rv)):
                a, b = got[int(rcu[i]) + t].cpu(), x[p].to(dtype)
                assert torch.equal(a.isnan(), b.isnan())
                assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)), (i, t, p)


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_is_not_finite_becomes_nan_and_leaves_the_rest(dtype):
    gen, pool, table, ctx, cu = _case((4, 2, 64, 16), [2], [3], 2)
    k = torch.randn(2, 2, 64, generator=gen).to(dtype)
    k[0, 0, 9], k[0, 0, 40], k[0, 1, 0] = float("inf"), float("nan"), float("-inf")
    k[1, 1] = float("nan")
    v = k.flip(0).contiguous()
    want = _expect(pool, k, v, table, ctx, cu)
    g = ops.Fp8KVCache(pool.codes.to(DEV), pool.scales.to(DEV))
    ops.kv_append_fp8(k.to(DEV), v.to(DEV), *g, table.to(DEV), ctx.to(DEV), cu.to(DEV))
    assert torch.equal(g.scales.cpu(), want[1])
    # a NaN's sign is no part of it
    nan = (want[0] & 127) == 127
    assert torch.equal((g.codes.cpu() & 127) == 127, nan)
    assert torch.equal(g.codes.cpu()[~nan], want[0][~nan])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES[:3])
@pytest.mark.parametrize("decode", [True, False])
def test_rotation_has_the_models_roundings(shape, dtype, decode):
    h, hkv, d, bs = shape
    counts, lens = ([1] * 6, [0, 5, 15, 16, 31, 9]) if decode else ([5, 1, 30], [0, 12, 3])
    gen, pool, table, ctx, cu = _case(shape, counts, lens, 3)
    total = int(cu[-1])
    # views of a fused projection's rows; cos and sin rows of a wider table
    qkv = torch.randn(total, (h + 2 * hkv) * d, generator=gen).to(dtype)
    q, k, v = (x.view(total, -1, d) for x in qkv.split([h * d, hkv * d, hkv * d], dim=-1))
    cs = torch.randn(total, 2 * d, generator=gen).to(dtype)
    cos, sin = cs[:, :d], cs[:, d:]
    qr, kr = paged_ref.apply_rope(q, k, cos, sin)
    want = _expect(pool, kr, v, table, ctx, cu)
    g = ops.Fp8KVCache(pool.codes.to(DEV), pool.scales.to(DEV))
    dqkv, dcs = qkv.to(DEV), cs.to(DEV)
    dq, dk, dv = (x.view(total, -1, d) for x in dqkv.split([h * d, hkv * d, hkv * d], dim=-1))
    got = ops.kv_append_fp8(dk, dv, *g, table.to(DEV), ctx.to(DEV),
                            None if decode else cu.to(DEV), q=dq, cos=dcs[:, :d], sin=dcs[:, d:])
    assert torch.equal(got.cpu().view(torch.int16), qr.contiguous().view(torch.int16))
    assert torch.equal(g.scales.cpu(), want[1]) and torch.equal(g.codes.cpu(), want[0])
    # k alone
    g2 = ops.Fp8KVCache(pool.codes.to(DEV), pool.scales.to(DEV))
    assert ops.kv_append_fp8(dk, dv, *g2, table.to(DEV), ctx.to(DEV),
                             None if decode else cu.to(DEV), cos=dcs[:, :d],
                             sin=dcs[:, d:]) is None
    assert torch.equal(g2.codes, g.codes) and torch.equal(g2.scales, g.scales)


def test_the_table_ends_and_bad_blocks():
    """Past the table's columns the last one is written again; an invalid id is not written."""
    shape = (4, 2, 64, 16)
    gen, pool, table, ctx, cu = _case(shape, [40, 3], [0, 2], 4)
    table = table[:, :2].contiguous()
    table[1, 0] = pool.codes.shape[1]     # one past the pool
    total = int(cu[-1])
    k, v = (torch.randn(total, 2, 64, generator=gen).bfloat16() for _ in range(2))
    # two positions share a slot past the end (the order of their writes is not defined): give
    # them the same row
    k[32:40], v[32:40] = k[16:24], v[16:24]
    want = _expect(pool, k, v, table, ctx, cu)
    g = ops.Fp8KVCache(pool.codes.to(DEV), pool.scales.to(DEV))
    ops.kv_append_fp8(k.to(DEV), v.to(DEV), *g, table.to(DEV), ctx.to(DEV), cu.to(DEV))
    assert torch.equal(g.codes.cpu(), want[0]) and torch.equal(g.scales.cpu(), want[1])


def test_rows_past_the_last_sequence_are_left():
    shape = (4, 2, 64, 16)
    gen, pool, table, ctx, cu = _case(shape, [3, 2], [0, 2], 5)
    k, v = (torch.randn(9, 2, 64, generator=gen).bfloat16() for _ in range(2))   # 4 of padding
    want = _expect(pool, k, v, table, ctx, cu)
    g = ops.Fp8KVCache(pool.codes.to(DEV), pool.scales.to(DEV))
    q = torch.randn(9, 4, 64, generator=gen).bfloat16()
    cos, sin = torch.ones(9, 64).bfloat16(), torch.zeros(9, 64).bfloat16()
    out = ops.kv_append_fp8(k.to(DEV), v.to(DEV), *g, table.to(DEV), ctx.to(DEV), cu.to(DEV),
                            q=q.to(DEV), cos=cos.to(DEV), sin=sin.to(DEV))
    assert torch.equal(g.codes.cpu(), want[0]) and torch.equal(g.scales.cpu(), want[1])
    assert torch.equal(out.cpu(), q)


def test_refusals():
    shape = (4, 2, 64, 16)
    gen, pool, table, ctx, cu = _case(shape, [3, 2], [0, 2], 6)
    g = ops.Fp8KVCache(pool.codes.to(DEV), pool.scales.to(DEV))
    k = torch.zeros(5, 2, 64, dtype=torch.bfloat16, device=DEV)
    t, c, u = table.to(DEV), ctx.to(DEV), cu.to(DEV)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        ops.kv_append_fp8(k.float(), k.float(), *g, t, c, u)
    with pytest.raises(TypeError, match="v dtype"):
        ops.kv_append_fp8(k, k.half(), *g, t, c, u)
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        ops.kv_append_fp8(k, k, g.codes.view(torch.int8), g.scales, t, c, u)
    with pytest.raises(ValueError, match="kv_scales must be"):
        ops.kv_append_fp8(k, k, g.codes, g.scales[:, :1], t, c, u)
    with pytest.raises(ValueError, match="head_dim 64 and 128"):
        ops.kv_append_fp8(k, k, g.codes[..., :32].contiguous(), g.scales, t, c, u)
    with pytest.raises(ValueError, match="power of two"):
        ops.kv_append_fp8(k, k, g.codes[:, :, :, :8].contiguous(),
                          g.scales[..., :8].contiguous(), t, c, u)
    with pytest.raises(ValueError, match="one token per sequence"):
        ops.kv_append_fp8(k, k, *g, t, c)
    with pytest.raises(ValueError, match="pass cos and sin"):
        ops.kv_append_fp8(k, k, *g, t, c, u, q=k)
    with pytest.raises(TypeError, match="dtype must be"):
        ops.kv_read_fp8(*g, t, c, u, 5, dtype=torch.float32)
    with pytest.raises(ValueError, match="num_seqs"):
        ops.kv_read_fp8(*g, t, c, u[:2], 5)
    assert ops.kv_append_fp8(k[:0], k[:0], *g, t, c, u) is None
    empty = ops.kv_read_fp8(*g, t, c, u, 0)
    assert empty[0].shape == (0, 2, 64)
    assert torch.equal(g.codes.cpu(), pool.codes)


def test_captured_steps_replay(monkeypatch):
    """Append and read in a graph, replayed with eager work and synchronisations between."""
    shape = (14, 2, 64, 16)
    gen, pool, table, ctx, cu = _case(shape, [4, 1, 9], [3, 20, 0], 7)
    total = int(cu[-1])
    k, v = (torch.randn(total, 2, 64, generator=gen).bfloat16().to(DEV) for _ in range(2))
    t, c, u = table.to(DEV), ctx.to(DEV), cu.to(DEV)
    g = ops.Fp8KVCache(pool.codes.to(DEV), pool.scales.to(DEV))
    e = ops.Fp8KVCache(pool.codes.to(DEV), pool.scales.to(DEV))

    def step(p):
        ops.kv_append_fp8(k, v, *p, t, c, u)
        return ops.kv_read_fp8(*p, t, c, u, total)

    step(g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(g)
    for r in range(4):
        k.normal_()
        v.normal_()
        want = step(e)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(g.codes, e.codes) and torch.equal(g.scales, e.scales), r
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), r


@pytest.mark.parametrize("shape", SHAPES[:3])
def test_q_is_rotated_in_place(shape):
    """out may be q itself."""
    h, hkv, d, bs = shape
    gen, pool, table, ctx, cu = _case(shape, [3, 20], [5, 0], 8)
    q, k, v = (torch.randn(23, n, d, generator=gen).bfloat16().to(DEV) for n in (h, hkv, hkv))
    cos, sin = (torch.randn(23, d, generator=gen).bfloat16().to(DEV) for _ in range(2))
    meta = [x.to(DEV) for x in (table, ctx, cu)]
    a, b = ([x.to(DEV) for x in pool] for _ in range(2))
    want = ops.kv_append_fp8(k, v, *a, *meta, q=q, cos=cos, sin=sin)
    got = ops.kv_append_fp8(k, v, *b, *meta, q=q, cos=cos, sin=sin, out=q)
    assert got is q and torch.equal(got, want)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
