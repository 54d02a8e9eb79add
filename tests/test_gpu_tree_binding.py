"""The native bindings of the trees' and the bounded caches' operators against ops.py's own path: the
same bytes for the calls they take, the same errors for the others."""
import pytest
import torch

from needle_amd import _lib, ops
from test_gpu_native_binding import _both, _same, native  # noqa: F401 - native is a fixture

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def test_mask_and_selection(native, monkeypatch):  # noqa: F811
    gen = torch.Generator().manual_seed(1)
    parents, cu = i32([-1, 0, 0, 1, -1, 0, 5]), i32([0, 4, 4, 7])
    assert native.tree_mask(parents, cu, 4) is not None
    for change in [dict(), dict(most=70), dict(most=1), dict(most=0), dict(most=-1),
                   dict(most=4.0), dict(parents=parents.long()), dict(parents=parents.cpu()),
                   dict(parents=parents[:0], cu=cu[:1]), dict(cu=cu.long()), dict(cu=cu[:0]),
                   dict(parents=i32([[1, 2], [3, 4]])[:, 0])]:
        a = dict(parents=parents, cu=cu, most=4) | change
        _same(*_both(monkeypatch, lambda: ops.tree_mask(a["parents"], a["cu"], a["most"])))
    mass = torch.rand(12, 2, 16, generator=gen).to(DEV)
    table, lens = i32([[0, 5, 3, 11], [2, 7, 8, 1]]), i32([60, 20])
    assert native.kv_select(mass, table, lens, 24, 4, 8) is not None
    for change in [dict(), dict(budget=100), dict(budget=0), dict(sinks=30), dict(recent=-1),
                   dict(budget=12.0), dict(mass=mass.double()), dict(mass=mass[:, :1]),
                   dict(mass=mass.cpu()), dict(mass=mass[0]), dict(table=table[:, 1:]),
                   dict(table=table[:, ::2]), dict(table=table.long()), dict(lens=lens[:1]),
                   dict(lens=-lens), dict(table=table[:0], lens=lens[:0]),
                   dict(table=table[:, :0])]:
        a = dict(mass=mass, table=table, lens=lens, budget=24, sinks=4, recent=8) | change
        _same(*_both(monkeypatch, lambda: ops.kv_select(
            a["mass"], a["table"], a["lens"], a["budget"], sinks=a["sinks"], recent=a["recent"])))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention(native, monkeypatch, dtype, fp8):  # noqa: F811
    gen = torch.Generator().manual_seed(2)
    h, hkv, d, bs, nb = 4, 2, 64, 16, 100
    if fp8:
        codes = torch.randint(0, 120, (2, nb, hkv, bs, d), generator=gen, dtype=torch.uint8)
        scales = torch.randint(118, 124, codes.shape[:4], generator=gen, dtype=torch.uint8)
        pool = ops.Fp8KVCache(codes.to(DEV).view(torch.float8_e4m3fn), scales.to(DEV))
    else:
        pool = torch.randn(2, nb, hkv, bs, d, generator=gen).to(dtype).to(DEV)
    q = torch.randn(14, h, d, generator=gen).to(dtype).to(DEV)
    table = torch.randperm(nb, generator=gen)[:90].to(torch.int32).view(3, 30).to(DEV)
    lens, cu = i32([7, 3, 400]), i32([0, 9, 9, 14])
    parents = i32([-1, 0, 1, 1, 2, 0, 3, 6, 6, -1, 0, 0, 1, 3])
    mask, _ = ops.tree_mask(parents, cu, 9)
    mass = torch.rand(nb, hkv, bs, generator=gen).to(DEV)
    base = dict(q=q, pool=pool, table=table, lens=lens, cu=cu, most=9, scale=0.125, h=h, d=d,
                bound=0, mask=mask, mass=mass, decay=0.5)

    def tree(a):
        return ops.tree_attention(a["q"], a["pool"], a["table"], a["cu"], a["lens"], a["mask"],
                                  a["most"], a["scale"], a["h"], hkv, a["d"],
                                  max_context_len=a["bound"])

    def weigh(a):
        m = a["mass"].clone()
        return ops.attention_mass(a["q"], a["pool"], a["table"], a["lens"], m, a["scale"], a["h"],
                                  hkv, a["d"], cu_seqlens=a["cu"], max_seqlen=a["most"],
                                  max_context_len=a["bound"], decay=a["decay"]), m
    taken = native.tree_attention(q, *(pool if fp8 else (pool, None)), table, cu, lens, mask, 9, 0,
                                  0.125, h, hkv, d)
    assert taken is not None
    changes = [dict(), dict(bound=400), dict(table=table.long()), dict(lens=lens[:2]),
               dict(table=table[:, ::2]), dict(table=table[:, 3:]), dict(table=table[:, :0]),
               dict(table=table.cpu()), dict(lens=-lens), dict(cu=cu[:3]), dict(cu=cu.long()),
               dict(q=q[..., :32]), dict(q=q.double()), dict(q=q.float()), dict(q=q[:0]),
               dict(scale=1), dict(most=0), dict(most=-1), dict(most=9.0), dict(h=3),
               dict(d=128), dict(bound=-1), dict(q=q.transpose(0, 1)),
               dict(q=q.to(torch.float16 if dtype == torch.bfloat16 else torch.bfloat16))]
    for change in changes + [dict(mask=mask[:5]), dict(mask=mask.int()), dict(mask=mask.cpu()),
                             dict(mask=mask.repeat(1, 3)), dict(mask=mask.repeat(1, 3)[:, :1]),
                             dict(mask=mask[:, :0]), dict(mask=mask[:, 0])]:
        if fp8 and "q" in change and change["q"].dtype in (torch.float16, torch.bfloat16) and \
                change["q"].dtype != dtype:
            continue                  # an 8-bit pool takes either
        _same(*_both(monkeypatch, lambda: tree(base | change)))
    if fp8:
        return
    assert native.attention_mass(q, pool, table, cu, lens, mass.clone(), 9, 0, 0.125, h, hkv, d,
                                 0.5) is not None
    for change in changes + [dict(cu=None, most=1, q=q[:3]), dict(cu=None, q=q[:3]),
                             dict(cu=None, most=1), dict(mass=mass[:50]), dict(decay=0),
                             dict(mass=mass.double()), dict(mass=mass.cpu()), dict(decay=0.0),
                             dict(mass=mass.transpose(1, 2)), dict(pool=pool[:, :50])]:
        _same(*_both(monkeypatch, lambda: weigh(base | change)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_verify(native, monkeypatch, dtype):  # noqa: F811
    gen = torch.Generator().manual_seed(3)
    vocab = 1003
    logits = torch.randn(9, vocab, generator=gen).to(dtype).to(DEV)
    ids = torch.randint(0, vocab, (9,), generator=gen).to(DEV)
    parents, cu = i32([-1, 0, 0, 1, -1, -1, 0, 0, 2]), i32([0, 4, 5, 9])
    u, t = torch.rand(9, generator=gen).to(DEV), torch.tensor([0.7, 0.0, 1.0], device=DEV)
    assert native.verify_tree(logits, ids, parents, cu, u, t) is not None
    wide = torch.randn(9, 2000, generator=gen).to(dtype).to(DEV)
    for change in [dict(), dict(t=None), dict(logits=wide[:, 7:7 + vocab]), dict(u=u[:8]),
                   dict(logits=logits.t()), dict(logits=logits[:8]), dict(logits=logits.cpu()),
                   dict(logits=logits.double()), dict(ids=ids.int()), dict(ids=ids.float()),
                   dict(ids=ids[:8]), dict(cu=cu.long()), dict(parents=parents.long()),
                   dict(parents=parents[:8]), dict(parents=parents.cpu()), dict(u=u.double()),
                   dict(t=t[:2]), dict(t=t.double()), dict(t=t.cpu()), dict(logits=logits[:, :1]),
                   dict(logits=logits[:0], ids=ids[:0], u=u[:0], cu=cu[:1], t=t[:0],
                        parents=parents[:0]), dict(logits=wide[:, :0])]:
        a = dict(logits=logits, ids=ids, parents=parents, cu=cu, u=u, t=t) | change
        _same(*_both(monkeypatch, lambda: ops.verify_tree(
            a["logits"], a["ids"], a["parents"], a["cu"], a["u"], temperature=a["t"])))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, "fp8"])
def test_compact(native, monkeypatch, dtype):  # noqa: F811
    gen = torch.Generator().manual_seed(4)
    shape = (2, 20, 2, 16, 64)
    if dtype == "fp8":
        pools = [ops.Fp8KVCache(
            torch.randint(0, 120, shape, generator=gen, dtype=torch.uint8).to(DEV).view(
                torch.float8_e4m3fn),
            torch.randint(0, 255, shape[:4], generator=gen, dtype=torch.uint8).to(DEV))
            for _ in range(3)]
        args = ([p.codes for p in pools], [p.scales for p in pools])
    else:
        pools = [torch.randn(shape, generator=gen).to(dtype).to(DEV) for _ in range(3)]
        args = (pools, None)
    mass = torch.rand(shape[1:4], generator=gen).to(DEV)
    table = i32([[0, 5, 3, 11], [2, 7, 8, 1]])
    keep = torch.stack([torch.randperm(60, generator=gen)[:9].sort().values for _ in range(4)])
    keep = keep.to(torch.int32).view(2, 2, 9).to(DEV)
    counts, first, cu, dst = i32([9, 4]), i32([2, 0]), i32([0, 9, 18]), i32([[13, 14], [15, 16]])
    assert native.kv_compact(*args, table, keep, counts, None, None, None, None) is True

    def compact(pools=pools, table=table, keep=keep, counts=counts, first=None, cu=None, dst=None,
                mass=None):
        if isinstance(pools, list) and dtype != "fp8":
            pools = [p.clone() for p in pools]
        elif isinstance(pools, list):
            pools = [ops.Fp8KVCache(*(x.clone() for x in p)) for p in pools]
        m = None if mass is None else mass.clone()
        ops.kv_compact(pools, table, keep, counts, first=first, cu_seqlens=cu, dst_table=dst,
                       mass=m)
        flat = tuple(x for p in pools for x in ((p,) if torch.is_tensor(p) else p))
        return flat if m is None else (*flat, m)
    flat = keep[:, 0].reshape(-1)
    for change in [dict(), dict(first=first), dict(keep=flat, cu=cu, first=first), dict(dst=dst),
                   dict(mass=mass), dict(dst=dst, mass=mass, first=first), dict(keep=keep.long()),
                   dict(keep=flat), dict(cu=cu), dict(keep=flat, cu=cu[:2]),
                   dict(counts=counts[:1]), dict(counts=-counts), dict(first=first[:1]),
                   dict(first=first.long()), dict(dst=dst[:1]), dict(dst=dst.long()),
                   dict(dst=dst[:, :0]), dict(mass=mass[:5]), dict(mass=mass.double()),
                   dict(table=table[:, 1:]), dict(table=table[:, ::2]), dict(table=table[:, :0]),
                   dict(keep=keep[..., ::2]), dict(keep=keep[..., :0]), dict(pools=[]),
                   dict(table=table[:0], keep=keep[:0], counts=counts[:0])]:
        _same(*_both(monkeypatch, lambda: compact(**change)))
