"""The native bindings of the 8-bit pool's operators and of the draft verification against ops.py's
own path: the same bytes for the calls they take, the same errors for the others."""
import pytest
import torch

from needle_amd import _lib, ops
from test_gpu_native_binding import _both, _same, native  # noqa: F401 - native is a fixture

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _pool(gen, nb, hkv, bs, d):
    codes = torch.randint(0, 120, (2, nb, hkv, bs, d), generator=gen, dtype=torch.uint8)
    scales = torch.randint(118, 124, codes.shape[:4], generator=gen, dtype=torch.uint8)
    return codes.to(DEV).view(torch.float8_e4m3fn), scales.to(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_cache_and_attention(native, monkeypatch, dtype):  # noqa: F811
    gen = torch.Generator().manual_seed(1)
    h, hkv, d, bs, new, ctx = 4, 2, 64, 16, [9, 0, 5], [7, 3, 400]
    n = sum(new)
    qkv = torch.randn(n, (h + 2 * hkv) * d, generator=gen).to(dtype).to(DEV)
    q, k, v = (x.view(n, -1, d) for x in qkv.split([h * d, hkv * d, hkv * d], dim=-1))
    codes, scales = _pool(gen, 100, hkv, bs, d)
    table = torch.randperm(100, generator=gen)[:3 * 30].to(torch.int32).view(3, 30).to(DEV)
    lens = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 9, 9, 14], dtype=torch.int32, device=DEV)
    ang = torch.rand(n, d, generator=gen)
    cos, sin = ang.cos().to(dtype).to(DEV), ang.sin().to(dtype).to(DEV)
    first3 = dict(q=q[:3], k=k[:3], v=v[:3], cos=cos[:3], sin=sin[:3], cu=None)

    def append(q=q, k=k, v=v, cos=cos, sin=sin, codes=codes, scales=scales, table=table,
               lens=lens, cu=cu):
        pool = codes.clone(), scales.clone()
        out = ops.kv_append_fp8(k, v, *pool, table, lens, cu, q=q, cos=cos, sin=sin)
        return pool if out is None else (*pool, out)

    def read(codes=codes, scales=scales, table=table, lens=lens, cu=cu, n=n, dtype=dtype):
        k, v = ops.kv_read_fp8(codes, scales, table, lens, cu, n, dtype=dtype)
        return k[:14], v[:14]         # what is past the last sequence is not written

    def chunk(q=q, codes=codes, scales=scales, table=table, lens=lens, cu=cu, most=9, scale=0.125,
              h=h, d=d, bound=400):
        return ops.varlen_prefill_fp8(q, codes, scales, table, cu, lens, most, scale, h, hkv, d,
                                      max_context_len=bound)

    def decode(q=q[:3], codes=codes, scales=scales, table=table, lens=lens, scale=0.125, h=h,
               d=d):
        return ops.paged_decode_fp8(q, codes, scales, table, lens, scale, h, hkv, d)

    assert native.kv_append_fp8(k, v, codes.clone(), scales.clone(), table, lens, cu, q, cos,
                                sin) is not None
    code = {torch.bfloat16: 0, torch.float16: 1}[dtype]
    assert native.kv_read_fp8(codes, scales, table, lens, cu, n, code) is not None
    assert native.fp8_attention(q, codes, scales, table, cu, lens, 9, 0, 0.125, h, hkv,
                                d) is not None
    changes = [dict(), dict(table=table.long()), dict(lens=lens[:2]), dict(table=table[:, ::2]),
               dict(table=table[:, 3:]), dict(table=table[:, :0]), dict(table=table.cpu()),
               dict(codes=codes.view(torch.uint8)), dict(codes=codes.view(torch.int8)),
               dict(codes=codes[:, :50]), dict(scales=scales[:, :50]), dict(scales=scales.int()),
               dict(scales=scales.cpu()), dict(lens=-lens)]
    ragged = [dict(cu=cu[:3]), dict(cu=cu.long())]
    for change in changes + ragged + [
            first3, dict(first3, q=None), dict(q=None), dict(q=None, cos=None, sin=None),
            dict(cos=None), dict(cos=cos[:5]), dict(cos=cos.double()), dict(sin=sin.cpu()),
            dict(q=q[:5]), dict(q=q.float()), dict(k=k[:5]), dict(k=k.double()),
            dict(v=v.transpose(0, 1)), dict(k=k.float(), v=v.float(), q=q.float()),
            dict(k=k[:0], v=v[:0], q=q[:0], cos=cos[:0], sin=sin[:0]), dict(cu=None),
            dict(k=qkv[:, 1:1 + hkv * d].view(n, hkv, d))]:
        _same(*_both(monkeypatch, lambda: append(**change)))
    for change in changes + ragged + [dict(n=0), dict(n=-1), dict(n=20), dict(n=9),
                                      dict(dtype=torch.float32), dict(n=14.0)]:
        if change.get("n") == 9:
            continue                  # num_tokens below cu_seqlens' end is not a call
        _same(*_both(monkeypatch, lambda: read(**change)))
    for change in changes + ragged + [
            dict(q=q[:5]), dict(q=q.double()), dict(q=q[..., :32]), dict(q=q[:0]), dict(scale=1),
            dict(most=0), dict(most=-1), dict(h=3), dict(d=128), dict(bound=None), dict(bound=5),
            dict(most=torch.tensor(9))]:
        if change.get("q") is not None and change["q"].shape[0] == 5 or "bound" in change and \
                change["bound"] == 5:
            continue                  # a bound below the call's sizes is not a call either
        _same(*_both(monkeypatch, lambda: chunk(**change)))
    for change in changes + [dict(q=q[:2]), dict(q=q[:3].transpose(0, 1)), dict(h=3),
                             dict(scale=-1.0)]:
        _same(*_both(monkeypatch, lambda: decode(**change)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_verify(native, monkeypatch, dtype):  # noqa: F811
    gen = torch.Generator().manual_seed(2)
    vocab = 1003
    logits = torch.randn(9, vocab, generator=gen).to(dtype).to(DEV)
    ids = torch.randint(0, vocab, (9,), generator=gen).to(DEV)
    cu = torch.tensor([0, 4, 5, 9], dtype=torch.int32, device=DEV)
    u = torch.rand(9, generator=gen).to(DEV)
    t = torch.tensor([0.7, 0.0, 1.0], device=DEV)
    probs = torch.softmax(torch.randn(6, vocab, generator=gen), -1).to(DEV)

    def verify(logits=logits, ids=ids, cu=cu, u=u, t=t, probs=probs):
        return ops.verify_drafts(logits, ids, cu, u, temperature=t, draft_probs=probs)

    assert native.verify_drafts(logits, ids, cu, u, t, probs) is not None
    wide = torch.randn(9, 2000, generator=gen).to(dtype).to(DEV)
    for change in [
            dict(), dict(t=None), dict(probs=None), dict(t=None, probs=None),
            dict(logits=wide[:, 7:7 + vocab]), dict(logits=logits.t()), dict(logits=logits[:8]),
            dict(logits=logits.cpu()), dict(logits=logits.double()), dict(ids=ids.int()),
            dict(ids=ids.float()), dict(ids=ids[:8]), dict(cu=cu.long()), dict(u=u[:8]),
            dict(u=u.double()), dict(t=t[:2]), dict(t=t.double()), dict(t=t.cpu()),
            dict(probs=probs[:5]), dict(probs=probs.double()), dict(probs=probs.t()),
            dict(logits=logits[:, :1], probs=probs[:, :1]),
            dict(logits=logits[:3], ids=ids[:3], u=u[:3], cu=torch.arange(
                4, dtype=torch.int32, device=DEV), probs=probs[:0]),
            dict(logits=logits[:0], ids=ids[:0], u=u[:0], cu=cu[:1], t=t[:0], probs=probs[:0]),
            dict(logits=wide[:, :0], probs=probs[:, :0])]:
        _same(*_both(monkeypatch, lambda: verify(**change)))
