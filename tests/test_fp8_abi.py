"""What the 8-bit pool's and the draft verification's entry points refuse before any launch, and
their oracle against known values (CPU)."""
import math

import pytest
import torch

from needle_amd import _lib
from oracle import fp8_ref

P = 1 << 20      # an aligned stand-in address that is never dereferenced


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_append_and_read_refusals(lib):
    def append(codes=P, scales=P, nb=4, hkv=2, bs=16, d=64, dtype=0, k=P, ks=128, v=P, vs=128,
               qo=None, q=None, qs=0, h=0, cos=None, sin=None, cs=0, table=P, stride=4, w=4,
               cu=None, ctx=P, n=3, t=3):
        return lib.ndl_kv_append_fp8(codes, scales, nb, hkv, bs, d, dtype, k, ks, v, vs, qo, q,
                                     qs, h, cos, sin, cs, table, stride, w, cu, ctx, n, t, None)
    for bad in (dict(dtype=2), dict(dtype=9), dict(d=96), dict(d=32), dict(bs=8), dict(bs=24),
                dict(bs=2048)):
        assert append(**bad) == -2, bad
    for bad in (dict(codes=None), dict(scales=None), dict(k=None), dict(table=None),
                dict(ctx=None), dict(t=2), dict(t=-1), dict(ks=120), dict(ks=132), dict(vs=4),
                dict(k=P + 8), dict(codes=P + 1), dict(nb=0), dict(w=0), dict(stride=3),
                dict(cos=P), dict(q=P, qo=P, qs=256, h=4), dict(cos=P, sin=P, cs=60),
                dict(q=P, cos=P, sin=P, cs=64), dict(q=P, qo=P, qs=64, h=4, cos=P, sin=P, cs=64)):
        assert append(**bad) == -1, bad
    assert append(t=0, n=0) == 0

    def read(ko=P, vo=P, codes=P, scales=P, nb=4, hkv=2, bs=16, d=64, dtype=0, table=P, stride=4,
             w=4, first=P, cu=P, n=3, t=3):
        return lib.ndl_kv_read_fp8(ko, vo, codes, scales, nb, hkv, bs, d, dtype, table, stride,
                                   w, first, cu, n, t, None)
    for bad in (dict(dtype=2), dict(d=256), dict(bs=20)):
        assert read(**bad) == -2, bad
    for bad in (dict(ko=None), dict(vo=P + 8), dict(codes=None), dict(first=None), dict(cu=None),
                dict(hkv=0), dict(t=-3)):
        assert read(**bad) == -1, bad
    assert read(t=0) == 0 and read(n=0) == 0


def test_attention_refusals(lib):
    def attend(out=P, q=P, qs=512, codes=P, scales=P, nb=4, table=P, stride=500, w=500, cu=P,
               ctx=P, n=3, t=9, most=3, keys=8000, h=8, hkv=2, d=64, bs=16, dtype=0, ws=P,
               size=0):
        return lib.ndl_fp8_attention(out, q, qs, codes, scales, nb, table, stride, w, cu, ctx, n,
                                     t, most, keys, h, hkv, d, bs, dtype, 0.1, ws, size, None)
    for bad in (dict(dtype=2), dict(d=96), dict(bs=12), dict(h=9), dict(h=34), dict(hkv=0),
                dict(nb=1 << 27), dict(w=1 << 30, stride=1 << 30)):
        assert attend(**bad) == -2, bad
    for bad in (dict(out=None), dict(q=None), dict(codes=None), dict(scales=None),
                dict(scales=P + 2), dict(table=None), dict(ctx=None), dict(qs=500), dict(qs=516),
                dict(q=P + 8), dict(most=0), dict(keys=0), dict(cu=None), dict(cu=None, t=3),
                dict(stride=3), dict(nb=0)):
        assert attend(**bad) == -1, bad
    need = lib.ndl_fp8_attention_workspace_bytes(3, 9, 3, 8000, 8, 2, 64, 16)
    assert need > 0
    assert attend(size=need - 1) == -3 and attend(ws=None, size=need) == -3
    assert attend(ws=P + 16, size=need) == -3
    assert attend(n=0) == 0 and attend(t=0) == 0
    # short tables need no workspace; nothing is sized for what is refused
    assert lib.ndl_fp8_attention_workspace_bytes(3, 9, 3, 64, 8, 2, 64, 16) == 0
    for bad in ((3, 9, 3, 8000, 9, 2, 64, 16), (0, 9, 3, 8000, 8, 2, 64, 16),
                (3, 9, 0, 8000, 8, 2, 64, 16), (3, 9, 3, 8000, 8, 2, 80, 16),
                (3, 9, 3, 8000, 8, 2, 64, 17)):
        assert lib.ndl_fp8_attention_workspace_bytes(*bad) == 0


def test_decode_append_refusals(lib):
    def step(out=P, q=P, qs=512, k=P, ks=128, v=P, vs=128, cos=P, sin=P, cs=64, codes=P, scales=P,
             nb=4, table=P, stride=500, w=500, ctx=P, n=3, h=8, hkv=2, d=64, bs=16, dtype=0, ws=P,
             size=0):
        return lib.ndl_fp8_decode_append(out, q, qs, k, ks, v, vs, cos, sin, cs, codes, scales, nb,
                                         table, stride, w, ctx, n, h, hkv, d, bs, dtype, 0.1, ws,
                                         size, None)
    for bad in (dict(dtype=2), dict(d=96, qs=768, ks=192, vs=192, cs=96), dict(bs=12), dict(h=9),
                dict(h=34), dict(nb=1 << 27), dict(w=1 << 30, stride=1 << 30)):
        assert step(**{**dict(qs=4096), **bad}) == -2, bad
    for bad in (dict(k=None), dict(v=None), dict(ks=120), dict(vs=132), dict(k=P + 8),
                dict(v=P + 2), dict(cos=None), dict(sin=None), dict(cs=60), dict(cs=68),
                dict(cos=P + 4), dict(out=None), dict(q=None), dict(ctx=None), dict(table=None),
                dict(codes=P + 8), dict(qs=500), dict(n=-1), dict(nb=0), dict(w=0),
                dict(stride=499)):
        assert step(**bad) == -1, bad
    need = lib.ndl_fp8_attention_workspace_bytes(3, 3, 1, 8000, 8, 2, 64, 16)
    assert need > 0
    assert step(size=need - 1) == -3 and step(ws=None, size=need) == -3
    assert step(n=0) == 0


def test_verify_refusals(lib):
    def verify(tokens=P, acc=P, logits=P, stride=100, dtype=0, ids=P, cu=P, u=P, temp=None,
               probs=None, ds=0, rows=4, n=2, vocab=100, ws=P, size=0):
        return lib.ndl_verify_drafts(tokens, acc, logits, stride, dtype, ids, 1, cu, u, temp,
                                     probs, ds, rows - n, rows, n, vocab, ws, size, None)
    assert verify(dtype=7) == -2 and verify(rows=70000) == -2
    for bad in (dict(tokens=None), dict(acc=None), dict(logits=None), dict(ids=None),
                dict(cu=None), dict(u=None), dict(stride=99), dict(probs=P, ds=99),
                dict(logits=P + 1), dict(dtype=2, logits=P + 2), dict(probs=P + 2, ds=100),
                dict(rows=0), dict(vocab=0)):
        assert verify(**bad) == -1, bad
    need = lib.ndl_verify_drafts_workspace_bytes(4, 2, 100)
    assert need > 0 and verify(size=need - 1) == -3 and verify(ws=P + 4, size=need) == -3
    assert verify(n=0) == 0
    assert lib.ndl_verify_drafts_workspace_bytes(0, 2, 100) == 0


def test_oracle_quantises_to_known_codes():
    codes, byte = fp8_ref.quantise_row([448.0, 1.0, -0.4375, 0.0, 2.0 ** -9, 2.0 ** -10,
                                        3 * 2.0 ** -10, math.nan, math.inf])
    assert byte == 127
    # ties go to the even code: 2^-10 to 0, 3 * 2^-10 to 2 steps of 2^-9
    assert codes == [0x7E, 0x38, 0xAE, 0x00, 0x01, 0x00, 0x02, 0x7F, 0x7F]
    assert fp8_ref.quantise_row([448.5])[1] == 128 and fp8_ref.quantise_row([0.0])[1] == 1
    table = fp8_ref.code_values()
    got = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(table.isnan(), got.isnan())
    assert torch.equal(table.nan_to_num(0.0), got.nan_to_num(0.0))


def test_oracle_verifies_a_known_case():
    p = torch.tensor([[0.5, 0.25, 0.25], [0.1, 0.8, 0.1], [0.2, 0.2, 0.6]])
    q = torch.tensor([[0.25, 0.5, 0.25], [0.9, 0.05, 0.05]])
    cu, ids = [0, 3], [9, 0, 0]
    # the first draft (p 0.5, q 0.25) always holds; the second while u * 0.9 < 0.1
    assert fp8_ref.verify(p.log(), ids, cu, [0.99, 0.1, 0.5], None, q) == ([0, 0, 2], [2])
    # rejected: max(p - q, 0) = (0, 0.75, 0.05)
    assert fp8_ref.verify(p.log(), ids, cu, [0.99, 0.2, 0.9], None, q) == ([0, 1, -1], [1])
    assert fp8_ref.verify(p.log(), ids, cu, [0.99, 0.2, 0.95], None, q) == ([0, 2, -1], [1])
    assert fp8_ref.verify(p.log(), [9, 0, 1], cu, [0.6, 0.2, 0.45], None, None) == ([1, -1, -1], [0])
    assert fp8_ref.verify(p.log(), [9, 0, 1], cu, [0.4, 0.2, 0.2], [0.0], None) == ([0, 1, 2], [2])
