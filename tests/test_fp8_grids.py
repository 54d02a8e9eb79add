"""The 8-bit pool's entry points refuse what one launch cannot hold: HIP counts a grid's threads in 32
bits and launches the rest of a larger one without an error (CPU; nothing is launched)."""
import pytest

from needle_amd import _lib

P = 1 << 20      # an aligned stand-in address that is never dereferenced


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


# (head_dim, kv heads): a wave's share of a launch is 2 rounds of 64 items in the append, 512 items in
# the read
@pytest.mark.parametrize("d,hkv,tokens", [(64, 1, 4 << 24), (128, 8, 4 << 24), (128, 32, 1 << 24)])
def test_append(lib, d, hkv, tokens):
    assert lib.ndl_kv_append_fp8(P, P, 1 << 20, hkv, 16, d, 0, P, hkv * d, P, hkv * d, None, None, 0,
                                 0, None, None, 0, P, 4, 4, P, P, 1, tokens, None) == -1


@pytest.mark.parametrize("d,hkv,tokens", [(64, 1, (4 << 24) * 32), (128, 8, (4 << 24) * 2)])
def test_read(lib, d, hkv, tokens):
    assert lib.ndl_kv_read_fp8(P, P, P, P, 1 << 20, hkv, 16, d, 0, P, 4, 4, P, P, 1, tokens,
                               None) == -1


@pytest.mark.parametrize("h,hkv,seqs", [(1, 1, 1 << 24), (32, 8, 1 << 21)])
def test_decode(lib, h, hkv, seqs):
    assert lib.ndl_fp8_attention(P, P, h * 64, P, P, 1 << 10, P, 4, 4, None, P, seqs, seqs, 1, 64, h,
                                 hkv, 64, 16, 0, 0.1, None, 0, None) == -1
    assert lib.ndl_fp8_decode_append(P, P, h * 64, P, hkv * 64, P, hkv * 64, None, None, 0, P, P,
                                     1 << 10, P, 4, 4, P, seqs, h, hkv, 64, 16, 0, 0.1, None, 0,
                                     None) == -1


def test_long_chunks(lib):
    """One chunk of 2^28 tokens of 8 kv heads: neither way holds it."""
    t, keys = 1 << 28, 1 << 28
    assert lib.ndl_fp8_attention(P, P, 8 * 64, P, P, 1 << 10, P, keys // 16, keys // 16, P, P, 1, t,
                                 t, keys, 8, 8, 64, 16, 0, 0.1, P, 1 << 40, None) == -1
