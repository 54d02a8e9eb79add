"""The workspace of the 8-bit pool's attention for long chunks: bounded whatever the batch, and out
of the memory that the runner's pool is sized for (CPU)."""
import pytest
import torch

from needle_amd import _lib, ops
from needle_amd.model.config import ModelConfig
from needle_amd.model.runner import ModelRunner

GIB = 1 << 30
SPLIT = 96 << 20       # the prefill's partial sums: two per workgroup, of eight waves


def _bytes(seqs, chunk, keys, h=32, hkv=8, d=128, bs=16):
    return ops.fp8_attention_workspace_bytes(seqs, seqs * chunk, chunk, keys, h, hkv, d, bs)


@pytest.mark.parametrize("seqs", [1, 2, 63, 64, 65, 300, 70000])
@pytest.mark.parametrize("keys", [1000, 4096, 33000])
def test_the_pool_is_bounded(seqs, keys):
    each = -(-keys // 16) * 16 * 8 * 128 * 4
    got = _bytes(seqs, 700, keys)
    groups = -(-seqs // (4 * GIB // each))
    held = -(-seqs // groups)                   # even groups
    assert held * each <= got <= held * each + held * (keys // 16 + 8) * 4 + SPLIT
    assert got <= 4 * GIB + SPLIT + (8 << 20) and _lib.NDL_FP8_UNPACK_BYTES == 4 * GIB


def test_one_sequence_may_take_more():
    each = 2000000 * 8 * 128 * 4
    assert each <= _bytes(5, 200, 2000000) <= each + SPLIT + (1 << 20)
    # past 16 GiB its chunk stays row blocks
    assert _bytes(1, 200, 5000000) < GIB


def test_a_wide_table_costs_no_more():
    """One long prompt among many short ones: the rectangle would be 16 GiB."""
    rect = 64 * 65536 * 8 * 128 * 4
    assert _bytes(64, 8192, 65536) < rect // 3


@pytest.mark.parametrize("kind", ["fp8", "auto"])
def test_the_runner_leaves_room_for_it(monkeypatch, kind):
    cfg = dict(hidden_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
               intermediate_size=64, vocab_size=50, max_position_embeddings=8192)
    r = ModelRunner(ModelConfig(**cfg), device="cpu", kv_cache_dtype=kind)
    r.device = torch.device("cuda:0")
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda dev: (20 * GIB, 30 * GIB))
    blocks, _ = r.profile_memory(0.9)
    used = blocks * r.bytes_per_block()
    room = int(20 * GIB * 0.9) - used
    if kind == "auto":
        assert room < r.bytes_per_block()
    else:
        for seqs, chunk in ((1, 8192), (9, 8192), (64, 4000), (512, 900), (2000, 300)):
            assert ops.fp8_attention_workspace_bytes(seqs, seqs * chunk, chunk, chunk, 4, 2, 128,
                                                     16) <= room + SPLIT
        assert room < 4 * GIB + SPLIT + (8 << 20)
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda dev: (GIB // 2, 30 * GIB))
    assert r.profile_memory(0.9)[0] >= 1
