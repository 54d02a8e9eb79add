"""kv_cache_dtype of the runner: its refusals and the bytes of a block (CPU)."""
import pytest

from needle_amd import ops
from needle_amd.model.config import ModelConfig
from needle_amd.model.runner import ModelRunner

CFG = dict(hidden_size=128, num_hidden_layers=3, num_attention_heads=2, num_key_value_heads=1,
           intermediate_size=64, vocab_size=50, max_position_embeddings=64)


def _runner(dtype="bfloat16", kind="fp8", **cfg):
    return ModelRunner(ModelConfig(**{**CFG, **cfg}), dtype=dtype, device="cpu",
                       kv_cache_dtype=kind)


def test_refusals():
    with pytest.raises(ValueError, match="'auto'"):
        _runner(kind="int8")
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        _runner(dtype="float32")
    with pytest.raises(ValueError, match="head_dim 64 and 128"):
        _runner(hidden_size=64)


def test_a_blocks_bytes_and_the_pool():
    r = _runner()
    assert r.bytes_per_block() == 3 * 2 * 16 * 65
    assert _runner(kind="auto").bytes_per_block() == 3 * 2 * 16 * 64 * 2
    assert _runner(kind="auto", dtype="float32").bytes_per_block() == 3 * 2 * 16 * 64 * 4
    r.init_kv_cache(7)
    assert len(r.kv_caches) == 3 and not r.cpu_kv_caches
    assert sum(x.nbytes for pool in r.kv_caches for x in pool) == 7 * r.bytes_per_block()
    assert isinstance(r.kv_caches[0], ops.Fp8KVCache) and r.kv_caches[0].shape[1] == 7
