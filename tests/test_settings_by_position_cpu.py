"""Settings by position: a field that is added comes behind those that were there."""
import dataclasses

from holon_b200.config import EngineConfig


def test_settings_by_position():
    names = ["model", "device", "dtype", "page_size", "max_seqs", "max_model_len", "max_step_tokens", "chunk_with_decode", "prefix_cache", "memory_fraction",
             "state_memory", "overlap", "cuda_graphs", "seed"]
    assert [f.name for f in dataclasses.fields(EngineConfig)][:len(names)] == names
    values = ["x", "cuda:0", "bfloat16", 32, 3, 512, 256, 8, True, 0.5, 1 << 20, False, False, 7]
    config = EngineConfig(*values)
    assert [getattr(config, name) for name in names] == values and (config.cache_dtype, config.shared_prefix) == ("auto", False)
