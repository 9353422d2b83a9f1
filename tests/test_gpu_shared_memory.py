"""Without graphs the account of memory holds what rows that share beginnings leave for one another."""
import pytest
import torch

from holon_b200.engine import Engine, EngineConfig
from holon_b200.weights import RandomSource
from test_gpu_cache8_engine import WIDE

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache_dtype", ["auto", "fp8"])
def test_memory_without_graphs(cache_dtype):
    def account(**kw):
        e = Engine(EngineConfig(model="", page_size=64, max_seqs=64, max_model_len=1024, max_step_tokens=512, memory_fraction=0.05, cuda_graphs=False,
                                cache_dtype=cache_dtype, **kw), source=RandomSource(WIDE, seed=5, device="cuda:0", dtype=torch.bfloat16))
        k, m = e.built.ctx.kernels, e.built.memory
        e.close()
        return k.shared_scratch(64, 8, 2, 128, 64), m
    account()                                                         # (what the matrix library keeps from its first call on is not counted twice)
    (scratch, apart), (_, together) = account(), account(shared_prefix=True)
    assert apart.graphs == together.graphs == 0 and scratch > 0
    # the measured steps are alike, up to the 2 MB in which the allocator takes memory from the device
    assert together.activations >= apart.activations + 4 * scratch - (2 << 20)
