"""The account of memory holds the scratch of shared beginnings for steps that run kernel by kernel, too."""
import pytest

import cache8_tools as c8
from helpers import TINY
from holon_b200.engine import build
from holon_b200.weights import RandomSource


class Table(c8.RefKernels8):
    def read_back_scratch(self, tokens, rows, longest, kv_heads, head_dim):
        return 1000 * rows

    def shared_scratch(self, rows, heads, kv_heads, head_dim, page_size):
        return rows * heads * page_size


@pytest.mark.parametrize("cache_dtype", ["auto", "fp8"])
@pytest.mark.parametrize("shared", [True, False])
def test_scratch_of_steps(cache_dtype, shared):
    config = TINY["b"][0]
    b = build(RandomSource(config, seed=1), dtype="bfloat16", device="cpu", kernels=Table(), page_size=32, max_seqs=4, max_model_len=512,
              max_step_tokens=512, pages=100, prefix_cache=True, cache_dtype=cache_dtype, shared_prefix=shared)
    back, together = 1000 * 5 * (cache_dtype == "fp8"), 4 * 5 * config["num_attention_heads"] * 32 * shared
    assert b.model.context_scratch(100, 5, 500) == back + together
    assert b.model.graph_scratch(5, 0, 500, 32) == together


def test_one_portion_of_scratch_at_a_time(monkeypatch):
    """Rows of several tokens that are read back in turns hold the scratch of one turn: that is what the account has."""
    import weakref

    import torch

    from test_cache8_cpu import attend
    empty, made, most = torch.empty, [], [0]

    def watched(*a, **kw):
        t = empty(*a, **kw)
        if t.dim() == 5:
            made.append(weakref.ref(t))
            most[0] = max(most[0], sum(r() is not None for r in made))
        return t

    monkeypatch.setattr(torch, "empty", watched)
    attend([100, 200, 300], [9, 50, 300], dim=64, READ_BACK_TOKENS=400)
    assert len(made) == 3 and most[0] == 1
