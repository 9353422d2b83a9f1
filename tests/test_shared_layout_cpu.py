"""Steps whose small arrays lie at other places in the upload are never replays of one graph, whatever the mixers answer."""
import numpy as np

import cache8_tools as c8
from helpers import TINY
from holon_b200.engine import StepEntry, build
from holon_b200.parts.attention import GQA
from holon_b200.weights import RandomSource


def test_a_mixer_that_does_not_speak_of_sharing(monkeypatch):
    """A mixer of a user's own over `PagedKV` pages need not know of shared beginnings: its plan is the same with and without them."""
    monkeypatch.setattr(GQA, "capture_plan", lambda self, step, longest: "mine")
    b = build(RandomSource(TINY["b"][0], seed=1), dtype="bfloat16", device="cpu", kernels=c8.RefKernels8(), page_size=16, max_seqs=4, max_model_len=512,
              max_step_tokens=512, pages=100, prefix_cache=True, shared_prefix=True)
    cache, runner = b.cache, b.runner
    same, plans, places = list(range(1, 301)), [], []
    for tokens in ([same, [5] * 300, [6] * 300], [same, same, [7] * 300]):
        slots = []
        for ids in tokens:
            slot = cache.admit(ids)
            start = int(cache.computed[slot])
            assert cache.reserve(slot, len(ids) + 1)
            runner.step([StepEntry(slot, ids[start:], start, [])])
            cache.publish(slot, ids)
            slots.append(slot)
        step = runner.context([StepEntry(s, [9], 300, [0]) for s in slots], pad_rows=1, extra={"top_k": np.arange(4, dtype=np.int32)})
        assert step.extra["top_k"].tolist() == [0, 1, 2, 3]
        plans.append(runner.plan(step, 512))
        places.append(step.extra["top_k"].storage_offset())
        for slot in slots:
            cache.release(slot)
    assert places[0] != places[1] and plans[0] != plans[1]
