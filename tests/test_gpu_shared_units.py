"""The join of shared beginnings that are cut into as many units as there may be, in every form of the kernel that weighs them."""
import pytest
import torch

import cache8_tools as c8
from test_gpu_shared_prefix import K, case, run, within  # noqa: F401  (K: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("pages", [480, 492, 592])                    # 30,720 tokens: 240 units of two blocks of keys; 31,488 and 37,888: fewer, larger ones
def test_the_most_units_a_tile(K, pages, fp8, monkeypatch):           # noqa: F811
    """One kv head of 64 with eight query heads off tcgen05: eight rows are one tile, and two CTAs an SM would cut it into 296 units."""
    q, kv, table, rows, shared = case([(pages, [1, 70, 33, 500, 64, 2, 129, 8])], [1 + 31 * i % 400 for i in range(470)], 8, 1, 64, 64, fp8)
    assert K._prefix_plan(8, 64, 64)[0] == 2 * K.sms and K._prefix_plan(8, 64, 64)[2] == 8
    sinks = torch.linspace(-2, 2, 8)
    want, mass = c8.attend(q, kv, table, rows, 0.125, 0, sinks)
    assert K._row_splits(int(fp8), rows.n_decode, 8, 1, 64, shared.longest_own, 0, True)[1] == 1       # the form for few keys
    within(run(K, q, kv, table, rows, 0.125, sinks, shared), want, mass)
    for form in ((1, 0, 0), (1, 1, 1), (4, 0, 0), (16, 0, 1)):
        monkeypatch.setattr(K, "_row_splits", lambda *a: form, raising=False)
        got = run(K, q, kv, table, rows, 0.125, sinks, shared)
        within(got, want, mass)
        assert torch.equal(got, run(K, q, kv, table, rows, 0.125, sinks, shared))


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("left", [float("nan"), 0.0, -1.0, 1e-40])    # as numbers of four bytes: large ones, zeros, negative ones, 71,362
def test_partial_results_that_were_not_left(K, fp8, left, monkeypatch):   # noqa: F811
    """A launch for the shared keys that gave up leaves rows without an entry: the join reports that and reads nothing by what it finds there."""
    q, kv, table, rows, shared = case([(16, [1, 130, 64, 3])], [60, 7], 8, 2, 128, 64, fp8)
    clean = run(K, q, kv, table, rows, 0.125, None, shared)
    call, empty = type(K)._call, torch.empty
    monkeypatch.setattr(K, "_call", lambda name, *a: None if name == "hb_attention_prefix" else call(K, name, *a), raising=False)
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: empty(*a, **kw).fill_(left))
    assert K.status() == 0
    try:
        got = run(K, q, kv, table, rows, 0.125, None, shared)
        torch.cuda.synchronize()
        assert K.status() >> 28 == 12
    finally:
        with torch.inference_mode():                                 # (the table may have been made in that mode)
            asked = K.tcgen05_status(), K.tcgen05_status()           # the file's own word, which asking clears
    assert asked[0] >> 28 == 12 and asked[1] == 0
    alone = [b for b in range(6) if int(shared.skip[b]) == 0]
    assert len(alone) == 2 and all(torch.equal(got[b], clean[b]) for b in alone)
    monkeypatch.undo()
    assert torch.equal(run(K, q, kv, table, rows, 0.125, None, shared), clean) and K.status() == 0


def test_as_many_ctas_as_an_sm_holds(K):                              # noqa: F811
    """Off tcgen05 two CTAs of the kernel for shared keys fit an SM, above heads of 128 one (160 KB of tiles)."""
    assert [K._prefix_plan(4, dim, 64)[0] // K.sms for dim in (64, 80, 144, 192, 256)] == [2, 2, 1, 1, 1]
    assert K._prefix_plan(4, 128, 16)[0] == 2 * K.sms and K._prefix_plan(4, 128, 64)[0] == K.sms
