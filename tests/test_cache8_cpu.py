"""The 8-bit cache and shared beginnings on the host: which rows make a group, what the settings refuse, the pools' sizes, and the
engine on the plain kernel table."""
from __future__ import annotations

import contextlib
import random
import types

import numpy as np
import pytest
import torch

import cache8_tools as c8
from helpers import TINY, make_folder, random_prompt
from holon_b200.cache import CacheManager
from holon_b200.engine import Engine, EngineConfig, SamplingParams, StepEntry, build
from holon_b200.engine.batch import SharedPrefix
from holon_b200.kernels.cuda import CudaKernels, KernelError
from holon_b200.parts import CacheEntry, PagedKV
from holon_b200.weights import RandomSource, SafetensorsSource


# ---------------------------------------------------------------- groups
def found(held, shared, page=16, pads=0):
    table, count = c8.paged(held, page, len(held), 0, shared)
    table = np.concatenate([table.numpy(), np.full((pads, table.shape[1]), count - 1, dtype=np.int32)])
    slots = np.arange(len(held) + pads)[::-1] + 3
    got = SharedPrefix.find(table, np.array(held + [1] * pads, dtype=np.int32), page, slots)
    if got is None:
        return None
    n = len(held) + pads
    assert got["skip"].shape == got["members"].shape == (n,) and got["groups"].shape == (4 * (n // 2),)
    assert all(a.dtype == np.int32 for a in (got["skip"], got["members"], got["groups"]))
    out, seen = [], set()
    for start, count_, tokens, slot in got["groups"].reshape(-1, 4).tolist():
        if count_:
            rows = got["members"][start:start + count_].tolist()
            assert slot in slots[rows]
            assert count_ > 1 and tokens > 0 and tokens % page == 0 and not seen & set(rows)
            assert all(got["skip"][r] == tokens < held[r] for r in rows)
            assert (table[rows, :tokens // page] == table[rows[0], :tokens // page]).all()
            seen |= set(rows)
            out.append((sorted(rows), tokens))
    assert all(got["skip"][r] == 0 for r in range(n) if r not in seen)
    assert got["saved"] == sum((len(rows) - 1) * tokens for rows, tokens in out)
    assert got["longest_own"] == max(h - int(s) for h, s in zip(held + [1] * pads, got["skip"]))
    return sorted(out)


def test_groups_of_rows():
    assert found([500, 600, 40], []) is None
    assert found([500, 600, 700], [([0, 2], 20)]) == [([0, 2], 320)]
    assert found([500, 600, 700, 800], [([0, 2], 20), ([1, 3], 30)], pads=3) == [([0, 2], 320), ([1, 3], 480)]
    assert found([100, 100], [([0, 1], 6)]) is None                                 # too little is saved
    assert found([100] * 4, [([0, 1, 2, 3], 6)]) == [([0, 1, 2, 3], 96)]
    assert found([320, 320, 321], [([0, 1, 2], 20)]) == [([0, 1, 2], 304)]          # a row's last token stays its own
    assert found([16], []) is None and found([1, 1, 1], [], pads=2) is None


def test_rows_that_share_more_with_some():
    table, _ = c8.paged([1000] * 6, 16, 6, 0, [(list(range(6)), 4)])
    table = table.numpy()
    table[1, 4:50], table[3, 4:50] = table[0, 4:50], table[2, 4:50]                 # 0 with 1 and 2 with 3 share 46 pages more
    got = SharedPrefix.find(table, np.full(6, 1000, dtype=np.int32), 16, np.arange(6))
    assert sorted(got["groups"].reshape(-1, 4)[:, 1:3].tolist()) == [[0, 0], [2, 800], [2, 800]]
    table[1, 6:], table[3, 6:] = -1, -2                                             # two pages more are not worth a cut
    got = SharedPrefix.find(table, np.full(6, 1000, dtype=np.int32), 16, np.arange(6))
    assert got["groups"].tolist() == [0, 6, 64, 0] + [0] * 8


def test_random_tables():
    rng = random.Random(3)
    for _ in range(200):
        n, page = rng.randint(1, 20), rng.choice((4, 16, 64))
        order, shared = rng.sample(range(n), n), []
        held = [rng.randint(1, 40 * page) for _ in range(n)]
        while len(order) > 1 and rng.random() < 0.7:
            rows = [order.pop() for _ in range(rng.randint(2, len(order)))]
            pages = rng.randint(0, min((held[r] - 1) // page for r in rows))
            if pages:
                shared.append((rows, pages))
        got = found(held, shared, page, rng.randint(0, 3))
        worth = sorted((sorted(rows), pages * page) for rows, pages in shared if pages * page * (len(rows) - 1) >= SharedPrefix.LEAST)
        assert (got or []) == worth


# ---------------------------------------------------------------- settings and pools
def test_settings_refuse():
    EngineConfig(model="x", cache_dtype="fp8", shared_prefix=True)
    for bad in (dict(cache_dtype="fp16"), dict(cache_dtype="fp8", dtype="float32"), dict(cache_dtype="fp8", page_size=24),
                dict(shared_prefix=True, dtype="float32"), dict(shared_prefix=True, prefix_cache=False)):
        with pytest.raises(ValueError):
            EngineConfig(model="x", **bad)


def built(config, **kw):
    args = dict(dtype="bfloat16", device="cpu", kernels=c8.RefKernels8(), page_size=16, max_seqs=8, max_model_len=256, max_step_tokens=128, pages=64,
                cache_dtype="fp8")
    args.update(kw)
    return build(RandomSource(config, seed=1), **args)


def test_build_refuses(tmp_path):
    config, _ = TINY["b"]
    built(config)
    for bad in (dict(cache_dtype="int8"), dict(dtype="float32"), dict(page_size=8), dict(cache_dtype="auto", shared_prefix=True, dtype="float32")):
        with pytest.raises(ValueError):
            built(config, **bad)
    with pytest.raises(ValueError, match="multiples of 16"):
        built(dict(config, head_dim=24))
    from rulorax_tools import CONFIGS
    with pytest.raises(ValueError, match="has none"):
        built(next(iter(CONFIGS.values())))


def test_pools_of_bytes():
    wide, narrow = PagedKV(2, 32, 0, False), PagedKV(2, 32, 0, True)
    assert narrow.page_shape(16) == (2, 2, 16, 33) and narrow.dtype == torch.uint8 and wide.dtype is None
    entries = [CacheEntry(0, 0, wide, ()), CacheEntry(1, 1, narrow, ()), CacheEntry(2, 2, narrow, ())]
    cache = CacheManager(entries, 16, 2, 64, torch.bfloat16, "cpu", state_memory=40 * (2 * 2 * 16 * (64 + 2 * 33)))
    assert [g.kv.dtype for g in cache.groups] == [torch.bfloat16, torch.uint8] and cache.pages == 39
    assert cache.kv_of_entry[2].shape == (40, 2, 2, 16, 33)
    assert cache.bytes == 40 * 2 * 2 * 16 * (64 + 2 * 33)


# ---------------------------------------------------------------- the engine
def step_through(b, ids, cut, want_all=True):
    slot, at, out = b.cache.admit(), 0, []
    for n in cut:
        assert b.cache.reserve(slot, at + n)
        out.append(b.runner.step([StepEntry(slot, ids[at:at + n], at, range(n))]))
        at += n
    return slot, torch.cat(out)


@pytest.mark.parametrize("name", ["b", "c"])
def test_the_step_function_on_codes(tmp_path, name):
    folder = make_folder(tmp_path, name)
    config, _ = TINY[name]
    ids = random_prompt(config["vocab_size"], 70, 5)
    make = lambda **kw: build(SafetensorsSource(folder), **(dict(dtype="bfloat16", device="cpu", kernels=c8.RefKernels8(), page_size=16, max_seqs=4,   # noqa: E731
                                                                 max_model_len=128, max_step_tokens=128, pages=40) | kw))
    eight, wide = make(cache_dtype="fp8"), make()
    s8, whole = step_through(eight, ids, [70])
    s16, _ = step_through(wide, ids, [70])
    # the first layer's keys and values come from the same inputs: half a step of a code (2^-4) and of bfloat16 (2^-8; the normed key
    # is rounded once more before its rotation there) of a number, and for small ones half the least code's step, 2^-10 of a scale that is
    # at most 2^-7.8 of the row's largest
    pages8 = c8.decode(eight.cache.kv_of_entry[0])[torch.from_numpy(eight.cache.groups[0].table[s8, :5]).long()]
    pages16 = wide.cache.kv_of_entry[0][torch.from_numpy(wide.cache.groups[0].table[s16, :5]).long()].double()
    a, b = (p.transpose(0, 3).reshape(16, -1, p.shape[-1]) for p in (pages8, pages16))
    bound = (2.0 ** -4 + 2.0 ** -7) * b.abs() + (2.0 ** -17 + 2.0 ** -8) * b.abs().amax(-1, keepdim=True)
    assert bool(((a - b).abs() <= bound).all()) and not torch.equal(a, b)
    # the cut of a prompt changes the order of sums only: bfloat16 roundings of both, which may move one code in 32 by a step
    _, parts = step_through(eight, ids, [16, 1, 20, 1, 1, 31])
    assert torch.linalg.norm(parts - whole) <= 5e-2 * torch.linalg.norm(whole)


def test_generation_with_both(tmp_path):
    """Sequences of one prompt share its pages: each step's one-token rows are found and handed to attention; greedy siblings agree."""
    folder = make_folder(tmp_path, "c")
    calls = []

    class Watched(c8.RefKernels8):
        def paged_attention(self, out, q, kv, block_table, rows, scale, window, sinks=None, shared=None):
            calls.append(None if shared is None else (rows.n_decode, shared.rows, shared.groups[:3].tolist()))
            super().paged_attention(out, q, kv, block_table, rows, scale, window, sinks)

    class Dear(Watched):
        def shared_least(self, decl):
            return 5 * 144 + 1                                                       # (the siblings save 4 x 144)

    for option, table in ((True, Watched), (False, Watched), (True, Dear)):
        engine = Engine(EngineConfig(model=str(folder), device="cpu", cache_dtype="fp8", shared_prefix=option, page_size=16, max_seqs=6,
                                     max_model_len=256, max_step_tokens=256, state_memory=4 << 20), kernels=table())
        engine.add(random_prompt(384, 150, 7), SamplingParams(temperature=0.0, max_tokens=6, n=5, ignore_eos=True), rid="a")
        engine.add(random_prompt(384, 20, 8), SamplingParams(temperature=0.0, max_tokens=6, ignore_eos=True), rid="b")
        got: dict = {}
        while engine.has_work():
            for d in engine.step():
                got.setdefault((d.rid, d.index), []).extend(d.token_ids)
        engine.built.cache.check()
        assert len(got) == 6 and all(len(t) == 6 for t in got.values())
        assert len({tuple(got["a", i]) for i in range(1, 5)}) == 1
        hits = [c for c in calls if c is not None]
        assert bool(hits) == (option and table is Watched)
        assert not hits or (6, 6, [0, 5, 144]) in hits
        calls.clear()


# ---------------------------------------------------------------- the kernel table's decisions
class Noted(CudaKernels):
    def __init__(self):
        self.device, self.called, self._pending, self._splits, self.sms = torch.device("cpu"), [], [], {}, 148
        self.prefill_attention, self.prefill_tile, self.attention_bf16 = "tcgen05", None, "fast"
        self.lib = types.SimpleNamespace(hb_attention_prefix_plan=self.plan, hb_attention_rows_capacity=lambda kv8, few, dim, group, s: 3 if s == 1 else 400 // s)

    def plan(self, dim, page, group, part_rows, tile_rows):
        part_rows._obj.value, tile_rows._obj.value = 64, 64 // group
        return 2 if group <= 64 else 0

    def _check(self, *tensors):
        assert all(t is None or t.is_contiguous() for t in tensors)

    def _call(self, name, *args):
        self.called.append(name)


def attend(held, new, dim=128, heads=8, kvh=2, page=64, kv8=True, shared=None, **attr):
    k = Noted()
    for name, value in attr.items():
        setattr(k, name, value)
    rows = c8.rows_of(held, new)
    table, count = c8.paged(held, page, len(held))
    kv = torch.zeros(count, 2, kvh, page, dim + 1, dtype=torch.uint8) if kv8 else torch.zeros(count, 2, kvh, page, dim, dtype=torch.bfloat16)
    q = torch.zeros(rows.n_tokens, heads, dim, dtype=torch.bfloat16)
    k.paged_attention(torch.zeros_like(q), q, kv, table, rows, 0.1, 0, None, shared=shared)
    return k.called


def test_which_kernels_run():
    assert attend([100, 200], [1, 1]) == ["hb_attention_rows"]
    assert attend([100, 200], [1, 50]) == ["hb_attention_rows", "hb_kv_read_rows", "hb_attention_prefill_tcgen05"]
    assert attend([100, 200], [9, 50], prefill_attention="mma") == ["hb_kv_read_rows", "hb_attention_prefill_bf16"]
    assert attend([100, 200], [9, 50], dim=64) == ["hb_kv_read_rows", "hb_attention_prefill_bf16"]
    assert attend([100, 200, 300], [9, 50, 300], dim=64, READ_BACK_TOKENS=400) == ["hb_kv_read_rows", "hb_attention_prefill_bf16"] * 3
    shared = SharedPrefix(*(torch.zeros(n, dtype=torch.int32) for n in (2, 2, 4)), 2, 50)
    assert attend([300, 400], [1, 1], shared=shared) == ["hb_attention_prefix", "hb_attention_rows"]
    assert attend([300, 400], [1, 1], kv8=False, shared=shared) == ["hb_attention_prefix", "hb_attention_rows"]
    assert attend([300, 400], [1, 1], heads=130, shared=shared) == ["hb_attention_rows"]
    with pytest.raises(KernelError, match="shared beginnings"):
        attend([300, 400, 500], [1, 1, 1], shared=shared)
    shared.page_size = 32                                                            # (whole pages of 32 tokens are none of 64)
    with pytest.raises(KernelError, match="shared beginnings"):
        attend([300, 400], [1, 1], shared=shared)
    assert attend([300, 400], [1, 1], page=32, shared=shared) == ["hb_attention_prefix", "hb_attention_rows"]


def test_a_rotation_table_without_rows():
    k, i32 = Noted(), lambda n: torch.zeros(n, dtype=torch.int32)
    q, qkv, kv = torch.zeros(1, 2, 32, dtype=torch.bfloat16), torch.zeros(1, 128, dtype=torch.bfloat16), torch.zeros(1, 2, 1, 16, 33, dtype=torch.uint8)
    for rows in (1, 0):
        with pytest.raises(KernelError, match="rotation table") if not rows else contextlib.nullcontext():
            k.qk_norm_rope_kv_write(q, qkv, i32(1), torch.zeros(rows, 32), 32, None, None, 1e-6, 0.0, kv, i32(1), 2, 1, 32)
    assert k.called == ["hb_qk_norm_rope_kv_write8"]


@pytest.mark.parametrize("kv8", [True, False])
def test_sharing_that_does_not_pay(kv8):
    least = -(-CudaKernels.SHARED_BYTES[kv8] // (2 * (258 if kv8 else 512)))
    decl = types.SimpleNamespace(kv_heads=2, head_dim=128, fp8=kv8)
    assert Noted().shared_least(decl) == least
    for saved, both in ((None, True), (least, True), (least - 1, False)):
        shared = SharedPrefix(*(torch.zeros(n, dtype=torch.int32) for n in (2, 2, 4)), 2, 50, saved)
        called = attend([200, 200], [1, 1], kv8=kv8, shared=shared, decode_splits=lambda *a: 1, _decode_mode_of=lambda rows: "equal")
        assert ("hb_attention_prefix" in called) == both and len(called) == 1 + both


def test_portions_that_are_read_back_at_once():
    k, rows = Noted(), c8.rows_of([1, 500, 100, 90, 700], [1, 3, 4, 5, 6])
    k.READ_BACK_TOKENS = 1024
    got = list(k._read_back_portions(rows, 6400))
    assert got == [(1, 3, 512), (3, 4, 128), (4, 5, 704)]
    assert all((b - a) * n <= 1024 or b - a == 1 for a, b, n in got)
    assert max((b - a) * n for a, b, n in got) * 2 * 2 * 128 * 2 <= k.read_back_scratch(18, 5, 704, 2, 128)
    rows.plan["any cut"], rows.max_kv = True, 1000
    assert list(k._read_back_portions(rows, 6400)) == [(1, 5, 1024)] and list(k._read_back_portions(rows, 768)) == [(1, 5, 768)]
    assert list(k._read_back_portions(c8.rows_of([4, 5], [1, 1]), 576)) == []
    assert k.read_back_scratch(1, 5, 704, 2, 128) == 0


def test_a_captured_step_is_planned_for_a_bucket_of_own_keys():
    k, rows = Noted(), c8.rows_of([700, 800], [1, 1])
    k.decode_attention = "auto"
    shared = SharedPrefix(None, None, None, 2, 70)
    plan = k.attention_capture_plan(rows, 4096)
    assert len(plan) == 2 and k.attention_capture_plan(rows, 4096, shared) == (*plan, 128) and shared.longest_own == 128
    assert k._prefix_units(64, 32, 8, 128, 64) == max(148 * 2, 8 * (4 + 32)) and k._prefix_units(256, 32, 8, 128, 64) == 8 * (16 + 128)
    assert k.shared_scratch(1, 32, 8, 128, 64) == 296 * 64 * 130 + 4 and k.shared_scratch(1, 130, 1, 128, 64) == 0
