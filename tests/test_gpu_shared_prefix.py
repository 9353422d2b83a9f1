"""Attention of one-token rows that share their first pages, over both kinds of pages: against 64 bits, against the same rows
without sharing, under graphs whose groups change between replays."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import cache8_tools as c8
from holon_b200.engine.batch import SharedPrefix
from holon_b200.kernels.cuda import KernelError
from test_gpu_cache8 import DEV, gpu_rows

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def K():
    from holon_b200.kernels import load_kernels
    table = load_kernels(DEV)
    table.SHARED_BYTES = 0, 0                 # (small groups share, too)
    yield table
    del table.SHARED_BYTES


def within(got, want, mass):
    """Half a step of bfloat16 on the result, half a step of it on the weights of the shared keys, 2^-12 for the 32-bit sums."""
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12) * mass * 1.01 + 1e-30
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), f"{(off / bound).max().item():.3g} times what rounding explains"


def case(groups, alone, heads, kvh, dim, page, fp8, seed=0, portion=None):
    """`groups`: (shared pages, tokens behind them of each member); `alone`: tokens of rows that share nothing. Rows come in a
    shuffled order; `portion` = (held, new) adds a row of several tokens."""
    held, shared = [], []
    for pages, tails in groups:
        shared.append((list(range(len(held), len(held) + len(tails))), pages))
        held += [pages * page + t for t in tails]
    held += alone
    rng = np.random.RandomState(seed)
    order = rng.permutation(len(held))                                # row r is request order[r]
    n_slots = len(held) + 1 + (portion is not None)
    table, count = c8.paged(held + [1] + ([portion[0]] if portion else []), page, n_slots, seed, shared)
    rows = c8.rows_of([held[i] for i in order] + ([portion[0]] if portion else []), [1] * len(held) + ([portion[1]] if portion else []))
    rows.row_slot = torch.tensor(list(order) + ([n_slots - 1] if portion else []), dtype=torch.int32)
    if fp8:
        kv = c8.random_pages(count, kvh, page, dim, seed)
    else:
        kv = torch.randn(count, 2, kvh, page, dim, generator=torch.Generator().manual_seed(seed)).to(BF16)
    q = (1.5 * torch.randn(rows.n_tokens, heads, dim, generator=torch.Generator().manual_seed(seed + 1))).to(BF16)
    found = SharedPrefix.of(table[rows.row_slot[:rows.n_decode].long()].numpy(), rows.host_kv_len[:rows.n_decode], page, DEV, rows.row_slot.numpy())
    return q, kv, table, rows, found


def run(K, q, kv, table, rows, scale, sinks, shared):
    out = torch.full(q.shape, float("nan"), dtype=BF16, device=DEV)
    K.paged_attention(out, q.to(DEV), kv.to(DEV), table.to(DEV), gpu_rows(rows), scale, 0, sinks.to(DEV) if sinks is not None else None, shared=shared)
    return out


CASES = [([(16, [1, 130, 64, 3])], [], 16, 8, 128, 64), ([(9, [7] * 70), (3, [80] * 9)], [4], 12, 2, 128, 64), ([(5, [3] * 3)], [9], 100, 1, 128, 128), ([(5, [9, 70]), (33, [1, 200, 500])], [77, 3], 8, 2, 128, 64),
         ([(30, [1 + 7 * i for i in range(40)])], [5], 4, 1, 96, 16), ([(4, [5] * 17), (9, [300] * 3), (2, [1] * 130)], [1], 6, 2, 64, 128),
         ([(6, [90] * 3)], [200], 5, 5, 80, 64), ([(7, [11] * 70)], [], 2, 1, 256, 80), ([(3, [40, 50])], [], 48, 1, 32, 128),
         ([(40, [20] * 6)], [30] * 3, 128, 2, 128, 16)]


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("groups,alone,heads,kvh,dim,page", CASES)
def test_shared(K, groups, alone, heads, kvh, dim, page, fp8):
    q, kv, table, rows, shared = case(groups, alone, heads, kvh, dim, page, fp8, seed=dim)
    assert shared is not None and int(shared.skip.max()) == max(p for p, t in groups) * page
    sinks = torch.randn(heads, generator=torch.Generator().manual_seed(3)) if heads % 3 else None
    want, mass = c8.attend(q, kv, table, rows, dim ** -0.5, 0, sinks)
    got = run(K, q, kv, table, rows, dim ** -0.5, sinks, shared)
    within(got, want, mass)
    assert torch.equal(got, run(K, q, kv, table, rows, dim ** -0.5, sinks, shared))
    within(run(K, q, kv, table, rows, dim ** -0.5, sinks, None), want, mass)


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("page", [16, 64])
def test_beside_a_portion(K, page, fp8):
    q, kv, table, rows, shared = case([(320 // page, [5, 90, 3])], [40], 8, 2, 128, page, fp8, portion=(500, 130))
    want, mass = c8.attend(q, kv, table, rows, 0.1)
    within(run(K, q, kv, table, rows, 0.1, None, shared), want, mass)


@pytest.mark.parametrize("fp8", [True, False])
def test_more_tiles_than_ctas(K, fp8, monkeypatch):
    """Units in turns: fewer CTAs than there are pieces of work, and one CTA for all."""
    plan = K._prefix_plan
    for ctas, dim, page in ((7, 128, 64), (1, 128, 64), (7, 64, 16), (1, 80, 64)):
        monkeypatch.setattr(K, "_prefix_plan", lambda *a: (ctas, *plan(*a)[1:]), raising=False)
        q, kv, table, rows, shared = case([(6 * 64 // page, [9] * 9), (11 * 64 // page, [30] * 5), (5 * 64 // page, [2, 2])], [5], 32, 2, dim, page,
                                          fp8, seed=1)
        want, mass = c8.attend(q, kv, table, rows, 0.1)
        within(run(K, q, kv, table, rows, 0.1, None, shared), want, mass)


def test_sizes_that_the_shared_kernels_do_not_take(K):
    """Such rows attend by themselves, sharing or not."""
    q, kv, table, rows, shared = case([(6, [9] * 3)], [], 72, 1, 64, 64, False)          # (72 heads a kv head)
    want, mass = c8.attend(q, kv, table, rows, 0.1)
    within(run(K, q, kv, table, rows, 0.1, None, shared), want, mass)
    with pytest.raises(KernelError):
        K.paged_attention(torch.empty_like(q, device=DEV), q.to(DEV), kv.to(DEV), table.to(DEV), gpu_rows(rows), 0.1, 64, shared=shared)
    shared.rows += 1
    with pytest.raises(KernelError):
        run(K, q, kv, table, rows, 0.1, None, shared)


@pytest.mark.parametrize("fp8", [True, False])
def test_numbers_that_are_none(K, fp8):
    """A NaN among the shared keys or values reaches every row that shares them, and no other; one behind a row's keys reaches none."""
    q, kv, table, rows, shared = case([(4, [9, 20]), (5, [30, 1])], [40], 4, 2, 64, 64, fp8)
    clean = run(K, q, kv, table, rows, 0.125, None, shared)
    mine = int(shared.members.cpu()[0])
    group = [b for b in range(5) if table[rows.row_slot[b].long(), 0] == table[rows.row_slot[mine].long(), 0]]
    page = int(table[rows.row_slot[mine].long(), 1])
    for part in (0, 1):
        bad = kv.clone()
        if fp8:
            bad.view(kv.shape[0], 2, 2, -1)[page, part, 1, 5 * 64 + 3] = 127
        else:
            bad[page, part, 1, 5, 3] = float("nan")
        got = run(K, q, bad, table, rows, 0.125, None, shared)
        for b in range(5):
            assert bool(got[b, 2:].isnan().any()) == (b in group) and not got[b, :2].isnan().any()
            assert b in group or torch.equal(got[b], clean[b])


@pytest.mark.parametrize("fp8", [True, False])
def test_graph(K, fp8):
    """A captured launch serves other groups, other lengths and no groups at all; two graphs and an eager call between them."""
    heads, kvh, dim, page = 8, 2, 128, 64
    cases = [case([(16, [1, 130, 64, 3])], [60, 7], heads, kvh, dim, page, fp8, seed=1),
             case([(3, [9, 70]), (12, [1, 200, 100])], [77], heads, kvh, dim, page, fp8, seed=2),
             case([(9, [100] * 6)], [], heads, kvh, dim, page, fp8, seed=3)]
    pages, width = max(c[1].shape[0] for c in cases), max(c[2].shape[1] for c in cases)
    def buffers():
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)               # noqa: E731
        q = torch.zeros(6, heads, dim, dtype=BF16, device=DEV)
        kv = torch.zeros(pages, *cases[0][1].shape[1:], dtype=cases[0][1].dtype, device=DEV)
        from holon_b200.engine.batch import Rows
        rows = Rows(i32(6), torch.arange(7, dtype=torch.int32, device=DEV), i32(6), 6, 6, 6, 1, 2048)
        return q, kv, i32(7, width), rows, SharedPrefix(i32(6), i32(6), i32(12), 6, 512), torch.zeros_like(q)
    def fill(b, c):
        q, kv, table, rows, shared = c
        b[0].copy_(q), b[1][:kv.shape[0]].copy_(kv), b[2].fill_(0)
        b[2][:, :table.shape[1]].copy_(table[:7])
        b[3].row_slot.copy_(rows.row_slot), b[3].kv_len.copy_(rows.kv_len)
        for name in ("skip", "members", "groups"):
            getattr(b[4], name).zero_()
            if shared is not None:
                getattr(b[4], name).copy_(getattr(shared, name))
    def call(b):
        K.paged_attention(b[5], b[0], b[1], b[2], b[3], 0.1, 0, None, shared=b[4])
    both = [buffers(), buffers()]
    graphs, pool = [], None
    for b, c in zip(both, cases):
        fill(b, c)
        call(b)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            call(b)
        pool = pool or g.pool()                                       # (the two share their scratch, as an engine's graphs do)
        graphs.append(g)
    nothing = cases[1][:4] + (None,)
    for first, second in ((0, 1), (2, 0), (1, 2)):
        for b, c in zip(both, (cases[first], nothing if second == 1 else cases[second])):
            fill(b, c)
        graphs[0].replay()
        run(K, *cases[2][:4], 0.1, None, cases[2][4])
        graphs[1].replay()
        torch.cuda.synchronize()
        for b, i in zip(both, (first, second)):
            q, kv, table, rows, _ = cases[i]
            want, mass = c8.attend(q, kv, table, rows, 0.1)
            within(b[5], want, mass)


def test_other_stream(K):
    q, kv, table, rows, shared = case([(16, [1, 130, 64, 3])], [60, 7], 8, 2, 128, 64, True)
    want, mass = c8.attend(q, kv, table, rows, 0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(K, q, kv, table, rows, 0.1, None, shared)
    side.synchronize()
    within(got, want, mass)
