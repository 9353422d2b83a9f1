"""The 8-bit cache on the GPU: codes and scales against their definition in 64 bits, pages read back exactly, attention over
them for one-token rows and for prompts' portions."""
from __future__ import annotations

import pytest
import torch

import cache8_tools as c8
from holon_b200.kernels.cuda import KernelError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def K():
    from holon_b200.kernels import load_kernels
    return load_kernels(DEV)


def gpu_rows(rows):
    from holon_b200.engine.batch import Rows
    return Rows(rows.row_slot.to(DEV), rows.query_start.to(DEV), rows.kv_len.to(DEV), rows.n_rows, rows.n_tokens, rows.n_decode, rows.max_q,
                rows.max_kv, rows.host_query_start, rows.host_kv_len)


def within(got, want, mass, halves: bool):
    """Half a step of bfloat16 on the result (2^-8 of it), and the weights' rounding on the sum of weight x |value|: half a
    step of a half (2^-11) or of bfloat16 (2^-8), of the weights and, in other kernels, of each tile's factor; 2^-12 for the 32-bit
    sums and the exponential's 2^-22 on exponents up to a few hundred."""
    slack = (2.0 ** -11 if halves else 2.0 ** -8) + 2.0 ** -12
    bound = 2.0 ** -8 * want.abs() + slack * mass * 1.01 + 1e-30
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), f"{(off / bound).max().item():.3g} times what rounding explains"


# ---------------------------------------------------------------- writing and reading
def written(x, kv, index, page):
    """What pages hold once rows x [tokens, 2, kv_heads, dim] (64-bit) are written at `index`."""
    codes, e = c8.encode(x)
    c, s = (t.clone() for t in c8.split(kv))
    for i, w in enumerate(index):
        if 0 <= w < kv.shape[0] * page:
            c[w // page, :, :, w % page] = codes[i]
            s[w // page, :, :, w % page] = (e[i] + 127).to(torch.uint8)
    return c, s


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("norm", [None, BF16, torch.float32])
@pytest.mark.parametrize("tokens,heads,kvh,dim,page,rotary", [
    (1, 4, 2, 128, 64, 128), (7, 8, 8, 128, 16, 0), (300, 4, 1, 128, 64, 64), (5, 6, 2, 96, 16, 48), (33, 3, 3, 16, 32, 16), (9, 2, 1, 256, 48, 250),
    (4, 2, 2, 1024, 16, 6), (64, 5, 5, 80, 80, 0)])
def test_write(K, tokens, heads, kvh, dim, page, rotary, norm, bias):
    g = torch.Generator().manual_seed(tokens * 131 + dim)
    rand = lambda *s: torch.randn(*s, generator=g)                                    # noqa: E731
    pages = tokens // page + 3
    qkv = (rand(tokens, heads + 2 * kvh, dim) * 2.0 ** (8 * torch.rand(tokens, heads + 2 * kvh, 1, generator=g) - 4)).to(BF16)
    add = rand((heads + 2 * kvh) * dim).to(BF16) if bias else None
    gains = [(1 + 0.2 * rand(dim)).to(norm) for _ in range(2)] if norm else [None, None]
    positions = torch.randint(0, 50, (tokens,), generator=g, dtype=torch.int32)
    turn = torch.cat([rand(50, rotary // 2).cos(), rand(50, rotary // 2).sin()], -1) if rotary else None
    index = torch.randperm(pages * page, generator=g)[:tokens].int()
    if tokens > 3:
        index[1], index[3] = -1, pages * page + 5                                      # (a padding token; a page that is not there)
    kv = c8.random_pages(pages, kvh, page, dim, seed=5)
    x = qkv.double() + (add.double().view(heads + 2 * kvh, dim) if bias else 0)
    for a, b, w in ((0, heads, gains[0]), (heads, heads + kvh, gains[1])):
        if w is not None:
            x[:, a:b] = x[:, a:b] / (x[:, a:b].square().mean(-1, keepdim=True) + 1e-6).sqrt() * (w.double() + 0.5)
        if rotary:
            h = rotary // 2
            cs = turn[positions.long()].double()[:, None]
            lo, hi = x[:, a:b, :h].clone(), x[:, a:b, h:rotary].clone()
            x[:, a:b, :h], x[:, a:b, h:rotary] = lo * cs[..., :h] - hi * cs[..., h:], hi * cs[..., :h] + lo * cs[..., h:]
    dev = lambda t: t.to(DEV) if t is not None else None                              # noqa: E731
    q, got = torch.full((tokens, heads, dim), float("nan"), dtype=BF16, device=DEV), kv.to(DEV)
    K.qk_norm_rope_kv_write(q, dev(qkv.reshape(tokens, -1)), dev(positions), dev(turn), rotary, dev(gains[0]), dev(gains[1]), 1e-6, 0.5, got,
                            dev(index), heads, kvh, dim, dev(add))
    want = x[:, :heads]
    assert bool(((q.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * want.abs().amax(-1, keepdim=True)).all())
    rows = torch.stack([x[:, heads:heads + kvh], x[:, heads + kvh:]], 1)
    codes, scales = c8.split(got.cpu())
    want_c, want_s = written(rows, kv, index.tolist(), page)
    # 32-bit arithmetic may move a number across the border between two codes, or a row's largest across that of its scale: as many
    # steps of 2^-24 as there are roundings on the way (under 200), of the row's largest number
    moved = codes != want_c
    values = c8.decode(got.cpu())
    exact = c8.decode(kv).clone()
    for i, w in enumerate(index.tolist()):
        if 0 <= w < pages * page:
            exact[w // page, :, :, w % page] = rows[i]
    scale = 2.0 ** (scales.double() - 127)[..., None]
    step = torch.maximum(2.0 ** torch.floor(torch.log2(values.abs().clamp(min=1e-300))) / 8, scale * 2.0 ** -9)
    assert bool(((values - exact).abs() <= step / 2 + 200 * 2.0 ** -24 * exact.abs().amax(-1, keepdim=True)).all())
    assert moved.double().mean() < 1e-3 and (scales != want_s).double().mean() < 1e-3
    untouched = torch.ones(pages * page, dtype=torch.bool)
    untouched[index[(index >= 0) & (index < pages * page)].long()] = False
    same = lambda a, b: torch.equal(a.permute(0, 3, 1, 2, *range(4, a.dim())).flatten(0, 1)[untouched],        # noqa: E731
                                    b.permute(0, 3, 1, 2, *range(4, b.dim())).flatten(0, 1)[untouched])
    old_c, old_s = c8.split(kv)
    assert same(codes, old_c) and same(scales, old_s)


def test_write_exactly(K):
    """Values as they are (no norm, no rotation): every code and scale to the bit, borders, subnormal codes, zeros, the largest
    bfloat16, NaN and infinities among others."""
    dim, page, kvh = 32, 16, 1
    steps = torch.arange(0, 449 * 4, 13).double() / 4
    rows = [steps[i:i + dim] for i in range(0, len(steps) - dim, dim)]
    rows += [torch.linspace(-1, 1, dim).double() * 2.0 ** e for e in (-130, -80, -70, -64, -20, 0, 60, 110, 127)]
    rows += [torch.zeros(dim).double(), torch.full((dim,), 3.3895313892515355e38).double(), torch.full((dim,), 1.75 * 2.0 ** 5).double(),
             torch.full((dim,), 1.7578125 * 2.0 ** 5).double()]
    odd = torch.linspace(-3, 3, dim).double()
    odd[3], odd[7], odd[9] = float("nan"), float("inf"), float("-inf")
    rows += [odd, torch.full((dim,), float("nan")).double(), torch.full((dim,), float("inf")).double()]
    v = torch.stack(rows).to(BF16)
    t = len(v)
    qkv = torch.cat([torch.zeros(t, dim), v.flip(-1).float(), v.float()], -1).to(BF16)
    kv = torch.zeros(-(-t // page), 2, kvh, page, dim + 1, dtype=torch.uint8, device=DEV)
    q = torch.empty(t, 1, dim, dtype=BF16, device=DEV)
    K.qk_norm_rope_kv_write(q, qkv.to(DEV), torch.zeros(t, dtype=torch.int32, device=DEV), None, 0, None, None, 0.0, 0.0, kv,
                            torch.arange(t, dtype=torch.int32, device=DEV), 1, kvh, dim)
    want_c, want_s = written(torch.stack([v.flip(-1), v], 1).double()[:, :, None], kv.cpu() * 0, range(t), page)
    codes, scales = c8.split(kv.cpu())
    nan = (want_c & 127) == 127
    assert torch.equal((codes & 127) == 127, nan)
    assert torch.equal(codes[~nan], want_c[~nan]) and torch.equal(scales, want_s)


def test_write_refusals(K):
    def call(dim=32, page=16, dtype=BF16, kv=None, heads=2, **change):
        kv = torch.zeros(2, 2, 1, page, dim + 1, dtype=torch.uint8, device=DEV) if kv is None else kv
        args = dict(positions=torch.zeros(3, dtype=torch.int32, device=DEV), index=torch.zeros(3, dtype=torch.int32, device=DEV)) | change
        K.qk_norm_rope_kv_write(torch.empty(3, heads, dim, dtype=dtype, device=DEV), torch.zeros(3, (heads + 2) * dim, dtype=dtype, device=DEV),
                                args["positions"], None, 0, None, None, 0.0, 0.0, kv, args["index"], heads, 1, dim)
    call()
    for bad in (dict(dtype=torch.float32), dict(dim=24), dict(page=8), dict(kv=torch.zeros(2, 2, 1, 16, 32, dtype=torch.uint8, device=DEV)),
                dict(kv=torch.zeros(2, 2, 2, 16, 33, dtype=torch.uint8, device=DEV)), dict(dim=1040),
                dict(positions=torch.zeros(2, dtype=torch.int32, device=DEV)), dict(index=torch.zeros(3, dtype=torch.int64, device=DEV))):
        with pytest.raises(KernelError):
            call(**bad)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("kvh,page,dim", [(2, 16, 256), (1, 64, 128), (3, 48, 16), (8, 64, 80)])
def test_read(K, dtype, kvh, page, dim):
    g = torch.Generator().manual_seed(dim)
    codes = torch.randint(0, 256, (9, 2, kvh, page, dim), generator=g).to(torch.uint8)
    e = torch.randint(c8.LOW, 119, (9, 2, kvh, page), generator=g)
    kv = c8.pack(codes, e)
    pages = torch.tensor([3, 0, 8, 3, -1, 9, 2 ** 31 - 1, 5], dtype=torch.int32)
    out = torch.full((8, 2, kvh, page, dim), 7.0, dtype=dtype, device=DEV)
    K.kv_read(out, kv.to(DEV), pages.to(DEV))
    want = torch.zeros(8, 2, kvh, page, dim, dtype=torch.float64)
    for i, p in enumerate(pages.tolist()):
        if 0 <= p < 9:
            want[i] = c8.decode(kv[p:p + 1])[0]
    assert torch.equal(out.cpu().double().isnan(), want.isnan())
    assert torch.equal(out.cpu().double().nan_to_num(0.0), want.nan_to_num(0.0))       # (exact in both types)
    K.kv_read(out[:0], kv.to(DEV), pages[:0].to(DEV))
    with pytest.raises(KernelError):
        K.kv_read(out[:2], kv.to(DEV), pages.to(DEV))
    with pytest.raises(KernelError):
        K.kv_read(out.half() if dtype == BF16 else out.to(torch.float64), kv.to(DEV), pages.to(DEV))


# ---------------------------------------------------------------- attention
def case(held, new, heads, kvh, dim, page, seed=0, spread=4.0, sharp=1.5):
    n_slots = len(held) + 2
    rows = c8.rows_of(held, new, n_slots=n_slots, seed=seed)
    by_slot = [1] * n_slots
    for s, n in zip(rows.row_slot.tolist(), held):
        by_slot[s] = max(1, n)
    table, count = c8.paged(by_slot, page, n_slots, seed)
    kv = c8.random_pages(count, kvh, page, dim, seed, spread)
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn(rows.n_tokens, heads, dim, generator=g) * sharp).to(BF16)
    return q, kv, table, rows


def run(K, q, kv, table, rows, scale, window=0, sinks=None):
    out = torch.full(q.shape, float("nan"), dtype=BF16, device=DEV)
    K.paged_attention(out, q.to(DEV), kv.to(DEV), table.to(DEV), gpu_rows(rows), scale, window, sinks.to(DEV) if sinks is not None else None)
    return out


ONES = [([1], 4, 2, 128, 64), ([400], 16, 8, 128, 64), ([64, 65, 63, 128, 1, 2], 8, 2, 128, 64), ([33, 900, 16, 17], 6, 2, 96, 16),
        ([77] * 5, 5, 5, 16, 48), ([500, 3], 40, 2, 64, 32), ([1025, 700], 4, 1, 256, 80), ([3000, 10, 1500], 12, 2, 80, 128),
        ([200] * 40, 8, 8, 32, 16), ([5000], 2, 1, 240, 64)]


@pytest.mark.parametrize("window", [0, 1, 50, 130])
@pytest.mark.parametrize("held,heads,kvh,dim,page", ONES)
def test_one_token_rows(K, held, heads, kvh, dim, page, window):
    q, kv, table, rows = case(held, [1] * len(held), heads, kvh, dim, page, seed=dim + page)
    sinks = torch.randn(heads, generator=torch.Generator().manual_seed(3)) if window != 50 else None
    want, mass = c8.attend(q, kv, table, rows, dim ** -0.5, window, sinks)
    got = run(K, q, kv, table, rows, dim ** -0.5, window, sinks)
    within(got, want, mass, halves=True)
    assert torch.equal(got, run(K, q, kv, table, rows, dim ** -0.5, window, sinks))    # (the same bits again)


@pytest.mark.parametrize("splits,few", [(1, 0), (2, 0), (3, 0), (5, 0), (8, 0), (11, 0), (16, 0), (1, 1)])
def test_cuts_of_a_row(K, splits, few, monkeypatch):
    """Any number of CTAs a row, more than it has tiles too; the form for few keys, which is not cut."""
    for held, heads, kvh, dim, page in (([700, 64, 1, 130], 8, 2, 128, 64), ([300, 9], 34, 2, 48, 16), ([2000], 3, 1, 256, 32)):
        q, kv, table, rows = case(held, [1] * len(held), heads, kvh, dim, page, seed=splits)
        monkeypatch.setattr(K, "_row_splits", lambda *a: (splits, few, splits & 1), raising=False)
        want, mass = c8.attend(q, kv, table, rows, dim ** -0.5)
        within(run(K, q, kv, table, rows, dim ** -0.5), want, mass, halves=True)


def test_the_form_for_few_keys_refuses_cuts(K, monkeypatch):
    q, kv, table, rows = case([700], [1], 8, 2, 128, 64, seed=1)
    monkeypatch.setattr(K, "_row_splits", lambda *a: (2, 1, 0), raising=False)
    with pytest.raises(KernelError, match="few keys"):
        run(K, q, kv, table, rows, 1.0)


def test_scales_far_apart(K):
    """Keys and values whose scales differ by up to 2^60: a value's scale must neither overflow a weight nor lose it."""
    for spread in (30.0, 60.0):
        q, kv, table, rows = case([300, 70], [1, 1], 4, 2, 64, 16, seed=9, spread=spread, sharp=0.0)
        want, mass = c8.attend(q, kv, table, rows, 1.0)                                # (equal weights: the values' sizes alone count)
        within(run(K, q, kv, table, rows, 1.0), want, mass, halves=True)
    q, kv, table, rows = case([300, 70], [1, 1], 4, 2, 64, 16, seed=9, spread=0.0, sharp=2000.0)
    want, mass = c8.attend(q, kv, table, rows, 2.0 ** -8)                              # (queries far outside a half's range)
    within(run(K, q, kv, table, rows, 2.0 ** -8), want, mass, halves=True)


def test_what_is_masked_does_not_count(K):
    """Bytes behind a row's last key, in pages of others and in the spare page may hold anything: NaN codes, any scale."""
    for window in (0, 40):
        held = [70, 33, 129, 1]
        q, kv, table, rows = case(held, [1] * 4, 4, 2, 64, 16, seed=2)
        want, mass = c8.attend(q, kv, table, rows, 0.125, window)
        flat, seen = kv.view(kv.shape[0], 2, 2, -1).clone(), torch.zeros(kv.shape[0], 16, dtype=torch.bool)
        for s, n in zip(rows.row_slot.tolist(), held):
            for j in range(max(0, n - window) if window else 0, n):
                seen[table[s, j // 16], j % 16] = True
        for p in range(kv.shape[0]):
            for o in range(16):
                if not seen[p, o]:
                    flat[p, :, :, o * 64:(o + 1) * 64] = 127
                    flat[p, :, :, 16 * 64 + o] = 255
        within(run(K, q, flat.view(kv.shape), table, rows, 0.125, window), want, mass, halves=True)


def test_numbers_that_are_none(K):
    """A NaN among a row's keys makes the heads that see it NaN, and only those; so does one in its query."""
    q, kv, table, rows = case([70, 33], [1, 1], 4, 2, 64, 16, seed=2)
    flat = kv.view(kv.shape[0], 2, 2, -1)
    flat[table[rows.row_slot[0], 2], 0, 1, 5 * 64 + 3] = 127                            # row 0, kv head 1, key 37
    got = run(K, q, kv, table, rows, 0.125)
    assert got[0, 2:].isnan().all() and not got[0, :2].isnan().any() and not got[1].isnan().any()
    q, kv, table, rows = case([70, 33], [1, 1], 4, 2, 64, 16, seed=2)
    q[1, 3, 7] = float("nan")
    got = run(K, q, kv, table, rows, 0.125)
    assert got[1, 3].isnan().all() and not got[1, :3].isnan().any() and not got[0].isnan().any()


def test_rows_without_keys_and_pages_that_are_not_there(K):
    q, kv, table, rows = case([20, 30], [1, 1], 4, 2, 64, 16, seed=4)
    rows.kv_len[0] = 0
    assert not run(K, q, kv, table, rows, 0.125)[0].any()
    q, kv, table, rows = case([40, 30], [1, 1], 4, 2, 64, 16, seed=4)
    table[rows.row_slot[0], 1], table[rows.row_slot[1], 0] = kv.shape[0], -7            # these keys count as zeros
    zeroed, at = torch.cat([kv, torch.zeros_like(kv[:1])]), table.clone()
    at[at < 0], at[at >= kv.shape[0]] = kv.shape[0], kv.shape[0]
    want, mass = c8.attend(q, zeroed, at, rows, 0.125)
    within(run(K, q, kv, table, rows, 0.125), want, mass, halves=True)


PROMPTS = [([300, 90], [300, 17], 8, 2, 128, 64), ([33, 900, 40], [2, 300, 40], 6, 2, 96, 16), ([1, 700, 64, 650, 400], [1, 1, 2, 650, 64], 4, 4, 128, 128),
           ([130, 257], [130, 129], 2, 1, 256, 32), ([50, 40], [3, 40], 5, 5, 16, 48), ([130, 300, 700, 2], [129, 256, 5, 2], 8, 8, 128, 16),
           ([1000, 128], [600, 128], 4, 1, 128, 48), ([2000], [257], 2, 2, 128, 64), ([40, 900], [1, 899], 16, 2, 128, 32)]


@pytest.mark.parametrize("window", [0, 37, 300])
@pytest.mark.parametrize("held,new,heads,kvh,dim,page", PROMPTS)
def test_portions(K, held, new, heads, kvh, dim, page, window, monkeypatch):
    q, kv, table, rows = case(held, new, heads, kvh, dim, page, seed=dim)
    sinks = torch.randn(heads, generator=torch.Generator().manual_seed(3)) if window else None
    want, mass = c8.attend(q, kv, table, rows, dim ** -0.5, window, sinks)
    whole = run(K, q, kv, table, rows, dim ** -0.5, window, sinks)
    within(whole, want, mass, halves=False)
    monkeypatch.setattr(K, "READ_BACK_TOKENS", 256, raising=False)                      # (a few rows, or one, at a time)
    assert len(list(K._read_back_portions(rows, table.shape[1] * page))) > 1 or sum(n > 1 for n in new) < 2 or sum(held) < 256
    assert torch.equal(run(K, q, kv, table, rows, dim ** -0.5, window, sinks), whole)


def test_portions_behind_what_is_masked(K):
    """Rows of several tokens beside NaN bytes in the tail of their last page."""
    for dim, page, window in ((128, 64, 0), (64, 16, 0), (128, 16, 0), (128, 16, 20), (64, 16, 20)):
        held = [270, 133]
        q, kv, table, rows = case(held, [40, 5], 4, 2, dim, page, seed=2)
        want, mass = c8.attend(q, kv, table, rows, 0.1, window)
        flat = kv.view(kv.shape[0], 2, 2, -1)
        for s, n, new in zip(rows.row_slot.tolist(), held, (40, 5)):
            flat[table[s, (n - 1) // page], :, :, ((n - 1) % page + 1) * dim:page * dim] = 127
            before = n - new - window + 1 if window else 0           # what lies before the first new token's window, too
            for j in range(before):
                flat[table[s, j // page], :, :, j % page * dim:(j % page + 1) * dim] = 127
                flat[table[s, j // page], :, :, page * dim + j % page] = 255
        within(run(K, q, kv, table, rows, 0.1, window), want, mass, halves=False)


def test_attention_refusals(K):
    q, kv, table, rows = case([40], [1], 4, 2, 64, 16)
    for bad_q, bad_kv in ((q.float(), kv), (q, kv[..., :-1].contiguous()), (q[..., :60].contiguous(), kv), (q[:, :3].contiguous(), kv),
                          (q, kv[:, :, :, :8].contiguous()), (q, kv[:, :1].contiguous())):
        with pytest.raises(KernelError):
            run(K, bad_q, bad_kv, table, rows, 0.125)
    with pytest.raises(KernelError):
        run(K, q, kv, table, rows, -0.125)
