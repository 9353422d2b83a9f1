"""The 8-bit cache in plain numbers, for tests: codes and scales from their definition in 64 bits, pages laid out from them,
attention over them, and the plain kernel table with an 8-bit cache."""
from __future__ import annotations

import math

import numpy as np
import torch

from holon_b200.engine.batch import Rows
from ref_kernels import RefKernels

LOW, HIGH = -64, 120


def code_values() -> torch.Tensor:
    """What each of the 256 codes stands for: a sign, four bits of exponent less 7, three of fraction."""
    out = []
    for b in range(256):
        e, f = (b >> 3) & 15, b & 7
        v = math.ldexp(f / 8, -6) if e == 0 else math.ldexp(1 + f / 8, e - 7)
        out.append(math.nan if b & 127 == 127 else -v if b & 128 else v)
    return torch.tensor(out, dtype=torch.float64)


VALUES = code_values()
POSITIVE = VALUES[:127].numpy()                                       # ascending: 0 .. 448


def encode(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of 64-bit numbers -> (codes uint8 [..., dim], exponents [...]): nearest code, ties to the even one."""
    x = x.double()
    a = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
    e = torch.full(a.shape, LOW, dtype=torch.int64)
    for k in range(LOW + 1, HIGH + 1):
        e = torch.where(a > 448 * 2.0 ** (k - 1), k, e)
    y = (x * 2.0 ** -e.double()[..., None]).numpy()
    mag = np.minimum(np.abs(np.nan_to_num(y, nan=0.0, posinf=0.0, neginf=0.0)), 448)
    hi = np.clip(np.searchsorted(POSITIVE, mag), 0, 126)              # the first code whose value is not below
    lo = np.maximum(hi - 1, 0)
    up, down = POSITIVE[hi] - mag, mag - POSITIVE[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = code | np.where(np.signbit(y), 128, 0)
    code = np.where(np.isfinite(y), code, 127)
    return torch.from_numpy(code.astype(np.uint8)), e


def pack(codes: torch.Tensor, e: torch.Tensor) -> torch.Tensor:
    """Codes [pages, 2, kv_heads, page, dim] and exponents [pages, 2, kv_heads, page] as pages of bytes."""
    p, two, kvh, page, dim = codes.shape
    out = torch.cat([codes.reshape(p, two, kvh, page * dim), (e + 127).to(torch.uint8)], -1)
    return out.reshape(p, two, kvh, page, dim + 1)


def split(kv: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scale bytes) of pages of bytes, as views into a copy."""
    p, two, kvh, page, d1 = kv.shape
    flat = kv.reshape(p, two, kvh, page * d1)
    return flat[..., :page * (d1 - 1)].reshape(p, two, kvh, page, d1 - 1), flat[..., page * (d1 - 1):]


def decode(kv: torch.Tensor) -> torch.Tensor:
    """The 64-bit values [pages, 2, kv_heads, page, dim] of pages of bytes (of pages in another type: their values)."""
    if kv.dtype != torch.uint8:
        return kv.double()
    codes, scales = split(kv)
    return VALUES[codes.long()] * 2.0 ** (scales.double() - 127)[..., None]


def attend(q, kv, table, rows, scale, window=0, sinks=None):
    """(out, sum of weight x |value|) in 64 bits: what the weights' rounding is a share of."""
    kv = decode(kv)
    page, heads, kvh, dim = kv.shape[3], q.shape[1], kv.shape[2], q.shape[2]
    out, mass = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    starts, slots, lens = rows.query_start.tolist(), rows.row_slot.tolist(), rows.kv_len.tolist()
    for b in range(rows.n_rows):
        s, e, n = starts[b], starts[b + 1], lens[b]
        if n == 0 or s == e:
            continue
        pages = table[slots[b], :-(-n // page)].long()
        k, v = (kv[pages, i].transpose(1, 2).reshape(-1, kvh, dim)[:n].repeat_interleave(heads // kvh, 1) for i in (0, 1))
        scores = torch.einsum("qhd,khd->hqk", q[s:e].double(), k) * scale
        pos, key = torch.arange(n - (e - s), n)[:, None], torch.arange(n)[None]
        hidden = key > pos
        if window > 0:
            hidden = hidden | (pos - key >= window)
        scores = scores.masked_fill(hidden, -math.inf)
        if sinks is not None:
            scores = torch.cat([scores, sinks.double()[:, None, None].expand(-1, e - s, 1)], -1)
        w = scores.softmax(-1)[..., :n]
        out[s:e] = torch.einsum("hqk,khd->qhd", w, v)
        mass[s:e] = torch.einsum("hqk,khd->qhd", w, v.abs())
    return out, mass


def rows_of(held, new, device="cpu", n_slots=None, seed=0):
    """Rows that hold `held` tokens after bringing `new` (ones first), in shuffled slots, and the slots."""
    slots = torch.randperm(n_slots or len(held), generator=torch.Generator().manual_seed(seed))[:len(held)].int()
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    held = np.asarray(held, dtype=np.int32)
    ones = sum(1 for n in new if n == 1)
    assert all(n == 1 for n in new[:ones])
    return Rows(slots.to(device), torch.from_numpy(starts).to(device), torch.from_numpy(held).to(device), len(held), int(starts[-1]), ones,
                int(max(new)), int(held.max()), starts, held)


def paged(held, page, n_slots, seed=0, shared=()):
    """A block table [n_slots, pages] (host) for slots that hold `held[slot]` tokens, pages in random order, one spare page more than
    used; `shared`: (slots, pages) groups whose first pages are the same ones. Unused cells name the spare page."""
    width = max(1, max(-(-n // page) for n in held))
    table = np.full((n_slots, width), -1, dtype=np.int64)
    count = 0
    for group, pages in shared:
        for s in group:
            table[s, :pages] = np.arange(count, count + pages)
        count += pages
    for s, n in enumerate(held):
        for i in range(-(-n // page)):
            if table[s, i] < 0:
                table[s, i] = count
                count += 1
    order = np.random.RandomState(seed).permutation(count + 1)        # (order[count]: the spare page)
    return torch.from_numpy(order[np.where(table < 0, count, table)].astype(np.int32)), count + 1


def random_pages(count, kvh, page, dim, seed=0, spread=4.0):
    """Pages of random codes (no NaN) whose rows' scales differ by factors of up to 2^spread, and values of order one."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(count, 2, kvh, page, dim, generator=g, dtype=torch.float64)
    x = x * 2.0 ** ((torch.rand(count, 2, kvh, page, 1, generator=g, dtype=torch.float64) - 0.5) * spread)
    return pack(*encode(x))


class RefKernels8(RefKernels):
    """The plain kernel table with an 8-bit cache; rows that share pages attend row by row here."""

    def qk_norm_rope_kv_write(self, q_out, qkv, positions, table, rotary_dim, q_weight, k_weight, eps, offset, kv, write_index, heads,
                              kv_heads, head_dim, bias=None):
        if kv is None or kv.dtype != torch.uint8:
            return super().qk_norm_rope_kv_write(q_out, qkv, positions, table, rotary_dim, q_weight, k_weight, eps, offset, kv,
                                                 write_index, heads, kv_heads, head_dim, bias)
        t, page = qkv.shape[0], kv.shape[3]
        wide = lambda x: None if x is None else x.float()                              # noqa: E731
        index = torch.arange(t, dtype=torch.int32)
        q, exact = torch.empty(t, heads, head_dim), torch.zeros(t, 2, kv_heads, 1, head_dim)
        super().qk_norm_rope_kv_write(q, qkv.float(), positions, table, rotary_dim, wide(q_weight), wide(k_weight), eps, offset, exact,
                                      index, heads, kv_heads, head_dim, wide(bias))
        q_out.copy_(q)
        codes, e = encode(exact[:, :, :, 0])
        flat = kv.view(kv.shape[0], 2, kv_heads, -1)
        for i, w in enumerate(write_index.tolist()):
            if 0 <= w < kv.shape[0] * page:
                p, off = divmod(w, page)
                flat[p, :, :, off * head_dim:(off + 1) * head_dim] = codes[i]
                flat[p, :, :, page * head_dim + off] = (e[i] + 127).to(torch.uint8)

    def kv_read(self, out, kv, pages):
        out.zero_()
        for i, p in enumerate(pages.tolist()):
            if 0 <= p < kv.shape[0]:
                out[i] = decode(kv[p:p + 1])[0].to(out.dtype)

    def paged_attention(self, out, q, kv, block_table, rows, scale, window, sinks=None, shared=None):
        super().paged_attention(out, q, decode(kv).float() if kv.dtype == torch.uint8 else kv, block_table, rows, scale, window, sinks)
