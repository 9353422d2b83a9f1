"""A step's batch: what the caller gives (`StepEntry`) and what the model sees on the device (`StepContext`).

The layout is the reference's: flat and token-major, rows marked by `query_start`, with a block table and write
indices per cache group (core/holon/api/batch.py:123-152; core/holon/api/state.py:56-68). A row is a request's
next tokens; a prompt portion and a single decoded token differ only in their length.
"""
from __future__ import annotations

import dataclasses
from collections.abc import Sequence

import numpy as np
import torch

from ..parts.model import LayerCache


@dataclasses.dataclass
class StepEntry:
    """Request in slot `slot` brings `tokens`, which take positions `start`, `start + 1`, …; `want` lists the places
    among these tokens whose logits the caller asks for (it may be empty)."""

    slot: int
    tokens: Sequence[int]
    start: int
    want: Sequence[int] = ()
    from_last: bool = False        # its one token is the one this request sampled last, still on the device


class Rows:
    """The step's rows as attention needs them. Device: `row_slot` [B], `query_start` [B+1], `kv_len` [B] (tokens a
    row holds after this step), all int32. Host: the same as numpy, and the counts kernels size their grids with.
    Rows that bring one token come first (`n_decode` of them)."""

    __slots__ = ("row_slot", "query_start", "kv_len", "n_rows", "n_tokens", "n_decode", "max_q", "max_kv",
                 "host_query_start", "host_kv_len", "plan")

    def __init__(self, row_slot, query_start, kv_len, n_rows, n_tokens, n_decode, max_q, max_kv,
                 host_query_start=None, host_kv_len=None) -> None:
        self.row_slot, self.query_start, self.kv_len = row_slot, query_start, kv_len
        self.n_rows, self.n_tokens, self.n_decode, self.max_q, self.max_kv = n_rows, n_tokens, n_decode, max_q, max_kv
        self.host_query_start, self.host_kv_len = host_query_start, host_kv_len
        self.plan: dict = {}                           # what the kernel table worked out for these rows, for the next layer


class SharedPrefix:
    """Which one-token rows of a step hold the same first pages, so that attention reads the keys there once for all of them.

    A group is two or more rows and the tokens that all of them share (whole pages, and fewer than any of them holds); a
    row is in one group at most. Device, int32: `skip` [rows] (tokens that the row shares, 0 outside the groups), `members`
    [rows] (the groups' rows, one group after the other; what follows is not read) and `groups` [4 · (rows // 2)] ((start in `members`,
    rows, tokens, the block-table row of one of them) a group, zeros behind the last). Host: `rows`; `longest_own`, the most tokens any row
    has beside those it shares; `saved`, the tokens that are read once in place of again (None: whatever they are, share);
    `page_size`, of the pages that the tokens are whole numbers of (0: not known)."""

    __slots__ = ("skip", "members", "groups", "rows", "longest_own", "saved", "page_size")

    LEAST = 256                # tokens that are read once in place of again (over a group's rows but one) from which a group is one

    def __init__(self, skip, members, groups, rows: int, longest_own: int, saved: int | None = None, page_size: int = 0) -> None:
        self.skip, self.members, self.groups, self.rows = skip, members, groups, rows
        self.longest_own, self.saved, self.page_size = longest_own, saved, page_size

    @classmethod
    def find(cls, table: np.ndarray, kv_len: np.ndarray, page_size: int, row_slot: np.ndarray, least: int = 0) -> dict | None:
        """The arrays (host), `longest_own` and `saved` for rows that hold `kv_len` tokens in the pages `table` [rows, pages], the rows
        `row_slot` of the block table; None where no group is worth it, or where the rows cannot save `least` tokens whatever they share
        (of each group one row's tokens are read, so at most all but the longest row's are saved). Rows that share more with some than with
        others go with the cut that saves most."""
        n = len(kv_len)
        limit = np.maximum((np.asarray(kv_len, dtype=np.int64) - 1) // page_size, 0)      # (a row's last token stays its own)
        if n < 2 or int(limit.sum() - limit.max()) * page_size < least:
            return None
        first = table[:, 0] if n > 1 and table.shape[1] else np.zeros(0, dtype=np.int32)
        if len(np.unique(first)) == len(first):                       # (no two rows begin alike)
            return None
        found: list[tuple[list[int], int]] = []
        for rows in cls._alike(range(n), table, limit, 0):
            found += cls._cut(rows, table, limit, 0, page_size)[1]
        if not found:
            return None
        skip, members, groups = np.zeros(n, dtype=np.int32), np.zeros(n, dtype=np.int32), np.zeros(4 * (n // 2), dtype=np.int32)
        at = 0
        for i, (rows, pages) in enumerate(found):
            skip[rows] = pages * page_size
            members[at:at + len(rows)] = rows
            groups[4 * i:4 * i + 4] = at, len(rows), pages * page_size, row_slot[rows[0]]
            at += len(rows)
        return {"skip": skip, "members": members, "groups": groups, "longest_own": int((np.asarray(kv_len) - skip).max()),
                "saved": sum((len(rows) - 1) * pages * page_size for rows, pages in found)}

    @staticmethod
    def _alike(rows, table, limit, page: int) -> list[list[int]]:
        """The rows that still share at page number `page`, two or more with the same page, in their order."""
        by: dict[int, list[int]] = {}
        for r in rows:
            if limit[r] > page:
                by.setdefault(int(table[r, page]), []).append(r)
        return [same for same in by.values() if len(same) > 1]

    @classmethod
    def _cut(cls, rows: list[int], table, limit, page: int, page_size: int) -> tuple[int, list]:
        """(tokens saved, groups as (rows, pages)) for rows that share all pages up to number `page`, and that one."""
        most = int(limit[rows].min())
        cells = table[rows, page:most]
        same = (cells == cells[0]).all(0)
        pages = most if same.all() else page + int(np.argmin(same))
        saved = pages * page_size * (len(rows) - 1)
        whole = (saved, [(rows, pages)]) if saved >= cls.LEAST else (0, [])
        parts = [cls._cut(more, table, limit, pages, page_size) for more in cls._alike(rows, table, limit, pages)]
        apart = sum(p[0] for p in parts), [g for p in parts for g in p[1]]
        return apart if apart[0] > whole[0] else whole

    @classmethod
    def of(cls, table: np.ndarray, kv_len: np.ndarray, page_size: int, device, row_slot: np.ndarray | None = None) -> "SharedPrefix | None":
        """`find`, its arrays on the device. `row_slot` None: `table` is the block table itself, a row of the step a row of it."""
        found = cls.find(table, kv_len, page_size, np.arange(len(kv_len)) if row_slot is None else row_slot)
        if found is None:
            return None
        on = [torch.from_numpy(found[name]).to(device) for name in ("skip", "members", "groups")]
        return cls(*on, len(kv_len), found["longest_own"], found["saved"], page_size)


class GroupStep:
    """One cache group's part of a step: the device block table and, per token, page · page_size + offset; `shared`: which of
    the one-token rows hold the same first pages of this group (None: none, or nobody asked)."""

    __slots__ = ("block_table", "write_index", "page_size", "decl", "shared")

    def __init__(self, block_table, write_index, page_size, decl=None, shared: SharedPrefix | None = None) -> None:
        self.block_table, self.write_index, self.page_size = block_table, write_index, page_size
        self.decl, self.shared = decl, shared


class StepContext:
    def __init__(self, token_ids, positions, logits_index, rows: Rows, groups: list[GroupStep], cache) -> None:
        self.token_ids, self.positions, self.logits_index, self.rows = token_ids, positions, logits_index, rows
        self.groups, self._cache = groups, cache
        self.extra: dict = {}
        self.shared: dict = {}       # what a layer leaves for later layers of the same step (an earlier layer's values, the
                                     # results of all layers so far), by a name the parts agree on
        self.link = None             # parts.base.Link: a block's offer to the product that ends its mixer or feed-forward
        self.from_last = None        # int32 [rows]: 1 where the row's token is fed from the device
        self.offset_of: dict = {}    # host: entry index -> offset of its first token among the step's tokens
        self.layout: tuple = ()      # host: what decides where the step's arrays lie beside its counts (the cache groups whose rows share)

    def entry_slots(self, entry: int) -> dict:
        """The fixed-size per-request tensors kept under cache entry `entry`, by name."""
        return {name: t for (e, name), t in self._cache.slot_states.items() if e == entry}

    def layer_cache(self, run) -> LayerCache:
        c = self._cache
        group = c.group_of_entry.get(run.cache)
        slots = {name: t for (entry, name), t in c.slot_states.items() if entry == run.cache}
        if group is None:
            return LayerCache(None, None, run.fills, slots)
        return LayerCache(c.kv_of_entry[run.cache], self.groups[group.index], run.fills, slots)


class Uploader:
    """One page-locked host buffer and one device buffer of int32: a step's small arrays are laid out one after the
    other on the host and go over in a single copy (core/holon/core/inputs.py:24-87). Two host buffers alternate, and
    a buffer is written again only after the copy that read it last has finished."""

    ALIGN = 4                                     # int32 elements: every array starts on a 16-byte boundary

    def __init__(self, capacity: int, device) -> None:
        self.device = torch.device(device)
        cuda = self.device.type == "cuda"
        self._host = [torch.zeros(capacity, dtype=torch.int32) for _ in range(2)]
        if cuda:
            self._host = [h.pin_memory() for h in self._host]
        self._np = [h.numpy() for h in self._host]
        self._events = [torch.cuda.Event() if cuda else None for _ in range(2)]
        self._used = [False, False]
        self.dev = torch.zeros(capacity, dtype=torch.int32, device=self.device)
        self._which, self._at, self._views = 0, 0, {}
        self.bytes_last = 0

    def begin(self) -> None:
        self._which ^= 1
        if self._used[self._which] and self._events[self._which] is not None:
            self._events[self._which].synchronize()
        self._at, self._views = 0, {}

    def put(self, name: str, array: np.ndarray) -> None:
        n = int(array.shape[0])
        if self._at + n > self.dev.shape[0]:
            raise ValueError(f"a step's arrays need more than the {self.dev.shape[0]} int32 the upload buffer holds")
        self._np[self._which][self._at:self._at + n] = array
        self._views[name] = (self._at, n)
        self._at = -(-(self._at + n) // self.ALIGN) * self.ALIGN

    def end(self) -> dict[str, torch.Tensor]:
        w, n = self._which, self._at
        if n:
            self.dev[:n].copy_(self._host[w][:n], non_blocking=True)
        if self._events[w] is not None:
            self._events[w].record()
            self._used[w] = True
        self.bytes_last = n * 4
        return {name: self.dev[a:a + m] for name, (a, m) in self._views.items()}
