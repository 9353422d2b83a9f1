"""Rows that cannot save what sharing has to save are not looked over, and no others are left out."""
import random

import numpy as np
import pytest

import cache8_tools as c8
from holon_b200.engine.batch import SharedPrefix


def test_rows_that_cannot_save_enough_are_not_looked_over(monkeypatch):
    table, _ = c8.paged([2100] * 16, 64, 16, 0, [(list(range(16)), 32)])
    args = table.numpy(), np.full(16, 2100, dtype=np.int32), 64, np.arange(16)
    assert SharedPrefix.find(*args, 15 * 2048)["saved"] == 15 * 2048
    monkeypatch.setattr(SharedPrefix, "_alike", lambda *a: pytest.fail("looked over"))
    assert SharedPrefix.find(*args, 15 * 2048 + 1) is None
    assert SharedPrefix.find(args[0][:1], args[1][:1], 64, args[3], 0) is None


def test_whatever_is_found_is_within_the_bound():
    rng = random.Random(5)
    for _ in range(300):
        n, page = rng.randint(2, 16), rng.choice((4, 16, 64))
        held, order, shared = [rng.randint(1, 40 * page) for _ in range(n)], rng.sample(range(n), n), []
        while len(order) > 1 and rng.random() < 0.8:
            rows = [order.pop() for _ in range(rng.randint(2, len(order)))]
            pages = min((held[r] - 1) // page for r in rows)
            if pages:
                shared.append((rows, pages))
        table, _ = c8.paged(held, page, n, 0, shared)
        args = table.numpy(), np.array(held, dtype=np.int32), page, np.arange(n)
        found = SharedPrefix.find(*args)
        if found is not None:
            again = SharedPrefix.find(*args, found["saved"])
            assert again is not None and all(np.array_equal(again[k], found[k]) for k in found)
