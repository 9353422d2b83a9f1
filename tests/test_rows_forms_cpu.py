"""Which form of the kernel for one-token rows a step takes."""
import types

import pytest
import torch

from holon_b200.kernels.cuda import CudaKernels


class Rooms(CudaKernels):
    """The table's decisions for a GPU of 148 SMs that holds `room[few]` CTAs of the kernel each."""

    def __init__(self, room):
        self.device, self._splits, self.sms = torch.device("cpu"), {}, 148
        self.lib = types.SimpleNamespace(hb_attention_rows_capacity=lambda kv8, few, dim, group, s: room[few] if s == 1 else 148 * room[0] // s)


@pytest.mark.parametrize("room,few", [((2, 4), 1), ((2, 3), 1), ((1, 2), 1), ((1, 1), 0), ((3, 3), 0)])
def test_the_form_for_few_keys_is_for_sms_that_hold_more_of_it(room, few):
    k = Rooms(room)
    assert k._row_splits(1, 64, 32, 8, 128, 256, 0, False)[:2] == (1, few)
    assert k._row_splits(1, 64, 32, 8, 128, 4096, 0, False)[1] == 0                     # (not few)
    assert k._row_splits(1, 2, 32, 8, 128, 256, 0, False)[1] == 0                       # (all of them run at once)


def test_the_longest_rows_start_first_where_that_pays():
    """Ranking the rows costs every CTA the square of their number: 1,024 short rows took 16 times as long with it as without."""
    k = Rooms((2, 4))
    order = lambda rows, longest: k._row_splits(1, rows, 32, 8, 128, longest, 0, False)[2]     # noqa: E731
    assert [order(rows, 4096) for rows in (8, 64, 72)] == [0, 1, 1]
    assert [order(rows, longest) for rows in (80, 256, 512, 1024) for longest in (300, 1000, 4096)] == [0] * 12
