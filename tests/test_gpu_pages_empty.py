"""Page pools of no sequences."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eight", [False, True])
def test_rows_of_no_sequence_have_no_slot(lngram, eight):
    pool = lngram.PagePool.allocate(0, 64, 5, 2, 32, page_size=8, device="cuda", eight=eight)
    cu = torch.zeros(1, dtype=torch.int32, device="cuda")
    for tokens in (6, 700, 0):
        used = torch.full((tokens,), 7, dtype=torch.int64, device="cuda")  # what the allocator hands out next
        del used
        slots, served = pool.extend(cu=cu, max_new=3, tokens=tokens)
        assert slots.shape == (tokens,) and (slots == -1).all() and served.shape == (0,)
    slots, served = pool.extend(2)
    assert slots.shape == (0, 2) and served.shape == (0,)
    pool.truncate(0)
    pool.reorder(torch.zeros(0, 4, dtype=torch.int64, device="cuda"))
    assert (pool.refs == 0).all() and lngram._lib.device_error() == 0
