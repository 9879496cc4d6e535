"""The device's error word: the code that was recorded first, whichever operator recorded it."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_memory import gpu_memory

pytestmark = pytest.mark.gpu


def test_the_first_code_is_reported(lngram):
    err = lngram._lib.device_error
    memory = gpu_memory(lngram, "tiny").module
    codes = torch.zeros(1, 8, 8, dtype=torch.int32, device="cuda")
    codes[0, 5, 3] = 200
    state = torch.zeros(2, 8, device="cuda")
    out_of_range = torch.tensor([[0, 2]], device="cuda")
    cache = lngram.PagedKVCache8.allocate(1, 64, 1, 64, device="cuda")
    cache.lengths.fill_(-5)
    rows = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16, device="cuda")
    records = [
        (1, lambda: memory._lookup_route_chunk(codes, None, 0, 8, None, None)),
        (4, lambda: lngram.beam_reorder(out_of_range, state)),
        (4, lambda: lngram.kv_append(cache, rows, rows)),
    ]
    with torch.no_grad():
        for first in records:
            for then in records:
                err()
                first[1]()
                then[1]()
                assert err(clear=False) == first[0]
                assert err() == first[0] and err() == 0
