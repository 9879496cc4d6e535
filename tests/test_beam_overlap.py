"""``beam_reorder`` refuses states whose rows meet; states side by side in one buffer pass (without a GPU they get as far
as the missing device)."""

from __future__ import annotations

import random

import pytest
import torch

from __graft_entry__ import load_package

lngram = load_package()
PARENTS = torch.zeros(2, 3, dtype=torch.int64)


def refused(*states, parents=PARENTS, **kw):
    with pytest.raises(ValueError, match="overlap"):
        lngram.beam_reorder(parents, *states, **kw)


def passes(*states, parents=PARENTS, **kw):
    with pytest.raises(RuntimeError, match="CUDA device"):
        lngram.beam_reorder(parents, *states, **kw)


def test_states_that_meet_are_refused():
    x, y = torch.zeros(6, 8, 5), torch.zeros(6, 9)
    refused(x, x)
    refused(x, y, x)
    refused(*[torch.zeros(6, 2) for _ in range(9)], x, x)  # (more than one launch's)
    refused(x, x[:, 3:5])
    refused(y[:, :5], y[:, 4:])
    refused(y.view(torch.uint8), y)
    buffer = torch.zeros(7, 4)
    refused(buffer[:6], buffer[1:])
    refused(x, x, length=1)
    flat = torch.zeros(100)
    refused(flat.as_strided((6, 3), (10, 1)), flat.as_strided((6, 3), (7, 1), 3))  # rows 3 of each


def test_states_side_by_side_pass():
    x = torch.zeros(6, 8, 5)
    passes(x)
    passes(x, x.clone())
    passes(x[:, :3], x[:, 3:])
    passes(x[:, :3], x[:, 3:], length=2)
    passes(x, x[:, 4:], length=4)  # what moves does not meet
    passes(x, x, length=0)
    both = torch.zeros(12, 4)
    passes(both[:6], both[6:])
    passes(both[::2], both[1::2])
    flat = torch.zeros(100)
    passes(flat.as_strided((6, 3), (14, 1)), flat.as_strided((6, 3), (7, 1), 3))
    passes(torch.zeros(6, 0), torch.zeros(6, 0))


def test_the_check_against_brute_force():
    """Rows of bytes of one buffer, all ways of lying there."""
    rng = random.Random(0)
    buffer = torch.zeros(400, dtype=torch.uint8)
    met = 0
    for _ in range(3000):
        groups, beams = rng.randint(1, 3), rng.randint(1, 3)
        rows, cells, states = groups * beams, [], []
        for _ in range(rng.randint(2, 3)):
            n = rng.randint(0, 6)
            stride = max(n, 1) + rng.choice([0, 1, 5, 9])
            at = rng.randint(0, 400 - rows * stride)
            states.append(buffer.as_strided((rows, n), (stride, 1), at))
            cells.append({at + r * stride + c for r in range(rows) for c in range(n)})
        meet = any(a & b for i, a in enumerate(cells) for b in cells[:i])
        met += meet
        (refused if meet else passes)(*states, parents=torch.zeros(groups, beams, dtype=torch.int64))
    assert 300 < met < 2700  # (both outcomes are well covered)
