"""The plain page pool that the GPU's is checked against keeps its own books (no GPU)."""

from __future__ import annotations

import random

import pytest

from tests.pages_model import Pool


@pytest.mark.parametrize("seed", range(8))
def test_books(seed):
    rng = random.Random(seed)
    groups, beams, page = rng.choice([(1, 1), (3, 4), (5, 2), (1, 7)]) + (rng.choice([1, 4, 8]),)
    batch = groups * beams
    pool = Pool(batch, rng.randint(1, 9), rng.randint(1, 40), page)
    for _ in range(200):
        what = rng.random()
        if what < 0.5:
            slots, served, _ = pool.extend([rng.choice([0, 1, 1, 2, page, 3 * page]) for _ in range(batch)])
            given = [s for row in slots for s in row if s >= 0]
            assert len(set(given)) == len(given)  # no two tokens share a slot
        elif what < 0.75:
            pool.truncate([rng.randint(0, 12 * page) for _ in range(batch)])
        else:
            pool.reorder([[rng.randrange(beams) for _ in range(beams)] for _ in range(groups)])
        pool.check()


def test_a_shared_last_page_is_copied_and_a_refused_sequence_suspended():
    pool = Pool(2, 4, 4, 4)
    pool.extend([6, 0])
    pool.reorder([[0, 0]])
    assert pool.refs == [2, 2, 0, 0]
    slots, served, copies = pool.extend([1, 1])
    assert served == [True, True] and copies == [(1, 2, 2), (1, 3, 2)] and pool.refs == [2, 0, 1, 1]
    assert slots == [[10], [14]]
    slots, served, _ = pool.extend([1, 9])
    assert served == [True, False] and pool.lengths == [8, -8] and slots[1] == [-1] * 9
    pool.truncate([8, 7])
    assert pool.lengths == [8, 7]
