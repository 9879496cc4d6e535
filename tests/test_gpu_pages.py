"""The page pool on the GPU against the plain one (tests/pages_model.py): tables, lengths, counts and slots equal."""

from __future__ import annotations

import random

import pytest
import torch

from tests.pages_model import Pool

pytestmark = pytest.mark.gpu


def make(lngram, batch, columns, pages, page, eight=False, layers=1, heads=2, dim=16):
    pool = lngram.PagePool.allocate(batch, columns * page, pages, heads, dim, page_size=page, device="cuda", eight=eight, layers=layers)
    return pool, Pool(batch, columns, pages, page)


def same(pool, model):
    assert pool.cache.table.tolist() == model.table
    assert pool.cache.lengths.tolist() == model.lengths
    assert pool.refs.tolist() == model.refs


@pytest.mark.parametrize("seed, groups, beams, page, columns, pages", [
    (0, 1, 1, 8, 3, 5), (1, 3, 4, 8, 6, 40), (2, 5, 2, 16, 4, 23), (3, 1, 7, 64, 5, 33), (4, 40, 16, 8, 4, 2000),
    (5, 1, 600, 8, 3, 900), (6, 2, 3, 32, 9, 70000), (7, 700, 1, 8, 20, 12000),
])
def test_random_walks(lngram, seed, groups, beams, page, columns, pages):
    rng = random.Random(seed)
    batch = groups * beams
    pool, model = make(lngram, batch, columns, pages, page)
    same(pool, model)
    for step in range(25):
        what = rng.random()
        if what < 0.35:
            n = rng.choice([1, 1, 2, page, 2 * page + 1])
            slots, served = pool.extend(n)
            want, ok, _ = model.extend([n] * batch)
            assert slots.tolist() == want and served.tolist() == ok
        elif what < 0.6:
            news = [rng.choice([0, 1, 1, 3, page, 3 * page]) for _ in range(batch)]
            lead, behind = rng.choice([0, 2]), rng.choice([0, 3])
            cu = [lead]
            for n in news:
                cu.append(cu[-1] + n)
            slots, served = pool.extend(cu=torch.tensor(cu, dtype=torch.int32, device="cuda"), max_new=3 * page, tokens=cu[-1] + behind)
            want, ok, _ = model.extend(news)
            assert slots.tolist() == [-1] * lead + [s for row in want for s in row] + [-1] * behind and served.tolist() == ok
        elif what < 0.8:
            if rng.random() < 0.3:
                most = rng.randint(0, columns * page)
                pool.truncate(most)
                model.truncate([most] * batch)
            else:
                keep = [rng.randint(-1, columns * page) for _ in range(batch)]
                pool.truncate(torch.tensor(keep, dtype=torch.int32, device="cuda"))
                model.truncate(keep)
        else:
            parents = [[rng.randrange(beams) for _ in range(beams)] for _ in range(groups)]
            pool.reorder(torch.tensor(parents, device="cuda"))
            model.reorder(parents)
        same(pool, model)
    model.check()
    assert lngram._lib.device_error() == 0


@pytest.mark.parametrize("eight, heads, dim, page", [(False, 3, 24, 16), (True, 3, 48, 16), (False, 1, 128, 64), (True, 10, 16, 8)])
def test_copies_of_shared_pages(lngram, eight, heads, dim, page):
    """Forked rows that write get copies, in every layer, of the filled slots alone; the original stays as it was."""
    pool, model = make(lngram, 3, 4, 12, page, eight, layers=3, heads=heads, dim=dim)
    for c in pool.caches:
        for t in (c.k, c.v) if not eight else (c.k.view(torch.uint8), c.v.view(torch.uint8)):
            t.copy_(torch.randint(0, 100, t.shape, device="cuda"))
        if eight:
            for e in (c.k_exp, c.v_exp):
                e.copy_(torch.randint(-9, 9, e.shape, device="cuda"))
    used = page // 2 + 1
    pool.extend(cu=torch.tensor([0, page + used, page + used, page + used + 2], dtype=torch.int32, device="cuda"), max_new=page + used)
    model.extend([page + used, 0, 2])
    parents = [[0, 0, 2]]
    pool.reorder(torch.tensor(parents, device="cuda"))
    model.reorder(parents)

    def bits(t):
        return t.view(torch.uint8).clone() if eight else t.clone()

    before = [[bits(c.k), bits(c.v)] + ([c.k_exp.clone(), c.v_exp.clone()] if eight else []) for c in pool.caches]
    pool.extend(1)
    _, _, copies = model.extend([1, 1, 1])
    same(pool, model)
    assert [c is None for c in copies] == [False, False, True]
    for c, old in zip(pool.caches, before):
        for t, o in zip((c.k, c.v), old):
            want = o.clone()
            for copy in copies:
                if copy:
                    want[copy[1], :, :copy[2]] = o[copy[0], :, :copy[2]]
            assert torch.equal(bits(t), want)
        if eight:
            for e, o in zip((c.k_exp, c.v_exp), old[2:]):
                want = o.clone()
                for copy in copies:
                    if copy:
                        want[copy[1]] = o[copy[0]]
                assert torch.equal(e, want)


def test_given_counts_and_strided_tables(lngram):
    """A server's own state: a table that is a slice of a wider one, counts that are already there."""
    wide = torch.full((4, 10), 77, dtype=torch.int32, device="cuda")
    k, v = (torch.zeros(30, 1, 8, 16, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    lengths = torch.tensor([9, 0, 16, 3], dtype=torch.int32, device="cuda")
    table = wide[:, 2:6]
    model = Pool(4, 4, 30, 8)
    model.table = [[5, 9, -1, -1], [-1] * 4, [20, 3, -1, -1], [28, -1, -1, -1]]
    model.lengths = [9, 0, 16, 3]
    model.refs = [int(p in (5, 9, 20, 3, 28)) for p in range(30)]
    table.copy_(torch.tensor(model.table, dtype=torch.int32))
    pool = lngram.PagePool(lngram.PagedKVCache(k, v, table, lengths), torch.tensor(model.refs, dtype=torch.int32, device="cuda"))
    for n in (1, 8, 2):
        slots, served = pool.extend(n)
        want, ok, _ = model.extend([n] * 4)
        assert slots.tolist() == want and served.tolist() == ok
        same(pool, model)
    pool.reorder(torch.tensor([[3, 3, 0, 1]], device="cuda"))
    model.reorder([[3, 3, 0, 1]])
    same(pool, model)
    assert (wide[:, :2] == 77).all() and (wide[:, 6:] == 77).all()


def test_wrong_books_and_parents_record_an_error(lngram):
    err = lngram._lib.device_error
    pool, model = make(lngram, 2, 3, 9, 8)
    pool.extend(9)
    model.extend([9, 9])
    err()
    pool.reorder(torch.tensor([[1, 2]], device="cuda"))    # row 1 stays as it is
    model.reorder([[1, 1]])
    assert err() == 4
    same(pool, model)
    pool.refs.zero_()
    pool.truncate(0)                                       # pages that nobody is said to hold
    assert err() == 4 and (pool.refs == 0).all() and (pool.cache.table == -1).all()
    pool.cache.lengths.copy_(torch.tensor([100, 5]))
    pool.extend(1)                                         # a length beyond the row; a last page that is none
    assert err() == 4 and pool.cache.lengths.tolist() == [-101, 6]


def test_captured(lngram):
    """A step's calls in a graph follow the device's state from replay to replay."""
    pool, model = make(lngram, 6, 5, 40, 8, eight=True)
    parents = [[0, 0, 2], [1, 2, 2]]
    on = torch.tensor(parents, device="cuda")
    keep = torch.zeros(6, dtype=torch.int32, device="cuda")
    pool.extend(3)
    pool.truncate(0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        slots, served = pool.extend(3)
        pool.reorder(on)
        pool.truncate(keep)
    for step in range(9):
        lens = [3 * step + 2 + b % 2 for b in range(6)]
        keep.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        want, ok, _ = model.extend([3] * 6)
        model.reorder(parents)
        model.truncate(lens)
        assert slots.tolist() == want and served.tolist() == ok
        same(pool, model)


@pytest.mark.parametrize("eight", [False, True])
def test_a_pool_without_pages_left(lngram, eight):
    """Sequences that get no pages are suspended: their tokens go nowhere, their rows are zero, nothing of theirs or of the
    others' is lost, and they go on when pages are there again."""
    err = lngram._lib.device_error
    pool = lngram.PagePool.allocate(3, 64, 5, 2, 32, page_size=8, device="cuda", eight=eight)
    other = (lngram.PagedKVCache8 if eight else lngram.PagedKVCache).allocate(3, 64, 2, 32, page_size=8, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)

    def rows(n):
        return [torch.randn(3, n, h, 32, generator=g, device="cuda").bfloat16() for h in (2, 2, 4)]

    err()
    k, v, q = rows(8)
    _, served = pool.extend(8)
    assert served.tolist() == [True] * 3
    other.extend(8)
    for c in (pool.cache, other):
        lngram.kv_append(c, k, v)
    # eight more for every sequence: pages for two of them are left
    k, v, q = rows(8)
    slots, served = pool.extend(8)
    assert served.tolist() == [True, True, False] and pool.cache.lengths.tolist() == [16, 16, -9] and (slots[2] == -1).all()
    other.extend(8)
    for c in (pool.cache, other):
        lngram.kv_append(c, k, v)
    assert err() == 4
    got, want = lngram.kv_attend(pool.cache, q), lngram.kv_attend(other, q)
    assert err() == 4 and torch.equal(got[:2], want[:2]) and (got[2] == 0).all()
    # the first one ends, the third is taken up again with its tokens
    pool.truncate(torch.tensor([0, 16, 16], dtype=torch.int32, device="cuda"))
    assert pool.cache.lengths.tolist() == [0, 16, 8] and int((pool.refs == 0).sum()) == 2
    slots, served = pool.extend(cu=torch.tensor([0, 0, 0, 8], dtype=torch.int32, device="cuda"), max_new=8, tokens=8)
    assert served.tolist() == [True] * 3 and pool.cache.lengths.tolist() == [0, 16, 16]
    cu = torch.tensor([0, 0, 0, 8], dtype=torch.int32, device="cuda")
    lngram.kv_append(pool.cache, k[2], v[2], cu=cu, max_new=8)
    got = lngram.kv_attend(pool.cache, q[2], cu=cu, max_new=8)
    assert torch.equal(got, want[2]) and err() == 0
