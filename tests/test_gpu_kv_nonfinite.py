"""Scores that are NaN or infinite, by every column of a key tile and in every kernel: a NaN or +inf score makes its
row NaN (as the softmax's definition does), a score of -inf hides its key, and no other row changes by a bit."""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_kv import Setup

pytestmark = pytest.mark.gpu


def same(a, b):
    return torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


def kinds(lngram, s, q):
    return [(0, 0, lambda: lngram.kv_attend(s.cache, q)), (40, 3, lambda: lngram.kv_attend(s.cache, q, window=40, sinks=3)),
            (0, 0, lambda: lngram.kv_prefix_attend(s.cache, q, s.prefix_table, s.prefix))]


@pytest.mark.parametrize("dtype, dim, fill", [("bf16", 64, "nan"), ("f16", 128, "nan"), ("bf16", 64, "inf"), ("f16", 128, "inf"),
                                              ("bf16", 64, "huge"), ("bf16", 128, "huge")])  # 2^130 is beyond fp32
@pytest.mark.parametrize("n, ctx", [(2, 130), (150, 0)])
def test_one_bad_key_in_every_column(lngram, dtype, dim, fill, n, ctx):
    """Keys of head 1 alone: the rows that see one are NaN in head 1's group, everything else keeps its bits."""
    s = Setup(lngram, [ctx, 5], [n, n], 8, 2, dim, 16, dtype, prefix=70).fill()
    q = s.normal(*s.lead, 8, dim)
    q[..., 0] = 2.0 ** 65 if fill == "huge" else 1.0
    if fill == "huge":
        s.cache.k[..., 0] = 0.0
    runs = kinds(lngram, s, q)
    clean = [f() for _, _, f in runs]
    assert all(torch.isfinite(x).all() for x in clean)
    bad = {"nan": math.nan, "inf": math.inf, "huge": 2.0 ** 65}[fill]
    places = torch.arange(ctx, ctx + n, device="cuda")
    for j in range(66):
        page, slot = s.table[0, j // 16].long(), j % 16
        old = s.cache.k[page, 1, slot, 0].clone()
        s.cache.k[page, 1, slot, 0] = bad
        for (window, sinks, f), a in zip(runs, clean):
            got = f()
            sees = places >= j
            if window:
                sees &= (j > places - window) | (j < sinks)
            assert torch.isnan(got[0, sees][:, 4:]).all(), (j, window)
            assert same(got[0, ~sees], a[0, ~sees]) and same(got[0, :, :4], a[0, :, :4]) and same(got[1], a[1]), (j, window)
        s.cache.k[page, 1, slot, 0] = old


@pytest.mark.parametrize("n, ctx", [(2, 130), (150, 0)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_one_bad_key_in_the_prefix(lngram, n, ctx, bad):
    s = Setup(lngram, [ctx, 5], [n, n], 8, 2, 64, 16, prefix=70).fill()
    q = s.normal(*s.lead, 8, 64)
    q[..., 0] = 1.0
    clean = lngram.kv_prefix_attend(s.cache, q, s.prefix_table, 70)
    for j in range(0, 70):
        page, slot = s.prefix_table[j // 16].long(), j % 16
        old = s.cache.k[page, 1, slot, 0].clone()
        s.cache.k[page, 1, slot, 0] = bad
        got = lngram.kv_prefix_attend(s.cache, q, s.prefix_table, 70)
        assert torch.isnan(got[:, :, 4:]).all() and same(got[:, :, :4], clean[:, :, :4]), j
        s.cache.k[page, 1, slot, 0] = old


@pytest.mark.parametrize("n, ctx", [(2, 130), (150, 0)])
def test_keys_of_score_minus_infinity_are_hidden(lngram, n, ctx):
    """As keys whose weight is too small for any format are (scores of -2^13)."""
    s = Setup(lngram, [ctx, 5], [n, n], 8, 2, 64, 16, prefix=70).fill()
    q = s.normal(*s.lead, 8, 64)
    q[..., 0] = -1.0
    runs = kinds(lngram, s, q)
    for j in list(range(1, 66, 5)) + [2, 3, 8, 9]:
        page, slot = s.table[0, j // 16].long(), j % 16
        old = s.cache.k[page, 1, slot, 0].clone()
        s.cache.k[page, 1, slot, 0] = 2.0 ** 16
        small = [f() for _, _, f in runs]
        s.cache.k[page, 1, slot, 0] = math.inf
        assert all(torch.isfinite(a).all() and same(f(), a) for (_, _, f), a in zip(runs, small)), j
        s.cache.k[page, 1, slot, 0] = old


@pytest.mark.parametrize("window, sinks", [(1, 0), (2, 0), (2, 1), (3, 0), (0, 0)])
@pytest.mark.parametrize("heads", [4, 16])
def test_nan_queries_by_position(lngram, window, sinks, heads):
    """A NaN query's row is NaN whatever columns its window leaves it, and no other row changes."""
    n = 80
    s = Setup(lngram, [0, 33], [n, n], heads, 2, 64, 16).fill()
    q = s.normal(*s.lead, heads, 64)
    clean = lngram.kv_attend(s.cache, q, window=window, sinks=sinks)
    for p in list(range(16)) + [63, 64, 79]:
        q2 = q.clone()
        q2[0, p, 1] = math.nan
        got = lngram.kv_attend(s.cache, q2, window=window, sinks=sinks)
        assert torch.isnan(got[0, p, 1]).all(), p
        got[0, p, 1] = clean[0, p, 1]
        assert same(got, clean), p
