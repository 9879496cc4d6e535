"""Ragged steps on an 8-bit cache whose first sequence does not begin at the first row: loose rows in front and behind,
sequences without tokens between (tolerances: test_gpu_kv8.py)."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_kv8 import Setup8, check_attend, check_pages, half_step, rotated

pytestmark = pytest.mark.gpu


def setup(lngram, ctx, new, page, front, seed):
    s = Setup8(lngram, ctx, new, 4, 2, 64, page, uniform=False, seed=seed)
    s.cu += front
    s.lead = (front + s.tokens + 2,)
    return s


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rotary", [64, 40])
@pytest.mark.parametrize("page", [8, 16, 64, 256])
@pytest.mark.parametrize("front", ["three", "past a page", "pages"])
@pytest.mark.parametrize("ctx, new", [
    ([5, 0, 31, 64], [1, 0, 1, 1]),
    ([0, 3, 0, 0, 100], [0, 33, 0, 0, 250]),
    ([255, 17, 9], [300, 0, 19]),
])
def test_append8_behind_loose_rows(lngram, interleaved, rotary, page, front, ctx, new):
    front = {"three": 3, "past a page": page + 1, "pages": 5 * page + 3}[front]
    s = setup(lngram, ctx, new, page, front, page + front).fill(ctx)
    q, k, v = s.normal(*s.lead, 4, 64), s.normal(*s.lead, 2, 64), s.normal(*s.lead, 2, 64)
    freq = (10000.0 ** (-torch.arange(rotary // 2, dtype=torch.float64) / (rotary // 2))).float().cuda()
    place = torch.cat([torch.arange(c, c + n) for c, n in zip(ctx, new)]).cuda()
    before = [[t.clone() for t in pair] for pair in ((s.cache.k, s.cache.k_exp), (s.cache.v, s.cache.v_exp))]
    out = torch.full_like(q, 7.0)
    lngram.kv_append(s.cache, k, v, q, inv_freq=freq, interleaved=interleaved, q_out=out, **s.kw())
    assert lngram._lib.device_error() == 0
    rows = slice(front, front + s.tokens)
    want, slack = rotated(q[rows], place, freq, interleaved, 64)
    assert ((out[rows].double() - want).abs() <= half_step(s.dtype) * want.abs() + slack).all()
    assert (out[:front] == 7).all() and (out[front + s.tokens:] == 7).all()
    check_pages(s, *rotated(k[rows], place, freq, interleaved, 64), "k", before[0])
    check_pages(s, *rotated(v[rows], place, None, False, 64), "v", before[1])


@pytest.mark.parametrize("page", [8, 64, 256])
@pytest.mark.parametrize("front", [3, 65, 500])
@pytest.mark.parametrize("ctx, new", [
    ([5, 0, 31, 64], [1, 0, 1, 1]),
    ([100, 3, 0, 90], [7, 0, 8, 2]),
    ([0, 3, 0, 0, 100], [0, 33, 0, 0, 250]),
    ([64 * i for i in range(40)], [i % 4 for i in range(40)]),
])
def test_attend8_behind_loose_rows(lngram, page, front, ctx, new):
    s = setup(lngram, ctx, new, page, front, page + front).fill()
    q = s.normal(*s.lead, 4, 64)
    out = torch.full_like(q, 7.0)
    lngram.kv_attend(s.cache, q, out=out, **s.kw())
    rows = slice(front, front + s.tokens)
    some = [i for i, n in enumerate(new) if n]
    s.table, s.ctx, s.new = s.table[some], [ctx[i] for i in some], [new[i] for i in some]
    check_attend(out[rows], *s.want(q[rows]))
    assert (out[:front] == 7).all() and (out[front + s.tokens:] == 7).all()
    assert lngram._lib.device_error() == 0
