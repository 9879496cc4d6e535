"""The paged cache on the GPU when lengths, counts or offsets are out of range: no key of another place is
touched, and what attention gives is defined.  Tolerances as in ``test_gpu_kv``."""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_kv import Setup, check_attend

pytestmark = pytest.mark.gpu


def bits(x):
    return x.contiguous().view(torch.int16)


@pytest.mark.parametrize("n, over", [(1, 1), (1, 9), (4, 2), (40, 1), (40, 39), (40, 70)])
def test_append_past_the_capacity(lngram, n, over):
    """The tokens that still fit go to their keys, the others nowhere; every other slot keeps its bits."""
    s = Setup(lngram, [0, 64 - n], [n, n], 4, 2, 64, 16).fill()
    cap = s.cache.capacity
    assert cap == 64
    s.lengths[0] = cap + over
    q, k, v = s.normal(2, n, 4, 64), s.normal(2, n, 2, 64), s.normal(2, n, 2, 64)
    freq = torch.rand(32, device="cuda")
    assert lngram._lib.device_error() == 0
    want = [s.cache.k.clone(), s.cache.v.clone()]
    fits = max(0, n - over)
    for pages, x in zip(want, (k, v)):
        for b, first, m in ((0, cap + over - n, fits), (1, cap - n, n)):
            j = torch.arange(first, first + m, device="cuda")
            pages[s.table[b, j // 16].long(), :, j % 16] = x[b, :m]
    lngram.kv_append(s.cache, k, v, q)
    assert lngram._lib.device_error() == 4
    assert torch.equal(bits(s.cache.k), bits(want[0])) and torch.equal(bits(s.cache.v), bits(want[1]))
    # queries are turned by the positions that the given length says, past the capacity too
    got = lngram.kv_append(s.cache, k, v, q, inv_freq=freq)
    at = torch.arange(n, device="cuda").view(1, n) + torch.tensor([[cap + over - n], [cap - n]], device="cuda")
    same = lngram.kv_append(s.cache, k, v, q, inv_freq=freq, positions=at)
    assert torch.equal(got, same) and lngram._lib.device_error() == 4


@pytest.mark.parametrize("heads, n", [(4, 1), (8, 4), (8, 40)])
@pytest.mark.parametrize("length", [65, 64 + 300, 2 ** 31 - 1, -1, -2 ** 31])
def test_attend_with_a_length_out_of_range(lngram, heads, n, length):
    """Such a sequence has no keys of its own to see: zeros, or the prefix alone."""
    s = Setup(lngram, [64 - n, 64 - n, 64 - n], [n] * 3, heads, 2, 64, 16, prefix=40).fill()
    q = s.normal(*s.lead, heads, 64)
    runs = (lambda: lngram.kv_attend(s.cache, q), lambda: lngram.kv_attend(s.cache, q, window=20, sinks=2),
            lambda: lngram.kv_prefix_attend(s.cache, q, s.prefix_table, 40))
    clean = [f() for f in runs]
    assert lngram._lib.device_error() == 0
    s.lengths[1] = 0
    empty = [f() for f in runs]
    assert lngram._lib.device_error() == 0
    s.lengths[1] = length
    for f, a, e in zip(runs, clean, empty):
        got = f()
        assert lngram._lib.device_error() == 4
        assert torch.equal(got[0], a[0]) and torch.equal(got[2], a[2]) and torch.equal(got[1], e[1])
    assert torch.equal(empty[0][1], torch.zeros_like(empty[0][1]))


@pytest.mark.parametrize("take", [1, 4, 40])
def test_more_rows_than_max_new(lngram, take):
    """``max_new`` below a sequence's count: its first rows are taken, each at its own place."""
    new = [take + 1, take, take + 5]
    s = Setup(lngram, [15, 9, 30], new, 4, 2, 64, 16, uniform=False).fill()
    q, k, v = s.normal(*s.lead, 4, 64), s.normal(*s.lead, 2, 64), s.normal(*s.lead, 2, 64)
    kept = torch.cat([torch.arange(b, b + min(n, take), device="cuda") for b, n in zip([0, take + 1, 2 * take + 1], new)])
    whole = s.want(q)
    got = lngram.kv_attend(s.cache, q, cu=s.cu, max_new=take)
    assert lngram._lib.device_error() == 4
    check_attend(got[kept], whole[0][kept], whole[1][kept])
    want = s.cache.k.clone()
    at = 0
    for row, c, n in zip(s.table, s.ctx, new):
        j = torch.arange(c, c + min(n, take), device="cuda")
        want[row[j // 16].long(), :, j % 16] = k[at:at + min(n, take)]
        at += n
    lngram.kv_append(s.cache, k, v, cu=s.cu, max_new=take)
    assert lngram._lib.device_error() == 4 and torch.equal(bits(s.cache.k), bits(want))


def test_a_loop_that_runs_too_long_leaves_the_cache_whole(lngram):
    """Steps past the end, then the cache is cut back to its capacity: every key is what was appended there."""
    cache = lngram.PagedKVCache.allocate(1, 32, 2, 64, page_size=16)
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(3, 1, 36, 2, 64, generator=g, device="cuda").to(torch.bfloat16)
    outs = [lngram.attention_step(cache, *(y[:, t:t + 1] for y in x)) for t in range(36)]
    assert lngram._lib.device_error() == 4
    cache.truncate(32)
    j = torch.arange(32, device="cuda")
    assert torch.equal(cache.k[cache.table[0, j // 16].long(), :, j % 16], x[1, 0, :32])
    assert all((o == 0).all() for o in outs[32:]) and not any((o == 0).all() for o in outs[:32])
    assert math.isfinite(outs[31].float().sum().item())


@pytest.mark.parametrize("take", [1, 4, 40])
@pytest.mark.parametrize("ctx", [[15, 9, 30], [700, 0, 1500]])
@pytest.mark.parametrize("batch", [3, 99])
def test_rows_past_max_new_stay_as_they_are(lngram, take, ctx, batch):
    """They belong to no sequence: neither written from states that nothing has made nor from the prefix's alone."""
    new, ctx = [take + 1, take, take + 5] * (batch // 3), ctx * (batch // 3)
    s = Setup(lngram, ctx, new, 4, 2, 64, 16, uniform=False, prefix=90, gap=2).fill()
    q = s.normal(*s.lead, 4, 64)
    at = torch.cat([torch.arange(n, device="cuda") for n in new] + [torch.full((2,), take, device="cuda")])
    kept = at < take
    prefix, out = torch.full_like(q, 7.0), torch.full_like(q, 7.0)
    torch.full((64 << 20,), math.nan, device="cuda")  # what a workspace made next finds in its memory
    lngram.kv_attend(s.cache, q, cu=s.cu, max_new=take, out=out)
    lngram.kv_prefix_attend(s.cache, q, s.prefix_table, 90, cu=s.cu, max_new=take, out=prefix)
    assert lngram._lib.device_error() == 4
    assert (out[~kept] == 7).all() and (prefix[~kept] == 7).all()
    for got, n in ((prefix, 90), (out, 0)):
        s.prefix = n
        want, tol = s.want(q[:s.tokens])
        check_attend(got[kept], want[kept[:s.tokens]], tol[kept[:s.tokens]])
