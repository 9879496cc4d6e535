"""A shared prompt and its continuations as a server runs them: the prompt is appended once to pages of its own, the
continuations' tokens behind it, rotated by the positions that count the prompt.  Tolerances as in ``test_gpu_kv``."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_kv import Setup, check_attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, dim, page, P", [("bf16", 64, 16, 77), ("f16", 128, 64, 200)])
@pytest.mark.parametrize("steps", [(1, 1, 3), (30, 1, 2)])
def test_continuations_of_one_prompt(lngram, dtype, dim, page, P, steps):
    B, heads, kv, total = 3, 8, 2, sum(steps)
    s = Setup(lngram, [0] * B, [total] * B, heads, kv, dim, page, dtype, prefix=P)
    freq = (10000.0 ** (-torch.arange(dim // 2, dtype=torch.float64) / (dim // 2))).float().cuda()
    # the prompt: a cache of one sequence over the same pages
    prompt = lngram.PagedKVCache(s.cache.k, s.cache.v, s.prefix_table.view(1, -1),
                                 torch.full((1,), P, dtype=torch.int32, device="cuda"))
    pk, pv = s.normal(1, P, kv, dim), s.normal(1, P, kv, dim)
    lngram.kv_append(prompt, pk, pv, inv_freq=freq)
    q, k, v = s.normal(B, total, heads, dim), s.normal(B, total, kv, dim), s.normal(B, total, kv, dim)
    s.lengths.zero_()
    got, turned, at = [], [], 0
    for n in steps:
        s.cache.extend(n)
        x = [y[:, at:at + n].contiguous() for y in (q, k, v)]
        places = torch.arange(P + at, P + at + n, device="cuda").expand(B, n).contiguous()
        turned.append(lngram.kv_append(s.cache, x[1], x[2], x[0], positions=places, inv_freq=freq))
        got.append(lngram.kv_prefix_attend(s.cache, turned[-1], s.prefix_table, P))
        at += n
    assert lngram._lib.device_error() == 0
    got, turned = torch.cat(got, 1), torch.cat(turned, 1)
    check_attend(got, *s.want(turned))
    # the same as sequences that hold the prompt themselves: its keys, and the positions that follow by themselves
    whole = lngram.PagedKVCache.allocate(B, P + total, kv, dim, page_size=page, dtype=s.dtype)
    whole.extend(P + total)
    turned2 = lngram.kv_append(whole, torch.cat((pk.expand(B, -1, -1, -1), k), 1), torch.cat((pv.expand(B, -1, -1, -1), v), 1),
                               torch.cat((s.normal(B, P, heads, dim), q), 1), inv_freq=freq)[:, P:].contiguous()
    assert torch.equal(turned2, turned)
    check_attend(lngram.kv_attend(whole, turned2), *s.want(turned))
