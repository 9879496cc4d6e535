"""Attention over 8-bit pages whose values' exponents lie far apart, where the page with the largest exponent adds next
to nothing: all of its slots hold zeros but one, which no token attends to.

Tolerances are those of test_gpu_kv8.py but for weights that are subnormal in fp16.  A row's reference lies at least 7
below its largest score + exponent (base 2), so that the largest weight is 2^7 at least, and a weight's rounding, 2^-25
where it is subnormal, is 2^-32 in units of the largest weight * 2^exponent.
"""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_kv8 import E4M3, LOG2E, Setup8, check_attend, half_step, power

pytestmark = pytest.mark.gpu


def want(s, q, scale):
    """(o, tolerance) in 64 bits, [tokens, heads, dim]."""
    u, group = half_step(s.dtype), s.heads // s.kv
    q = q.reshape(-1, s.heads, s.dim).double()
    outs, tols, at = [], [], 0
    for row, c, n in zip(s.table, s.ctx, s.new):
        (k, ek), (v, ev) = s.raw(row, c + n, "k"), s.raw(row, c + n, "v")
        kk = (k * power(ek)[..., None]).transpose(0, 1).repeat_interleave(group, 0)  # [heads, L, dim]
        vv = v.transpose(0, 1).repeat_interleave(group, 0)
        pv = power(ev).t().repeat_interleave(group, 0)[:, None]                     # [heads, 1, L]
        qq = q[at:at + n].transpose(0, 1)
        hidden = torch.arange(c + n, device="cuda")[None] > c + torch.arange(n, device="cuda")[:, None]
        score = (scale * qq @ kk.transpose(1, 2)).masked_fill(hidden, -math.inf)
        most = (scale * qq.abs() @ kk.abs().transpose(1, 2)).masked_fill(hidden, 0).amax(-1, keepdim=True)
        w = torch.softmax(score, -1)
        o, a = (w * pv) @ vv, (w * pv) @ vv.abs()
        ds = (s.dim + 4) * 2.0 ** -24 * most + 3 * 2.0 ** -24 * (most + 40 / LOG2E)
        tol = (1.01 * 2.0 ** -11 + 2 * (2.0 ** -16 + ds)) * a + u * o.abs()
        tol = tol + 1.01 * 2.0 ** -32 * (w * pv).amax(-1, keepdim=True) * ((~hidden).double() @ vv.abs())
        if s.dtype == torch.float16:
            tol = tol + 2.0 ** -25
        outs.append(o.transpose(0, 1))
        tols.append(tol.transpose(0, 1))
        at += n
    return torch.cat(outs), torch.cat(tols)


@pytest.mark.parametrize("gap", [18, 21, 26])
@pytest.mark.parametrize("n, page", [(1, 16), (3, 8), (3, 64), (8, 16), (40, 16), (40, 64), (150, 32)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_a_page_of_a_large_exponent_that_adds_nothing(lngram, gap, n, page, dtype):
    s = Setup8(lngram, [300, 170], [n, n], 4, 2, 64, page, dtype, seed=gap + n).fill()
    s.cache.k_exp.fill_(-6)
    s.cache.v_exp.fill_(-8)
    k, v = s.cache.k.view(torch.uint8), s.cache.v.view(torch.uint8)
    k[..., 0] = 0
    for row in s.table:
        hot = row[70 // page].long()
        s.cache.v_exp[hot] = -8 + gap
        v[hot, :, :] = 0
        v[hot, :, 70 % page] = torch.full((2, 64), 300.0, device="cuda").to(E4M3).view(torch.uint8)
        k[hot, :, 70 % page] = 0
        k[hot, :, 70 % page, 0] = torch.full((2,), -448.0, device="cuda").to(E4M3).view(torch.uint8)  # a score of -28
    q = s.normal(*s.lead, 4, 64)
    q[..., 0] = 32
    check_attend(lngram.kv_attend(s.cache, q), *want(s, q, 64 ** -0.5))
    assert lngram._lib.device_error() == 0
