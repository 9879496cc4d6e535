"""The paged cache in 8 bits on the GPU against plain implementations in 64 bits.

Tolerances.
* A stored value: half a step of e4m3 under its page's exponent e, max(2^-4 |x|, 2^(e - 10)), of a value that rotation
  in fp32 puts within slack = 2^-20 (|a| + |b|) of the exact one (test_gpu_kv.py derives that).  Earlier keys under a
  grown exponent have been rounded twice: a second half step, which only subnormals take.
* An exponent: that of the largest value; where the largest is within its slack of 448 * 2^e, either neighbour.
* Attention: e4m3 and the scaled queries are exact in fp16, products are summed in fp32.  Weights are rounded to fp16 once:
  u_w = 2^-11 relative, or 2^-25 where they are subnormal, in units of the row's largest weight * 2^exponent; the
  result is rounded to the rows' type, u.  A score's error in base 2 is (dim + 4) 2^-24 sum |q k| scale log2(e) and three
  roundings of |score| + |exponent| <= |score| + 40, exponentials are held to 2^-16.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
E4M3 = torch.float8_e4m3fn
LOG2E = 1.4426950408889634


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def power(e):
    return torch.ldexp(torch.ones(e.shape, dtype=torch.float64, device=e.device), e.int())


class Setup8:
    """An 8-bit cache with shuffled pages; slots that no sequence holds are NaN."""

    def __init__(self, lngram, ctx, new, heads, kv, dim, page, dtype="bf16", seed=0, nhd=False, uniform=None, gap=0, spread=3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.g, self.dtype, self.page, self.kv, self.dim, self.heads = g, DT[dtype], page, kv, dim, heads
        self.ctx, self.new = list(ctx), list(new)
        self.lens = [c + n for c, n in zip(ctx, new)]
        per = max([-(-n // page) for n in self.lens] + [1])
        pages = len(ctx) * per + 2
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        shape = (pages, page, kv, dim) if nhd else (pages, kv, page, dim)
        k, v = (torch.full(shape, 0x7f, device="cuda", dtype=torch.uint8).view(E4M3) for _ in range(2))
        if nhd:
            k, v = k.transpose(1, 2), v.transpose(1, 2)
        k_exp, v_exp = (torch.randint(-7 - spread, -6 + spread, (pages, kv), generator=g, device="cuda").to(torch.int8) for _ in range(2))
        self.table = order[:len(ctx) * per].view(len(ctx), per).contiguous()
        self.lengths = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        self.cache = lngram.PagedKVCache8(k, v, k_exp, v_exp, self.table, self.lengths, dtype=self.dtype)
        uniform = len(set(new)) == 1 if uniform is None else uniform
        self.tokens = sum(new)
        self.cu = None if uniform else torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
        self.lead = (len(new), new[0]) if uniform else (self.tokens + gap,)
        self.max_new = max(list(new) + [1])

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device="cuda").to(self.dtype)

    def fill(self, lens=None):
        """Random e4m3 values in every slot that a sequence holds."""
        for row, n in zip(self.table, self.lens if lens is None else lens):
            j = torch.arange(n, device="cuda")
            for pages in (self.cache.k, self.cache.v):
                x = (torch.randn(n, self.kv, self.dim, generator=self.g, device="cuda") * 64).to(E4M3)
                pages.view(torch.uint8)[row[j // self.page].long(), :, j % self.page] = x.view(torch.uint8)
        return self

    def raw(self, row, n, which):
        """(e4m3 values, exponents) of a sequence: [n, kv, dim], [n, kv]."""
        pages, exps = (self.cache.k, self.cache.k_exp) if which == "k" else (self.cache.v, self.cache.v_exp)
        j = torch.arange(n, device="cuda")
        p = row[j // self.page].long()
        return pages.view(torch.uint8)[p, :, j % self.page].view(E4M3).double(), exps[p]

    def kw(self):
        return {} if self.cu is None else dict(cu=self.cu, max_new=self.max_new)

    def want(self, q, window=0, sinks=0, scale=None):
        """(o, tolerance) in 64 bits for every token of a sequence, [tokens, heads, dim]."""
        scale = self.dim ** -0.5 if scale is None else scale
        u, group = half_step(self.dtype), self.heads // self.kv
        q = q.reshape(-1, self.heads, self.dim).double()
        outs, tols, at = [], [], 0
        for row, c, n in zip(self.table, self.ctx, self.new):
            (k, ek), (v, ev) = self.raw(row, c + n, "k"), self.raw(row, c + n, "v")
            k = k * power(ek)[..., None]
            p = c + torch.arange(n, device="cuda")[:, None]
            j = torch.arange(c + n, device="cuda")[None]
            seen = j <= p
            if window:
                seen &= (j > p - window) | (j < sinks)
            kk, vv = (x.transpose(0, 1).repeat_interleave(group, 0) for x in (k, v))      # [heads, L, dim]
            pv = power(ev).t().repeat_interleave(group, 0)[:, None]                      # [heads, 1, L]
            qq = q[at:at + n].transpose(0, 1)
            s = scale * qq @ kk.transpose(1, 2)
            mag = (scale * qq.abs() @ kk.abs().transpose(1, 2)).masked_fill(~seen, 0)
            s = s.masked_fill(~seen, -math.inf)
            top = s.amax(-1, keepdim=True)
            e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
            w = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
            o, a = (w * pv) @ vv, (w * pv) @ vv.abs()
            mx = mag.amax(-1, keepdim=True)
            ds = (self.dim + 4) * 2.0 ** -24 * mx + 3 * 2.0 ** -24 * (mx + 40 / LOG2E)
            tol = (1.01 * 2.0 ** -11 + 2 * (2.0 ** -16 + ds)) * a + u * o.abs() + 1e-30
            tol = tol + 1.01 * 2.0 ** -25 * (w * pv).amax(-1, keepdim=True) * (seen.double() @ vv.abs())
            if self.dtype == torch.float16:
                tol = tol + 2.0 ** -25
            outs.append(o.transpose(0, 1))
            tols.append(tol.transpose(0, 1))
            at += n
        return torch.cat(outs), torch.cat(tols)


def check_attend(got, want, tol):
    got = got.reshape(-1, *want.shape[1:])[:want.shape[0]].double()
    assert torch.isfinite(got).all()
    worst = ((got - want).abs() / tol).max().item() if want.numel() else 0.0
    assert worst <= 1.0, f"error is {worst:.2f} of the tolerance"


# ---------------------------------------------------------------------------------------------- append
def exponent(a):
    """The least e with a <= 448 * 2^e, in [-40, 40]."""
    m, e = torch.frexp(a)
    e = torch.where(m > 0.875, e - 8, e - 9)
    return torch.where(a > 0, e, -40).clamp(-40, 40)


def check_pages(s, x, tol, which, before, ctx=None, new=None):
    """The cache's keys (or values) against the exact rows x [tokens, kv, dim] within tol, page by page; every other
    slot as it was."""
    pages, exps = (s.cache.k, s.cache.k_exp) if which == "k" else (s.cache.v, s.cache.v_exp)
    old_pages, old_exps = before
    bits, old_bits = pages.contiguous().view(torch.uint8), old_pages.contiguous().view(torch.uint8)
    values, old_values = pages.double(), old_pages.double()
    written = torch.zeros(pages.shape[0], s.page, dtype=torch.bool, device="cuda")
    touched = torch.zeros(pages.shape[0], dtype=torch.bool, device="cuda")
    at = 0
    for row, c, n in zip(s.table, ctx or s.ctx, new or s.new):
        for col in range(c // s.page, -(-(c + n) // s.page) if n else 0):
            a, b = max(c, col * s.page), min(c + n, (col + 1) * s.page)
            p, first = int(row[col]), a - col * s.page
            rows, slack = x[at + a - c:at + b - c].transpose(0, 1), tol[at + a - c:at + b - c].transpose(0, 1)  # [kv, m, dim]
            fine = torch.isfinite(rows)
            most, give = torch.where(fine, rows.abs(), 0).amax((1, 2)), slack.amax((1, 2))
            lo, hi = exponent((most - give).clamp_min(0)), exponent(most + give)
            e = exps[p].int()
            if first > 0:
                lo, hi = torch.maximum(lo, old_exps[p].int()), torch.maximum(hi, old_exps[p].int())
            assert ((e >= lo) & (e <= hi)).all(), (which, col, e, lo, hi)
            f = power(e)[:, None, None]
            got = values[p][:, first:first + b - a] * f
            limit = 448 * f
            want = torch.where(fine, rows.clamp(-limit, limit), 0.0)
            near = torch.maximum(want.abs() / 16, f * 2.0 ** -10) + slack
            assert (torch.isnan(got) == ~fine).all()
            assert ((torch.where(fine, got, 0.0) - want).abs() <= near).all()
            if first > 0:
                earlier, was = values[p][:, :first] * f, old_values[p][:, :first] * power(old_exps[p])[:, None, None]
                grown = e > old_exps[p].int()
                assert torch.equal(bits[p][~grown, :first], old_bits[p][~grown, :first])
                there = ~torch.isnan(was)
                assert (torch.isnan(earlier) == ~there).all()
                # to nearest under the new exponent: exact unless subnormal
                assert (torch.where(there, (earlier - was).abs(), 0.0) <= torch.where(was.abs() < f * 2.0 ** -6, f * 2.0 ** -10, 0.0)).all()
                written[p, :first] = True
            written[p, first:first + b - a] = True
            touched[p] = True
        at += n
    keep = ~written[:, None, :, None].expand_as(bits)
    assert torch.equal(bits[keep], old_bits[keep])
    assert torch.equal(exps[~touched], old_exps[~touched])


def rotated(x, place, freq, interleaved, dim):
    """Rows [tokens, heads, dim] rotated in 64 bits, and the slack of fp32's rotation."""
    x = x.double()
    y, tol = x.clone(), torch.zeros_like(x)
    if freq is not None:
        half = freq.numel()
        angle = place.double()[:, None] * freq.double()
        cos, sin = angle.cos()[:, None], angle.sin()[:, None]
        i = torch.arange(half, device="cuda")
        ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        a, b = x[..., ia], x[..., ib]
        y[..., ia], y[..., ib] = a * cos - b * sin, b * cos + a * sin
        slack = (2.0 ** -20 + place.double().abs().max() * 2.0 ** -51) * (a.abs() + b.abs())
        tol[..., ia] = tol[..., ib] = slack
    return y, tol


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("ctx, new, heads, kv, dim, page, rotary, far, nhd", [
    ([0], [1], 1, 1, 16, 8, 16, 0, False),
    ([5, 0, 31], [1, 1, 1], 16, 4, 64, 16, 64, 0, False),
    ([0, 3, 100, 7], [33, 1, 0, 250], 7, 1, 128, 64, 64, 10 ** 6, True),
    ([9, 90], [700, 700], 6, 3, 80, 32, 40, 2 ** 40, False),
    ([2, 1], [5, 4], 4, 2, 96, 256, 20, 12345, False),
    ([250, 130], [300, 1], 2, 2, 128, 256, 128, 0, False),
    ([2, 1], [5, 4], 4, 2, 48, 16, 0, 0, False),
    ([3], [20], 40, 40, 32, 8, 32, 0, True),
])
def test_append8(lngram, dtype, interleaved, ctx, new, heads, kv, dim, page, rotary, far, nhd):
    s = Setup8(lngram, ctx, new, heads, kv, dim, page, dtype, nhd=nhd).fill(ctx)
    fused = s.normal(*s.lead, heads + 2 * kv, dim)
    q, k, v = fused[..., :heads, :], fused[..., heads:heads + kv, :], fused[..., heads + kv:, :]
    half = rotary // 2
    freq = (10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))).float().cuda() if half else None
    place = torch.cat([torch.arange(c, c + n) for c, n in zip(ctx, new)]).cuda()
    positions = (place + far).view(s.lead) if far else None
    before = [[t.clone() for t in pair] for pair in ((s.cache.k, s.cache.k_exp), (s.cache.v, s.cache.v_exp))]
    q_out = lngram.kv_append(s.cache, k, v, q, positions=positions, inv_freq=freq, interleaved=interleaved, **s.kw())
    assert lngram._lib.device_error() == 0
    qx, qt = rotated(q.reshape(s.tokens, heads, dim), place + far, freq, interleaved, dim)
    got = q_out.reshape(qx.shape).double()
    assert ((got - qx).abs() <= half_step(s.dtype) * qx.abs() + qt + 2.0 ** -24 * (dtype == "f16")).all()
    check_pages(s, *rotated(k.reshape(s.tokens, kv, dim), place + far, freq, interleaved, dim), "k", before[0])
    check_pages(s, *rotated(v.reshape(s.tokens, kv, dim), place, None, False, dim), "v", before[1])


def test_append8_grows_and_keeps_exponents(lngram):
    """Values of falling and rising size, one token after another into one page."""
    s = Setup8(lngram, [0, 0], [1, 1], 2, 2, 32, 16)
    s.lengths.zero_()
    for step, size in enumerate([1.0, 0.01, 0.0, 30.0, 1e-3, 4e4, 1.0, 1e30, 2.0]):
        x = (s.normal(2, 1, 2, 32).float() * size).to(s.dtype)
        before = [[t.clone() for t in pair] for pair in ((s.cache.k, s.cache.k_exp), (s.cache.v, s.cache.v_exp))]
        s.cache.extend(1)
        lngram.kv_append(s.cache, x, x)
        exact = x.reshape(2, 2, 32).double()
        for which, b in zip("kv", before):
            check_pages(s, exact, torch.zeros_like(exact), which, b, ctx=[step, step], new=[1, 1])
    assert s.cache.k_exp[s.table[:, 0].long()].min() == 40  # 1e30 saturates at 448 * 2^40
    assert lngram._lib.device_error() == 0


def test_append8_of_nan_and_infinities(lngram):
    s = Setup8(lngram, [3, 8], [4, 4], 2, 2, 64, 16).fill([3, 8])
    k = s.normal(2, 4, 2, 64)
    k[0, 1, 0, 5], k[0, 2, 1, 0], k[1, 0, 1, 63], k[1, 3, 0, 1] = math.nan, math.inf, -math.inf, math.nan
    before = [[t.clone() for t in pair] for pair in ((s.cache.k, s.cache.k_exp), (s.cache.v, s.cache.v_exp))]
    lngram.kv_append(s.cache, k, k)
    exact = k.reshape(8, 2, 64).double()
    for which, b in zip("kv", before):
        check_pages(s, exact, torch.zeros_like(exact), which, b)


def test_append8_rotates_queries_in_place_and_skips_loose_rows(lngram):
    s = Setup8(lngram, [3, 8], [4, 2], 4, 2, 64, 16, uniform=False, gap=3).fill([3, 8])
    q, k, v = s.normal(*s.lead, 4, 64), s.normal(*s.lead, 2, 64), s.normal(*s.lead, 2, 64)
    freq = torch.rand(32, device="cuda")
    want = lngram.kv_append(s.cache, k, v, q, inv_freq=freq, **s.kw())
    keys = s.cache.k.view(torch.uint8).clone()
    old = q.clone()
    assert lngram.kv_append(s.cache, k, v, q, inv_freq=freq, q_out=q, **s.kw()) is q
    assert torch.equal(q[:6], want[:6]) and torch.equal(q[6:], old[6:]) and not torch.equal(q[:6], old[:6])
    assert torch.equal(s.cache.k.view(torch.uint8), keys)


@pytest.mark.parametrize("nhd", [False, True])
def test_values(lngram, nhd):
    s = Setup8(lngram, [70], [1], 3, 3, 48, 32, nhd=nhd, spread=33)
    codes = torch.arange(256, device="cuda", dtype=torch.uint8).repeat(s.cache.k.numel() // 256 + 1)
    s.cache.k.copy_(codes[:s.cache.k.numel()].view(E4M3).view(s.cache.k.shape))
    k, v = s.cache.values()
    want = s.cache.k.float() * power(s.cache.k_exp)[..., None, None].float()
    assert torch.equal(k.isnan(), want.isnan()) and torch.equal(k.float().nan_to_num(), want.nan_to_num())
    assert v.isnan().all() and v.dtype == torch.bfloat16


# ---------------------------------------------------------------------------------------------- attend
SHAPES = [
    # ctx, new, heads, kv, dim, page
    ([0], [1], 1, 1, 64, 16),
    ([0], [1], 8, 8, 16, 8),
    ([63, 0, 64], [1, 1, 1], 16, 4, 64, 64),
    ([4095], [1], 16, 4, 64, 64),
    ([1, 300, 31, 2000, 77], [1] * 5, 7, 1, 128, 32),
    ([200, 33, 5], [2, 2, 2], 16, 2, 96, 16),
    ([130, 0, 7], [16, 3, 1], 3, 3, 80, 256),
    ([500, 10], [5, 5], 12, 4, 32, 8),
    ([100, 17], [16, 16], 16, 4, 64, 64),
    ([0, 0], [128, 128], 2, 2, 64, 128),
    ([0], [129], 4, 2, 128, 16),
    ([0, 5, 900], [257, 1, 300], 8, 2, 128, 32),
    ([40, 0, 1], [77, 500, 0], 14, 2, 48, 64),
    ([300], [40], 96, 1, 128, 64),
    ([9, 300], [3, 1], 128, 1, 64, 8),
    ([0], [1100], 3, 1, 64, 64),
    (list(range(0, 400, 9)), [1] * 45, 16, 4, 128, 64),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("ctx, new, heads, kv, dim, page", SHAPES)
def test_attend8(lngram, dtype, ctx, new, heads, kv, dim, page):
    s = Setup8(lngram, ctx, new, heads, kv, dim, page, dtype, seed=len(ctx) + dim).fill()
    q = s.normal(*s.lead, heads, dim)
    check_attend(lngram.kv_attend(s.cache, q, **s.kw()), *s.want(q))
    assert lngram._lib.device_error() == 0


@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (7, 0), (16, 4), (64, 70), (100, 1), (128, 64), (129, 200),
                                           (1 << 30, 3)])
@pytest.mark.parametrize("ctx, new, heads, kv, dim, page", [SHAPES[4], SHAPES[5], SHAPES[8], SHAPES[11], SHAPES[15]])
def test_attend8_through_a_window(lngram, window, sinks, ctx, new, heads, kv, dim, page):
    s = Setup8(lngram, ctx, new, heads, kv, dim, page, "bf16", seed=window).fill()
    q = s.normal(*s.lead, heads, dim)
    want = s.want(q, window, sinks)
    # pages that no token sees any more have been given back: no page stands in the table
    for i, (c, n) in enumerate(zip(ctx, new)):
        lo = max(0, c + 1 - window) // page
        for p in range(-(-sinks // page), lo):
            s.cache.k.view(torch.uint8)[s.table[i, p].long()] = 0x7f
            s.cache.v.view(torch.uint8)[s.table[i, p].long()] = 0x7f
            s.table[i, p] = -1
    check_attend(lngram.kv_attend(s.cache, q, window=window, sinks=sinks, **s.kw()), *want)
    assert lngram._lib.device_error() == 0


@pytest.mark.parametrize("n, heads", [(1, 4), (3, 4), (40, 4)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_attend8_under_far_apart_exponents(lngram, n, heads, dtype):
    """Pages whose values differ by many orders of magnitude, and queries of all sizes."""
    s = Setup8(lngram, [200, 70], [n, n], heads, 2, 64, 16, dtype, seed=3).fill()
    s.cache.v_exp.copy_(torch.randint(-20, 5, s.cache.v_exp.shape, generator=s.g, device="cuda"))
    s.cache.k_exp.copy_(torch.randint(-12, -4, s.cache.k_exp.shape, generator=s.g, device="cuda"))
    q = s.normal(*s.lead, heads, 64)
    q[0] *= 2.0 ** -12
    if dtype == "bf16":
        # (a row of large queries, its keys small: scores stay moderate)
        q[1, :, 0] *= 2.0 ** 40
        s.cache.k_exp[s.table[1].long()] = -40
    check_attend(lngram.kv_attend(s.cache, q), *s.want(q))


def test_attend8_large_scores_and_scale(lngram):
    s = Setup8(lngram, [700, 3], [140, 140], 4, 2, 64, 16, "bf16").fill()
    q = s.normal(*s.lead, 4, 64) * 24
    check_attend(lngram.kv_attend(s.cache, q, scale=0.5), *s.want(q, scale=0.5))
    q1 = q[:, :1].contiguous()
    s.new = [1, 1]
    s.ctx = [n - 1 for n in s.lens]
    check_attend(lngram.kv_attend(s.cache, q1, scale=0.5), *s.want(q1, scale=0.5))


@pytest.mark.parametrize("n", [1, 4, 40])
def test_attend8_rows_without_keys_are_zero(lngram, n):
    s = Setup8(lngram, [0, 0, 50], [n, n, n], 8, 2, 64, 16).fill()
    q = s.normal(*s.lead, 8, 64)
    full = lngram.kv_attend(s.cache, q)
    short = max(0, n - 3)
    s.lengths.copy_(torch.tensor([0, short, 50 + n], dtype=torch.int32))
    got = lngram.kv_attend(s.cache, q)
    assert torch.equal(got[0], torch.zeros_like(got[0])) and torch.equal(got[1, :n - short], torch.zeros_like(got[1, :n - short]))
    assert torch.isfinite(got).all() and torch.equal(got[2], full[2])


def test_attend8_loose_rows_stay_as_they_are(lngram):
    for new in ([2, 1, 0], [60, 1, 0]):
        s = Setup8(lngram, [40, 0, 9], new, 8, 2, 64, 16, uniform=False, gap=5).fill()
        q = s.normal(*s.lead, 8, 64)
        out = torch.full_like(q, 7.0)
        lngram.kv_attend(s.cache, q, out=out, **s.kw())
        assert (out[s.tokens:] == 7).all()
        check_attend(out, *s.want(q))


@pytest.mark.parametrize("n", [1, 50])
def test_attend8_strided_rows_and_transposed_pages(lngram, n):
    s = Setup8(lngram, [90, 90], [n, n], 8, 4, 64, 32, nhd=True).fill()
    fused = s.normal(2, n, 5, 8, 64)
    q = fused[:, :, 2]
    out = torch.full_like(fused, 3.0)
    check_attend(lngram.kv_attend(s.cache, q, out=out[:, :, 1]), *s.want(q))
    rest = [i for i in range(5) if i != 1]
    assert (out[:, :, rest] == 3).all()
    check_attend(out[:, :, 1], *s.want(q))


@pytest.mark.parametrize("n", [1, 3, 40])
def test_attend8_nonfinite_scores_make_their_rows_nan(lngram, n):
    """A NaN key makes every row that sees it NaN in all columns, and no other; so does a NaN or infinite query."""
    s = Setup8(lngram, [100, 100], [n, n], 4, 2, 64, 16, seed=5).fill()
    q = s.normal(*s.lead, 4, 64)
    clean = lngram.kv_attend(s.cache, q)
    s.cache.k.view(torch.uint8)[s.table[0, 2].long(), 1, 3, 7] = 0x7f  # key 35 of sequence 0, key head 1
    if n > 1:
        q[1, n - 1, 0, 9] = math.nan
    got = lngram.kv_attend(s.cache, q)
    want_nan = torch.zeros(2, n, 4, dtype=torch.bool, device="cuda")
    want_nan[0, :, 2:] = True
    if n > 1:
        want_nan[1, n - 1, 0] = True
    assert torch.equal(got.isnan().all(-1), want_nan) and torch.equal(got.isnan().any(-1), want_nan)
    assert torch.equal(got[~want_nan], clean[~want_nan])


@pytest.mark.parametrize("n", [1, 3, 40])
def test_bad_pages_and_lengths_record_an_error(lngram, n):
    err = lngram._lib.device_error
    s = Setup8(lngram, [100, 60], [n, n], 4, 2, 64, 16, seed=6).fill()
    q, k = s.normal(*s.lead, 4, 64), s.normal(*s.lead, 2, 64)
    good = lngram.kv_attend(s.cache, q)
    err()
    s.table[0, 2] = 10 ** 6
    got = lngram.kv_attend(s.cache, q)
    assert err() == 4 and torch.isfinite(got).all() and torch.equal(got[1], good[1])
    before = [t.view(torch.uint8).clone() for t in (s.cache.k, s.cache.v)]
    s.table[0, 100 // 16:] = -1
    s.lengths[1] = s.cache.capacity + n + 5
    lngram.kv_append(s.cache, k, k)
    assert err() == 4
    for t, b in zip((s.cache.k, s.cache.v), before):
        assert torch.equal(t.view(torch.uint8), b)
    s.lengths[1] = -5
    got = lngram.kv_attend(s.cache, q)
    assert err() == 4 and (got[1] == 0).all()
    lngram.kv_append(s.cache, k, k)
    assert err() == 4
    for t, b in zip((s.cache.k, s.cache.v), before):
        assert torch.equal(t.view(torch.uint8), b)


def test_a_step_past_the_capacity_writes_what_fits(lngram):
    err = lngram._lib.device_error
    err()
    s = Setup8(lngram, [10], [22], 2, 2, 32, 16).fill([10])   # two pages: 32 keys
    k = s.normal(1, 25, 2, 32)
    s.lengths[0] = 35
    before = [[t.clone() for t in pair] for pair in ((s.cache.k, s.cache.k_exp), (s.cache.v, s.cache.v_exp))]
    lngram.kv_append(s.cache, k, k)
    assert err() == 4
    exact = k[0, :22].double()
    for which, b in zip("kv", before):
        check_pages(s, exact, torch.zeros_like(exact), which, b, ctx=[10], new=[22])


def test_attention_step_in_a_graph_and_on_another_stream(lngram):
    """Steps of a captured graph follow the lengths; what another stream runs at the same time does not meet them."""
    s = Setup8(lngram, [33, 5], [1, 1], 8, 2, 64, 16, seed=8).fill([33, 5])
    s.lengths.copy_(torch.tensor([33, 5], dtype=torch.int32))
    per = s.table.shape[1]
    q, k, v = s.normal(2, 1, 8, 64), s.normal(2, 1, 2, 64), s.normal(2, 1, 2, 64)
    freq = torch.rand(32, device="cuda")
    state = [t.clone() for t in (s.cache.k.view(torch.uint8), s.cache.v.view(torch.uint8), s.cache.k_exp, s.cache.v_exp, s.lengths)]

    def restore():
        for t, b in zip((s.cache.k.view(torch.uint8), s.cache.v.view(torch.uint8), s.cache.k_exp, s.cache.v_exp, s.lengths), state):
            t.copy_(b)

    want = [lngram.attention_step(s.cache, q, k, v, inv_freq=freq).clone() for _ in range(per * 16 - 34)]
    restore()
    lngram.attention_step(s.cache, q, k, v, inv_freq=freq)
    restore()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = lngram.attention_step(s.cache, q, k, v, inv_freq=freq)
    restore()
    other = Setup8(lngram, [300] * 8, [1] * 8, 8, 2, 64, 16, seed=9).fill()
    oq = other.normal(8, 1, 8, 64)
    owant = lngram.kv_attend(other.cache, oq)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for w in want:
        with torch.cuda.stream(side):
            got = lngram.kv_attend(other.cache, oq)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w) and torch.equal(got, owant)


@pytest.mark.parametrize("window, sinks", [(0, 0), (70, 3), (500, 0), (129, 200)])
@pytest.mark.parametrize("ctx, new, heads, kv, dim, page", [
    ([1000, 37, 0, 2000], [16, 16, 16, 16], 16, 4, 64, 64),
    ([1000, 37, 0, 700], [16, 9, 20, 1], 16, 4, 48, 16),
    ([300], [128], 1, 1, 64, 128),
    ([77 * i for i in range(20)], [5] * 20, 32, 4, 32, 8),
    ([64 * i + 60 for i in range(90)], [7] * 90, 8, 2, 64, 32),
    ([190, 255, 256, 257], [1, 1, 1, 1], 128, 1, 16, 32),
])
def test_attend8_of_up_to_a_row_tile(lngram, window, sinks, ctx, new, heads, kv, dim, page):
    """Rows that fill a row tile at most: between the few rows of a decode step and the many of a prompt."""
    s = Setup8(lngram, ctx, new, heads, kv, dim, page, "f16", seed=len(ctx)).fill()
    q = s.normal(*s.lead, heads, dim)
    for max_len in (None, max(s.lens)):
        check_attend(lngram.kv_attend(s.cache, q, window=window, sinks=sinks, max_len=max_len, **s.kw()), *s.want(q, window, sinks))
    assert lngram._lib.device_error() == 0


@pytest.mark.parametrize("rows", [1, 3, 8, 9, 16, 17, 31, 32, 33, 64])
@pytest.mark.parametrize("dim, batch", [(64, 40), (128, 40), (64, 2), (128, 2)])
def test_attend8_by_rows_a_key_head(lngram, rows, dim, batch):
    """Every count of rows that is handled in a way of its own, many pairs and few."""
    heads, new = (rows, 1) if rows < 10 or rows % 2 else (rows // 2, 2)
    s = Setup8(lngram, [(97 * i) % 611 for i in range(batch)], [new] * batch, heads * 4, 4, dim, 32, "bf16", seed=rows).fill()
    q = s.normal(*s.lead, heads * 4, dim)
    check_attend(lngram.kv_attend(s.cache, q), *s.want(q))


def test_offsets_past_32_bits_and_strided_exponents(lngram):
    """Pages beyond 4 GB of keys, exponents in columns of a wider tensor: append, attend and values in the last pages."""
    pages, heads, page, dim = 70000, 8, 64, 128
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    k, v = (torch.zeros(pages, heads, page, dim, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
    wide = torch.full((pages, 40), 77, dtype=torch.int8, device="cuda")
    k_exp, v_exp = wide[:, 3:11], wide[:, 20:28]
    table = torch.tensor([[pages - 1, pages - 3, 2], [pages - 2, 65540, pages - 5]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([130, 190], dtype=torch.int32, device="cuda")
    cache = lngram.PagedKVCache8(k, v, k_exp, v_exp, table, lengths)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = [torch.randn(320, heads, dim, generator=g, device="cuda").bfloat16() for _ in range(2)]
    cu = torch.tensor([0, 130, 320], dtype=torch.int32, device="cuda")
    lngram.kv_append(cache, *x, cu=cu, max_new=190)
    for pages_, exps, rows in ((k, k_exp, x[0]), (v, v_exp, x[1])):
        for b, (at, n) in enumerate(((0, 130), (130, 190))):
            j = torch.arange(n, device="cuda")
            p = table[b][j // page].long()
            got = pages_.view(torch.uint8)[p, :, j % page].view(E4M3).double() * power(exps[p])[..., None]
            want = rows[at:at + n].double()
            assert ((got - want).abs() <= torch.maximum(want.abs() / 16, power(exps[p])[..., None] * 2.0 ** -10)).all()
    assert (wide[:, :3] == 77).all() and (wide[:, 11:20] == 77).all() and (wide[:, 28:] == 77).all()
    s = Setup8.__new__(Setup8)
    s.cache, s.table, s.page, s.kv, s.dim, s.heads, s.dtype = cache, table, page, heads, dim, 16, torch.bfloat16
    for new in ([1, 1], [40, 40]):
        s.ctx, s.new = [n - m for n, m in zip((130, 190), new)], new
        q = torch.randn(2, new[0], 16, dim, generator=g, device="cuda").bfloat16()
        check_attend(lngram.kv_attend(cache, q), *s.want(q))
    del s
    values = cache.values()[0]
    assert torch.equal(values[pages - 1].double(), k[pages - 1].double() * power(k_exp[pages - 1])[:, None, None])
    assert lngram._lib.device_error() == 0


def test_two_caches_appended_to_at_once(lngram):
    """Steps on two streams: what one writes and returns is what it would alone."""
    setups = [Setup8(lngram, [100 * i + 7, 3], [70, 70], 8, 2, 64, 16, seed=i).fill([100 * i + 7, 3]) for i in range(2)]
    rows = [(s.normal(2, 70, 2, 64), s.normal(2, 70, 2, 64), s.normal(2, 70, 8, 64)) for s in setups]
    freq = torch.rand(32, device="cuda")
    keep = [(s.cache.k.view(torch.uint8).clone(), s.cache.k_exp.clone()) for s in setups]

    def step(s, r):
        q = lngram.kv_append(s.cache, *r, inv_freq=freq)
        return q, lngram.kv_attend(s.cache, q)

    want = [[t.clone() for t in step(s, r)] + [s.cache.k.view(torch.uint8).clone()] for s, r in zip(setups, rows)]
    streams = [torch.cuda.Stream() for _ in setups]
    for _ in range(10):
        for s, (k, e) in zip(setups, keep):
            s.cache.k.view(torch.uint8).copy_(k)
            s.cache.k_exp.copy_(e)
        torch.cuda.synchronize()
        got = []
        for s, r, stream in zip(setups, rows, streams):
            with torch.cuda.stream(stream):
                got.append(step(s, r))
        torch.cuda.synchronize()
        for s, g, w in zip(setups, got, want):
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1]) and torch.equal(s.cache.k.view(torch.uint8), w[2])
