"""The paged key/value cache on the GPU against plain implementations in 64 bits.

Tolerances.  u is half a step of the cache's type (2^-8 bf16, 2^-11 fp16 relative).
* Rotation: a cos - b sin in fp32 from an angle reduced in 64 bits and rounded to fp32 (|angle| <= pi: an error of
  2^-23 at most), sine and cosine within 2 ulp (2^-23), three fp32 roundings: below 2^-20 (|a| + |b|), then one
  rounding u |x|.
* Attention: weights are rounded to u once for the product with v (the sum keeps them unrounded), the result
  once more: u (sum p |v|) + u |o|.  Exponentials are held to 2^-16, and a score's fp32 error is at most
  (dim + 4) 2^-24 sum |q k| scale, which enters every weight and the sum: 2 (2^-16 + that) sum p |v|.
  fp16 weights below 2^-14 are subnormal: 2^-25 each, relative to a sum of at least one.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


class Setup:
    """A cache with shuffled pages; unused slots hold NaN (they must never be read into a result)."""

    def __init__(self, lngram, ctx, new, heads, kv, dim, page, dtype="bf16", seed=0, nhd=False, uniform=None, prefix=0,
                 gap=0, magnitude=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.g, self.dtype, self.page, self.kv, self.dim, self.heads = g, DT[dtype], page, kv, dim, heads
        self.ctx, self.new = list(ctx), list(new)
        self.lens = [c + n for c, n in zip(ctx, new)]
        per = max([-(-n // page) for n in self.lens] + [1])
        self.shared = -(-prefix // page)
        pages = self.shared + len(ctx) * per + 2
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        shape = (pages, page, kv, dim) if nhd else (pages, kv, page, dim)
        k, v = (torch.full(shape, math.nan, device="cuda", dtype=self.dtype) for _ in range(2))
        if nhd:
            k, v = k.transpose(1, 2), v.transpose(1, 2)
        self.table = order[self.shared:self.shared + len(ctx) * per].view(len(ctx), per).contiguous()
        self.prefix_table = order[:self.shared].contiguous()
        self.prefix = prefix
        self.lengths = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        self.cache = lngram.PagedKVCache(k, v, self.table, self.lengths)
        uniform = len(set(new)) == 1 if uniform is None else uniform
        self.tokens = sum(new)
        self.cu = None if uniform else torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
        self.lead = (len(new), new[0]) if uniform else (self.tokens + gap,)
        self.max_new = max(list(new) + [1])
        self.magnitude = magnitude

    def normal(self, *shape):
        x = torch.randn(*shape, generator=self.g, device="cuda") * self.magnitude
        return x.to(self.dtype)

    def fill(self):
        """Random keys and values in every slot that a sequence (or the prefix) holds."""
        for row, n in [(self.table[i], n) for i, n in enumerate(self.lens)] + [(self.prefix_table, self.prefix)]:
            j = torch.arange(n, device="cuda")
            for pages in (self.cache.k, self.cache.v):
                pages[row[j // self.page].long(), :, j % self.page] = self.normal(n, self.kv, self.dim)
        return self

    def keys(self, row, n):
        j = torch.arange(n, device="cuda")
        return tuple(p[row[j // self.page].long(), :, j % self.page].double().transpose(0, 1)
                     for p in (self.cache.k, self.cache.v))

    def kw(self):
        return {} if self.cu is None else dict(cu=self.cu, max_new=self.max_new)

    def want(self, q, window=0, sinks=0, scale=None):
        """(o, tolerance) in 64 bits for every token of a sequence, [tokens, heads, dim]."""
        scale = self.dim ** -0.5 if scale is None else scale
        u, group = half_step(self.dtype), self.heads // self.kv
        q = q.reshape(-1, self.heads, self.dim).double()
        pk, pv = self.keys(self.prefix_table, self.prefix) if self.prefix else (None, None)
        outs, tols, at = [], [], 0
        for row, c, n in zip(self.table, self.ctx, self.new):
            k, v = self.keys(row, c + n)
            p = c + torch.arange(n, device="cuda")[:, None]
            j = torch.arange(c + n, device="cuda")[None]
            seen = j <= p
            if window:
                seen &= (j > p - window) | (j < sinks)
            if self.prefix:
                k, v = torch.cat((pk, k), 1), torch.cat((pv, v), 1)
                seen = torch.cat((torch.ones(n, self.prefix, dtype=torch.bool, device="cuda"), seen), 1)
            kk, vv = (x.repeat_interleave(group, 0) for x in (k, v))          # [heads, L, dim]
            qq = q[at:at + n].transpose(0, 1)                                 # [heads, n, dim]
            s = scale * qq @ kk.transpose(1, 2)
            mag = (scale * qq.abs() @ kk.abs().transpose(1, 2)).masked_fill(~seen, 0)
            s = s.masked_fill(~seen, -math.inf)
            top = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_zeros(*s.shape[:2], 1)
            e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
            total = e.sum(-1, keepdim=True)
            w = e / torch.where(total == 0, 1.0, total)
            o, a = w @ vv, w @ vv.abs()
            ds = (self.dim + 4) * 2.0 ** -24 * (mag.amax(-1, keepdim=True) if mag.shape[-1] else 0.0)
            tol = (1.01 * u + 2 * (2.0 ** -16 + ds)) * a + u * o.abs() + 1e-30
            if self.dtype == torch.float16:
                tol = tol + 2.0 ** -25 * (seen.double() @ vv.abs()) + 2.0 ** -25
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
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("ctx, new, heads, kv, dim, page, rotary, far, nhd", [
    ([0], [1], 1, 1, 8, 8, 8, 0, False),
    ([5, 0, 31], [1, 1, 1], 16, 4, 64, 16, 64, 0, False),
    ([0, 3, 100, 7], [33, 1, 0, 250], 7, 1, 128, 64, 64, 10 ** 6, True),
    ([9, 90], [700, 700], 6, 3, 80, 32, 40, 2 ** 40, False),
    ([2, 1], [5, 4], 4, 2, 96, 256, 20, 12345, False),
    ([2, 1], [5, 4], 4, 2, 72, 16, 0, 0, False),
])
def test_append(lngram, dtype, interleaved, ctx, new, heads, kv, dim, page, rotary, far, nhd):
    s = Setup(lngram, ctx, new, heads, kv, dim, page, dtype, nhd=nhd)
    # slices of one fused projection
    fused = s.normal(*s.lead, heads + 2 * kv, dim)
    q, k, v = fused[..., :heads, :], fused[..., heads:heads + kv, :], fused[..., heads + kv:, :]
    half = rotary // 2
    freq = (10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))).float().cuda() if half else None
    place = torch.cat([torch.arange(c, c + n) for c, n in zip(ctx, new)]).cuda()
    positions = (place + far).view(s.lead) if far else None
    before = [s.cache.k.clone(), s.cache.v.clone()]
    q_out = lngram.kv_append(s.cache, k, v, q, positions=positions, inv_freq=freq, interleaved=interleaved, **s.kw())
    assert lngram._lib.device_error() == 0
    u = half_step(s.dtype)

    def rotated(x):
        x = x.reshape(s.tokens, -1, dim).double()
        y, tol = x.clone(), torch.zeros_like(x)
        if half:
            angle = (place + far).double()[:, None] * freq.double()
            cos, sin = angle.cos()[:, None], angle.sin()[:, None]
            i = torch.arange(half, device="cuda")
            ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            a, b = x[..., ia], x[..., ib]
            y[..., ia], y[..., ib] = a * cos - b * sin, b * cos + a * sin
            # (far positions: 2^-52 of the product p f itself, taken by both sides)
            slack = (2.0 ** -20 + far * 2.0 ** -51) * (a.abs() + b.abs())
            tol[..., ia] = u * y[..., ia].abs() + slack
            tol[..., ib] = u * y[..., ib].abs() + slack
        return y, tol

    for got, src in ((q_out, q), (None, k)):
        want, tol = rotated(src)
        if got is None:
            got = torch.cat([s.cache.k[row[j // page].long(), :, j % page] for row, c, n in zip(s.table, ctx, new)
                             for j in [torch.arange(c, c + n, device="cuda")]])
        got = got.reshape(want.shape).double()
        assert ((got - want).abs() <= tol + 2.0 ** -24 * (s.dtype == torch.float16)).all()
    mask = torch.zeros(s.cache.k.shape[0], page, dtype=torch.bool, device="cuda")
    at = 0
    for row, c, n in zip(s.table, ctx, new):
        j = torch.arange(c, c + n, device="cuda")
        assert torch.equal(s.cache.v[row[j // page].long(), :, j % page], v.reshape(s.tokens, kv, dim)[at:at + n])
        mask[row[j // page].long(), j % page] = True
        at += n
    for pages, old in zip((s.cache.k, s.cache.v), before):  # every other slot as it was
        bits = lambda x: x.transpose(1, 2)[~mask].contiguous().view(torch.int16)  # noqa: E731
        assert torch.equal(bits(pages), bits(old))


def test_append_rotates_queries_in_place_and_skips_loose_rows(lngram):
    s = Setup(lngram, [3, 8], [4, 2], 4, 2, 64, 16, uniform=False, gap=3)
    q, k, v = s.normal(*s.lead, 4, 64), s.normal(*s.lead, 2, 64), s.normal(*s.lead, 2, 64)
    freq = torch.rand(32, device="cuda")
    want = lngram.kv_append(s.cache, k, v, q, inv_freq=freq, **s.kw())
    keys = s.cache.k.clone()
    old = q.clone()
    assert lngram.kv_append(s.cache, k, v, q, inv_freq=freq, q_out=q, **s.kw()) is q
    assert torch.equal(q[:6], want[:6]) and torch.equal(q[6:], old[6:]) and not torch.equal(q[:6], old[:6])
    assert torch.equal(s.cache.k.view(torch.int16), keys.view(torch.int16))


# ---------------------------------------------------------------------------------------------- attend
SHAPES = [
    # ctx, new, heads, kv, dim, page
    ([0], [1], 1, 1, 64, 16),
    ([0], [1], 8, 8, 8, 8),
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
    ([40, 0, 1], [77, 500, 0], 14, 2, 72, 64),
    ([300], [40], 96, 1, 128, 64),
    ([9, 300], [3, 1], 128, 1, 64, 16),
    ([0], [1100], 3, 1, 64, 64),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("ctx, new, heads, kv, dim, page", SHAPES)
def test_attend(lngram, dtype, ctx, new, heads, kv, dim, page):
    s = Setup(lngram, ctx, new, heads, kv, dim, page, dtype, seed=len(ctx) + dim).fill()
    q = s.normal(*s.lead, heads, dim)
    check_attend(lngram.kv_attend(s.cache, q, **s.kw()), *s.want(q))
    assert lngram._lib.device_error() == 0


@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (7, 0), (16, 4), (64, 70), (100, 1), (128, 64), (129, 200),
                                           (1 << 30, 3)])
@pytest.mark.parametrize("ctx, new, heads, kv, dim, page", [SHAPES[4], SHAPES[5], SHAPES[8], SHAPES[11], SHAPES[15]])
def test_attend_through_a_window(lngram, window, sinks, ctx, new, heads, kv, dim, page):
    s = Setup(lngram, ctx, new, heads, kv, dim, page, "bf16", seed=window).fill()
    q = s.normal(*s.lead, heads, dim)
    want = s.want(q, window, sinks)
    # pages that no token sees any more have been given back: no page stands in the table, NaN in the slots
    for i, (c, n) in enumerate(zip(ctx, new)):
        lo = max(0, c + 1 - window) // page
        for p in range(-(-sinks // page), lo):
            s.cache.k[s.table[i, p].long()] = math.nan
            s.cache.v[s.table[i, p].long()] = math.nan
            s.table[i, p] = -1
    check_attend(lngram.kv_attend(s.cache, q, window=window, sinks=sinks, **s.kw()), *want)
    assert lngram._lib.device_error() == 0


def test_large_scores_and_scale(lngram):
    """Scores of many hundreds: the running maximum, not exp, carries them."""
    s = Setup(lngram, [700, 3], [140, 140], 4, 2, 64, 16, "bf16", magnitude=6.0).fill()
    q = s.normal(*s.lead, 4, 64)
    check_attend(lngram.kv_attend(s.cache, q, scale=0.5), *s.want(q, scale=0.5))
    q1 = q[:, :1].contiguous()
    s.new = [1, 1]
    s.ctx = [n - 1 for n in s.lens]
    check_attend(lngram.kv_attend(s.cache, q1, scale=0.5), *s.want(q1, scale=0.5))


@pytest.mark.parametrize("n", [1, 4, 40])
def test_rows_without_keys_are_zero(lngram, n):
    """Lengths shorter than the step (and zero): the tokens before the sequence's start see nothing."""
    s = Setup(lngram, [0, 0, 50], [n, n, n], 8, 2, 64, 16).fill()
    q = s.normal(*s.lead, 8, 64)
    full = lngram.kv_attend(s.cache, q)
    short = max(0, n - 3)
    s.lengths.copy_(torch.tensor([0, short, 50 + n], dtype=torch.int32))
    got = lngram.kv_attend(s.cache, q)
    assert torch.equal(got[0], torch.zeros_like(got[0])) and torch.equal(got[1, :n - short], torch.zeros_like(got[1, :n - short]))
    assert torch.isfinite(got).all() and torch.equal(got[2], full[2])
    if short:  # the last tokens are the first ones of the whole sequence, moved by n - short
        s.ctx, s.new, s.lens = [0], [short], [short]
        s.table = s.table[1:2]
        check_attend(got[1, n - short:], *s.want(q[1, n - short:]))


def test_loose_rows_stay_as_they_are(lngram):
    for new in ([2, 1, 0], [60, 1, 0]):
        s = Setup(lngram, [40, 0, 9], new, 8, 2, 64, 16, uniform=False, gap=5).fill()
        q = s.normal(*s.lead, 8, 64)
        out = torch.full_like(q, 7.0)
        lngram.kv_attend(s.cache, q, out=out, **s.kw())
        assert (out[s.tokens:] == 7).all()
        check_attend(out, *s.want(q))
        out2 = torch.full_like(q, 7.0)
        lngram.kv_prefix_attend(s.cache, q, s.prefix_table, 0, out=out2, **s.kw())
        assert (out2[s.tokens:] == 7).all()
        check_attend(out2, *s.want(q))


@pytest.mark.parametrize("n", [1, 50])
def test_strided_rows_and_transposed_pages(lngram, n):
    s = Setup(lngram, [90, 90], [n, n], 8, 4, 64, 32, nhd=True).fill()
    fused = s.normal(2, n, 5, 8, 64)
    q = fused[:, :, 2]
    out = torch.full_like(fused, 3.0)
    check_attend(lngram.kv_attend(s.cache, q, out=out[:, :, 1]), *s.want(q))
    rest = [i for i in range(5) if i != 1]
    assert (out[:, :, rest] == 3).all()
    check_attend(out[:, :, 1], *s.want(q))


# ---------------------------------------------------------------------------------------------- prefix
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("prefix, ctx, new, heads, kv, dim, page", [
    (1, [0, 0], [1, 1], 1, 1, 64, 16),
    (1000, [0, 87, 5, 30, 2], [3] * 5, 16, 4, 64, 16),
    (129, [0, 0, 700], [1] * 3, 14, 2, 128, 64),
    (2049, list(range(40)), [1] * 40, 32, 8, 128, 64),
    (640, [3, 50], [40, 1], 8, 2, 96, 32),
    (77, [0], [300], 4, 4, 80, 128),
    (0, [10, 0], [2, 2], 8, 2, 64, 16),
    (515, [1, 2, 3], [1, 1, 1], 128, 1, 64, 8),
])
def test_prefix(lngram, dtype, prefix, ctx, new, heads, kv, dim, page):
    s = Setup(lngram, ctx, new, heads, kv, dim, page, dtype, prefix=prefix, seed=prefix).fill()
    q = s.normal(*s.lead, heads, dim)
    check_attend(lngram.kv_prefix_attend(s.cache, q, s.prefix_table, prefix, **s.kw()), *s.want(q))
    assert lngram._lib.device_error() == 0


def test_prefix_with_nothing_behind_it(lngram):
    """Sequences without a key of their own (length 0) still see the whole prefix."""
    s = Setup(lngram, [0, 9], [1, 1], 8, 2, 64, 16, prefix=50).fill()
    q = s.normal(*s.lead, 8, 64)
    s.lengths[0] = 0
    got = lngram.kv_prefix_attend(s.cache, q, s.prefix_table, 50)
    k, v = s.keys(s.prefix_table, 50)
    w = torch.softmax(q[0, 0].double().view(2, 4, 64) @ k.transpose(1, 2) / 8, -1)
    assert (got[0, 0].double().view(2, 4, 64) - w @ v).abs().max() <= 3 * half_step(s.dtype) * v.abs().max()


# ------------------------------------------------------------------------- errors, graphs, streams
def test_bad_pages_and_lengths_record_an_error(lngram):
    err = lngram._lib.device_error
    for n in (1, 40):
        s = Setup(lngram, [70, 70], [n, n], 8, 2, 64, 16).fill()
        q, k = s.normal(*s.lead, 8, 64), s.normal(*s.lead, 2, 64)
        clean = lngram.kv_attend(s.cache, q)
        good = s.table.clone()
        assert err() == 0
        s.table[1, 2] = s.cache.k.shape[0]
        got = lngram.kv_attend(s.cache, q)
        assert err() == 4 and torch.equal(got[0], clean[0]) and torch.isfinite(got).all()
        s.table[1, 4:] = -3
        before = s.cache.k.clone()
        lngram.kv_append(s.cache, k, k)
        assert err() == 4
        own = s.table[0].long()
        others = torch.ones(before.shape[0], dtype=torch.bool, device="cuda")
        others[own] = False
        assert torch.equal(before[others].view(torch.int16), s.cache.k[others].view(torch.int16))
        s.table.copy_(good)
        s.fill()
        s.lengths[1] = s.cache.capacity + 9
        clean = lngram.kv_attend(s.cache, q)
        assert err() == 4 and torch.isfinite(clean[0]).all()


@pytest.mark.parametrize("n", [1, 24])
def test_captured_steps_follow_table_and_lengths(lngram, n):
    """Two captured steps over two caches, replayed in turn as the sequences grow and pages move."""
    graphs = []
    for seed in (1, 2):
        s = Setup(lngram, [5 * seed, 200], [n, n], 8, 2, 64, 16, seed=seed, prefix=100).fill()
        s.table = torch.cat((s.table, s.table.flip(0)), 1).contiguous()  # room that is not used
        s.cache = lngram.PagedKVCache(s.cache.k, s.cache.v, s.table, s.lengths)
        q = s.normal(*s.lead, 8, 64)
        run = lambda: (lngram.kv_attend(s.cache, q, window=60, sinks=2), lngram.kv_attend(s.cache, q),  # noqa: E731
                       lngram.kv_prefix_attend(s.cache, q, s.prefix_table, 100))
        run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = run()
        graphs.append((s, q, g, outs))
    for step in range(3):
        for s, q, g, outs in graphs:
            g.replay()
        for s, q, g, outs in graphs:
            prefix, s.prefix = s.prefix, 0
            check_attend(outs[0], *s.want(q, 60, 2))
            check_attend(outs[1], *s.want(q))
            s.prefix = prefix
            check_attend(outs[2], *s.want(q))
            # the sequences grow or shrink, and the first one's pages trade places
            s.ctx = [c + 3 - 2 * step for c in s.ctx]
            s.lens = [c + n for c in s.ctx]
            s.lengths.copy_(torch.tensor(s.lens, dtype=torch.int32))
            pages = -(-(5 + 8 + n) // 16)
            s.table[0, :pages] = s.table[0, :pages].flip(0)
            s.fill()
            q.copy_(s.normal(*s.lead, 8, 64))


def test_two_streams_at_once(lngram):
    runs = []
    for seed, n in ((3, 1), (4, 30)):
        s = Setup(lngram, [900, 20], [n, n], 8, 2, 128, 16, seed=seed, prefix=300).fill()
        q = s.normal(*s.lead, 8, 128)
        runs.append((s, q, torch.cuda.Stream(), []))
    torch.cuda.synchronize()
    for _ in range(5):
        for s, q, st, outs in runs:
            with torch.cuda.stream(st):
                outs.append((lngram.kv_attend(s.cache, q), lngram.kv_prefix_attend(s.cache, q, s.prefix_table, 300)))
    torch.cuda.synchronize()
    for s, q, st, outs in runs:
        both = s.want(q)
        s.prefix = 0
        alone = s.want(q)
        for a, b in outs:
            check_attend(a, *alone)
            check_attend(b, *both)


def test_results_repeat(lngram):
    s = Setup(lngram, [3000, 20, 700], [1, 1, 1], 16, 4, 64, 16, prefix=700).fill()
    q = s.normal(*s.lead, 16, 64)
    a = [(lngram.kv_attend(s.cache, q), lngram.kv_prefix_attend(s.cache, q, s.prefix_table, 700)) for _ in range(4)]
    assert all(torch.equal(x, a[0][0]) and torch.equal(y, a[0][1]) for x, y in a)


def test_offsets_past_32_bits(lngram):
    """A cache of more than 2^32 bytes a side: the last pages, in use, lie behind that."""
    page, kv, dim = 64, 8, 128
    pages = (2 ** 32 // 2) // (page * kv * dim) + 40
    k, v = (torch.empty(pages, kv, page, dim, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    s = Setup(lngram, [100, 30], [1, 1], 16, kv, dim, page)
    s.table = torch.arange(pages - s.table.numel(), pages, dtype=torch.int32, device="cuda").view(s.table.shape)
    s.cache = lngram.PagedKVCache(k, v, s.table, s.lengths)
    s.fill()
    q, kn, vn = (s.normal(2, 1, h, dim) for h in (16, kv, kv))
    lngram.kv_append(s.cache, kn, vn)
    assert torch.equal(s.cache.k[s.table[0, 1].long(), :, 100 - 64], kn[0, 0])
    check_attend(lngram.kv_attend(s.cache, q), *s.want(q))
    s40 = s.normal(2, 40, 16, dim)
    s.ctx, s.new = [61, -9], [40, 40]
    got = lngram.kv_attend(s.cache, s40)
    s.ctx, s.new, s.table = [61], [40], s.table[:1]
    check_attend(got[0], *s.want(s40[0]))


# --------------------------------------------------------------------------------- a run of them together
def test_a_decode_loop_beside_the_memory_layer(lngram):
    """A prompt and decode steps of one layer as a user's loop runs them -- attention over the paged cache and the
    memory block over its own -- equal the whole sequence's attention and memory at once."""
    B, T, steps, d, heads, kv, dim, window, sinks = 2, 37, 9, 64, 8, 2, 16, 16, 3
    torch.manual_seed(0)
    mem = lngram.LngramMemory(d, {"routes": 6, "mem_dim": 16, "kv_heads": 2, "q_heads": 4, "head_dim": 16, "ngrams": [2, 3],
                                  "bits_per_route": 4}, norm_eps=1e-5, device="cuda").eval()
    mem.module.readout_o_proj.weight.data.normal_(0, 0.1)
    total = T + steps
    h = torch.randn(B, total, d, device="cuda")
    qkv = torch.randn(B, total, heads + 2 * kv, dim, device="cuda").to(torch.bfloat16)
    freq = (10000.0 ** (-torch.arange(dim // 2, dtype=torch.float64) / (dim // 2))).float().cuda()
    cache = lngram.PagedKVCache.allocate(B, total, kv, dim, page_size=8)
    mcache = lngram.MemoryCache(mem.module, B, total)
    att, out = [], []
    for a, b in [(0, T)] + [(t, t + 1) for t in range(T, total)]:
        x = qkv[:, a:b]
        x = x.contiguous()
        q, k, v = x[:, :, :heads], x[:, :, heads:heads + kv], x[:, :, heads + kv:]
        att.append(lngram.attention_step(cache, q, k, v, inv_freq=freq, window=window, sinks=sinks))
        out.append(lngram.decode_memory_step(mem, mcache, h[:, a:b], h[:, a:b]))
        mcache.length = b
    att, out = torch.cat(att, 1), torch.cat(out, 1)
    assert cache.lengths.tolist() == [total, total]
    with torch.no_grad():
        whole = mem(h, h)
    assert (out - whole).abs().max() <= 1e-5 * whole.abs().max()
    # the whole sequence at once: append and attend in one step over a second cache
    other = lngram.PagedKVCache.allocate(B, total, kv, dim, page_size=64)
    whole = lngram.attention_step(other, qkv[:, :, :heads], qkv[:, :, heads:heads + kv], qkv[:, :, heads + kv:], inv_freq=freq,
                                  window=window, sinks=sinks)
    u = half_step(torch.bfloat16)
    s = Setup(lngram, [0, 0], [total, total], heads, kv, dim, 64)
    s.cache, s.table = other, other.table
    q = torch.empty(B, total, heads, dim, device="cuda", dtype=torch.bfloat16)
    lngram.kv_append(other, qkv[:, :, heads:heads + kv], qkv[:, :, heads + kv:], qkv[:, :, :heads], inv_freq=freq, q_out=q)
    want, tol = s.want(q, window, sinks)
    check_attend(whole, want, tol)
    check_attend(att, want, tol)
    # two drafted tokens are rejected and the cache rolls back
    cache.truncate(total - 2)
    again = lngram.attention_step(cache, *(x.contiguous() for x in (qkv[:, -2:, :heads], qkv[:, -2:, heads:heads + kv],
                                                                   qkv[:, -2:, heads + kv:])), inv_freq=freq, window=window,
                                  sinks=sinks)
    check_attend(again, want.view(B, total, heads, dim)[:, -2:].reshape(-1, heads, dim),
                 tol.view(B, total, heads, dim)[:, -2:].reshape(-1, heads, dim))
    assert u > 0 and lngram._lib.device_error() == 0


@pytest.mark.parametrize("ctx, new, heads, kv, dim", [
    ([5] * 90, [17] * 90, 8, 4, 64),                                   # several units a CTA, one row tile each
    (list(range(0, 600, 6)), [40 + i % 50 for i in range(100)], 4, 2, 128),  # ragged, two row tiles
    ([0] * 3, [900, 1, 1300], 16, 8, 64),
])
def test_many_units(lngram, ctx, new, heads, kv, dim):
    """More units of work than SMs: every CTA of the tile kernel walks several."""
    s = Setup(lngram, ctx, new, heads, kv, dim, 32, seed=len(ctx)).fill()
    q = s.normal(*s.lead, heads, dim)
    want = s.want(q)
    for _ in range(5):
        check_attend(lngram.kv_attend(s.cache, q, **s.kw()), *want)
    check_attend(lngram.kv_attend(s.cache, q, window=100, sinks=3, **s.kw()), *s.want(q, 100, 3))
    assert lngram._lib.device_error() == 0


@pytest.mark.parametrize("n", [1, 60])
def test_nan_queries_stay_nan_and_alone(lngram, n):
    """A query of NaN (a padded row, say) gives NaN for its row and head, and no other."""
    s = Setup(lngram, [300, 20], [n, n], 8, 2, 64, 16, prefix=90).fill()
    q = s.normal(*s.lead, 8, 64)
    runs = (lambda x: lngram.kv_attend(s.cache, x), lambda x: lngram.kv_prefix_attend(s.cache, x, s.prefix_table, 90))
    clean = [f(q) for f in runs]
    q2 = q.clone()
    q2[1, n // 2, 3] = math.nan
    for f, a in zip(runs, clean):
        b = f(q2)
        assert torch.isnan(b[1, n // 2, 3]).all()
        b[1, n // 2, 3] = a[1, n // 2, 3]
        assert torch.equal(a, b)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch, n, heads", [(1, 1, 8), (1, 4, 8), (1, 3, 10), (4, 2, 16), (5, 2, 16), (5, 1, 32), (80, 1, 14), (80, 4, 8)])
def test_few_rows_of_few_and_many_pairs(lngram, batch, n, heads, dim):
    """Up to 16 rows for each of 2 key heads, over both sides of every choice of kernel and share."""
    ctx = [(i * 389) % 700 for i in range(batch)] if batch > 1 else [2500]
    s = Setup(lngram, ctx, [n] * batch, heads, 2, dim, 16, "bf16", seed=batch + n).fill()
    q = s.normal(*s.lead, heads, dim)
    check_attend(lngram.kv_attend(s.cache, q, **s.kw()), *s.want(q))
    check_attend(lngram.kv_attend(s.cache, q, window=90, sinks=5, **s.kw()), *s.want(q, 90, 5))
    assert lngram._lib.device_error() == 0
