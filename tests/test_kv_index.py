"""The index arithmetic of the paged cache (``csrc/kv_index.cuh``), compiled for the host and compared with
brute force over every key: spans of new tokens, visible keys, the tiles a block of queries visits, pages."""

from __future__ import annotations

import ctypes as C
import random
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "lngram-decode_b200" / "csrc"

SHIM = r"""
#include "kv_index.cuh"
using namespace lng;
extern "C" {
void span(const int32_t* cu, const int32_t* len, int64_t b, int64_t tokens, int32_t max_new, int32_t cap, int64_t* o) {
  SeqSpan s = seq_span(cu, len, b, tokens, max_new, cap);
  o[0] = s.first; o[1] = s.n; o[2] = s.len; o[3] = s.bad;
}
int visible(int32_t j, int32_t p, int32_t w, int32_t s) { return key_visible(j, p, w, s); }
int needed(int32_t p0, int32_t p1, int32_t w, int32_t s, int32_t j) { return key_needed(key_span(p0, p1, w, s), j); }
int any_(int32_t p0, int32_t p1, int32_t w, int32_t s, int32_t a, int32_t b) { return any_needed(key_span(p0, p1, w, s), a, b); }
int all_(int32_t p0, int32_t p1, int32_t w, int32_t s, int32_t a, int32_t b) { return all_needed(key_span(p0, p1, w, s), a, b); }
int allvis(int32_t a, int32_t b, int32_t p0, int32_t p1, int32_t w, int32_t s) { return all_visible(a, b, p0, p1, w, s); }
int tiles(int32_t p0, int32_t p1, int32_t w, int32_t s, int32_t bk, int32_t* out) {
  KeyTiles t = key_tiles(key_span(p0, p1, w, s), bk);
  for (int j = 0; j < t.count; ++j) out[j] = tile_index(t, j);
  return t.count;
}
int page(const int32_t* row, int32_t j, int32_t shift, int64_t pages) { return page_of(row, j, shift, pages); }
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv_index")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", str(CSRC), "-o", str(d / "shim.so"),
                    str(d / "shim.cpp")], check=True)
    so = C.CDLL(str(d / "shim.so"))
    so.span.argtypes = [C.c_void_p, C.c_void_p, C.c_int64, C.c_int64, C.c_int32, C.c_int32, C.c_void_p]
    so.page.argtypes = [C.c_void_p, C.c_int32, C.c_int32, C.c_int64]
    return so


def test_spans_stay_inside_the_rows(lib):
    rng = random.Random(1)
    for _ in range(3000):
        batch, tokens, max_new, cap = rng.randint(1, 5), rng.randint(0, 20), rng.randint(1, 6), rng.choice([0, 7, 16])
        good = rng.random() < 0.5
        cu = sorted(rng.randint(0, tokens) for _ in range(batch + 1)) if good else [rng.randint(-30, 40) for _ in range(batch + 1)]
        lens = [rng.randint(-3, cap + 3) for _ in range(batch)]
        for use_cu in (True, False):
            rows = tokens if use_cu else batch * max_new
            for b in range(batch):
                out = (C.c_int64 * 4)()
                lib.span((C.c_int32 * (batch + 1))(*cu) if use_cu else None, (C.c_int32 * batch)(*lens), b, rows, max_new, cap, out)
                first, n, length, bad = out
                assert 0 <= first and 0 <= n <= max_new and (n == 0 or first + n <= rows) and 0 <= length <= cap
                right = 0 <= lens[b] <= cap and (not use_cu or (0 <= cu[b] <= cu[b + 1] <= rows and cu[b + 1] - cu[b] <= max_new))
                assert bool(bad) == (not right)
                if right and use_cu:
                    assert (first, n, length) == (cu[b], cu[b + 1] - cu[b], lens[b])


def test_tiles_and_spans_against_every_key(lib):
    rng = random.Random(2)
    for _ in range(4000):
        length = rng.randint(0, 90)
        n = rng.randint(1, 40)
        a = rng.randint(0, n - 1)
        p0, p1 = length - n + a, length - n + rng.randint(a, n - 1)
        window = rng.choice([0, 0, 1, 2, 5, 17, 64, 200, 1 << 30])
        sinks = rng.choice([0, 0, 1, 3, 9, 40, 1 << 30])
        bk = rng.choice([4, 8, 16, 32])
        seen = {j for p in range(p0, p1 + 1) for j in range(max(p + 1, 0))
                if window == 0 or j > p - window or j < sinks}
        for p in (p0, p1):
            assert [j for j in range(100) if lib.visible(j, p, window, sinks)] == \
                [j for j in range(max(p + 1, 0)) if window == 0 or j > p - window or j < sinks]
        need = {j for j in range(128) if lib.needed(p0, p1, window, sinks, j)}
        assert need == seen
        out = (C.c_int32 * 64)()
        got = list(out[:lib.tiles(p0, p1, window, sinks, bk, out)])
        assert got == sorted({j // bk for j in seen})
        for t in range(128 // bk):
            lo, hi = t * bk, (t + 1) * bk
            inside = [j in seen for j in range(lo, hi)]
            assert bool(lib.any_(p0, p1, window, sinks, lo, hi)) == any(inside)
            if lib.all_(p0, p1, window, sinks, lo, hi):
                assert all(inside)
            every = all(j <= p and (window == 0 or j > p - window or j < sinks) for p in range(p0, p1 + 1) for j in range(lo, hi))
            if lib.allvis(lo, hi, p0, p1, window, sinks):
                assert every


def test_full_tiles_need_no_mask(lib):
    assert lib.allvis(0, 32, 31, 40, 0, 0) and not lib.allvis(0, 32, 30, 40, 0, 0)
    assert lib.allvis(32, 64, 63, 70, 39, 0) and not lib.allvis(32, 64, 63, 71, 39, 0)
    assert lib.allvis(0, 32, 100, 200, 5, 32) and not lib.allvis(0, 32, 100, 200, 5, 31)


def test_pages_out_of_the_cache_are_found(lib):
    row = (C.c_int32 * 4)(2, -1, 5, 0)
    assert [lib.page(row, j, 3, 5) for j in (0, 7, 8, 16, 31)] == [2, 2, -1, -1, 0]
