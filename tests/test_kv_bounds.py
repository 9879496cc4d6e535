"""Where the paged cache puts a step's tokens when lengths or offsets are out of range (``csrc/kv_index.cuh``
compiled for the host): every token at the key its given length, count and row say, or nowhere."""

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
extern "C" void span(const int32_t* cu, const int32_t* len, int64_t b, int64_t tokens, int32_t max_new, int32_t cap, int64_t* o) {
  SeqSpan s = seq_span(cu, len, b, tokens, max_new, cap);
  o[0] = s.first; o[1] = s.n; o[2] = s.len; o[3] = s.bad; o[4] = s.pos;
}
"""


@pytest.fixture(scope="module")
def span(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv_bounds")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", str(CSRC), "-o", str(d / "shim.so"),
                    str(d / "shim.cpp")], check=True)
    so = C.CDLL(str(d / "shim.so"))
    so.span.argtypes = [C.c_void_p, C.c_void_p, C.c_int64, C.c_int64, C.c_int32, C.c_int32, C.c_void_p]

    def call(cu, lens, b, tokens, max_new, cap):
        out = (C.c_int64 * 5)()
        so.span((C.c_int32 * len(cu))(*cu) if cu else None, (C.c_int32 * len(lens))(*lens), b, tokens, max_new, cap, out)
        return tuple(out)

    return call


def test_a_step_past_the_capacity(span):
    assert span(None, [65], 0, 1, 1, 64) == (0, 1, 0, 1, 64)      # key 64 is no key of the cache
    assert span(None, [66], 0, 4, 4, 64) == (0, 4, 0, 1, 62)      # keys 62 and 63 are, 64 and 65 are not
    assert span(None, [-1], 0, 2, 2, 64) == (0, 2, 0, 1, -3)
    assert span(None, [2 ** 31 - 1], 0, 1, 1, 64)[4] == 2 ** 31 - 2


def test_more_rows_than_max_new(span):
    # five rows, four of them taken: they stand where they would with the fifth, and see no key behind the fourth
    assert span([0, 5], [20], 0, 5, 4, 64) == (0, 4, 19, 1, 15)
    assert span([-2, 3], [20], 0, 5, 9, 64) == (0, 3, 20, 1, 17)
    assert span([3, 9], [20], 0, 5, 9, 64) == (3, 2, 16, 1, 14)


def test_every_kept_token_has_its_own_place(span):
    rng = random.Random(3)
    for _ in range(20000):
        batch, tokens, max_new, cap = rng.randint(1, 4), rng.randint(0, 20), rng.randint(1, 6), rng.choice([0, 8, 16])
        cu = [rng.randint(-4, 24) for _ in range(batch + 1)] if rng.random() < 0.7 else None
        lens = [rng.randint(-3, cap + 5) for _ in range(batch)]
        rows = tokens if cu else batch * max_new
        for b in range(batch):
            first, n, length, bad, pos = span(cu, lens, b, rows, max_new, cap)
            assert 0 <= n <= max_new and (n == 0 or 0 <= first <= first + n <= rows) and 0 <= length <= cap
            begin, end = (cu[b], cu[b + 1]) if cu else (b * max_new, (b + 1) * max_new)
            for i in range(n):
                assert pos + i == lens[b] - (end - begin) + (first + i - begin)
            fits = 0 <= lens[b] <= cap
            if not fits:
                assert bad and length == 0
            elif n and pos + n >= 0:
                assert length == pos + n <= lens[b]
