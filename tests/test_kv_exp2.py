"""2^x as the tile kernel's fma pipe forms it (constants of ``csrc/exp2_poly.cuh``, the kernel's steps one by one on
the host): within 2.7e-6 of 2^x over the whole range that the kernel asks for."""

from __future__ import annotations

import ctypes as C
import subprocess
from pathlib import Path

import numpy as np

CSRC = Path(__file__).resolve().parents[1] / "lngram-decode_b200" / "csrc"

SHIM = r"""
#include <math.h>
#include <stdint.h>
#include <string.h>
#include "exp2_poly.cuh"
using namespace lng;
extern "C" void exp2_all(const float* x, float* y, int64_t n) {
  for (int64_t i = 0; i < n; ++i) {
    const float v = fmaxf(x[i], EXP2_LOW);
    volatile float t = v + EXP2_ROUND, whole = t - EXP2_ROUND;
    const float f = fmaf(whole, -1.f, v), tt = t;
    float r = fmaf(f, EXP2_C4, EXP2_C3);
    r = fmaf(r, f, EXP2_C2);
    r = fmaf(r, f, EXP2_C1);
    r = fmaf(r, f, EXP2_C0);
    uint32_t a, b;
    memcpy(&a, &r, 4);
    memcpy(&b, &tt, 4);
    a += b << 23;
    memcpy(&y[i], &a, 4);
  }
}
"""


def test_exp2_over_its_range(tmp_path):
    (tmp_path / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-ffp-contract=off", "-shared", "-fPIC", "-I", str(CSRC), "-o",
                    str(tmp_path / "shim.so"), str(tmp_path / "shim.cpp")], check=True)
    so = C.CDLL(str(tmp_path / "shim.so"))
    so.exp2_all.argtypes = [C.c_void_p, C.c_void_p, C.c_int64]

    def run(x):
        y = np.empty_like(x)
        so.exp2_all(x.ctypes.data, y.ctypes.data, x.size)
        return y

    rng = np.random.default_rng(0)
    whole = np.arange(-126, 9, dtype=np.float32)
    half = whole[:-1] + np.float32(0.5)
    x = np.concatenate([np.linspace(-126, 8, 1 << 20, dtype=np.float32), whole, half, np.nextafter(half, np.float32(-200)),
                        np.nextafter(half, np.float32(200)), rng.uniform(-1, 1, 1 << 18).astype(np.float32) * np.float32(1e-3)])
    want = np.exp2(x.astype(np.float64))
    # the fit's 2.7e-6, and fp32's roundings of five steps (2^-24 each; what stands before the last is half of it at most)
    assert np.max(np.abs(run(x) / want - 1)) <= 2.7e-6 + 3 * 2.0 ** -24
    low = np.array([-126.5, -127, -1e4, -3e38, -np.inf, np.nan], np.float32)
    got = run(low)
    assert np.all(np.abs(got / 2.0 ** -126 - 1) <= 2.7e-6 + 3 * 2.0 ** -24)
