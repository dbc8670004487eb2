"""The polynomial form of 2^x in the chunk kernel, restated with numpy from the constants
in the source, against 64 bits."""

from __future__ import annotations

import re
from pathlib import Path

import numpy as np

SOURCE = (Path(__file__).resolve().parents[1] / "twilight-cpu-gpu-offloading_b200" / "csrc"
          / "tensor.cuh")


def coefficients():
    body = SOURCE.read_text().split("void ex2_fma(")[1].split("\n}\n")[0]
    return [float.fromhex(x) for x in re.findall(r"pair\((0x1\.[0-9a-f]+p-\d+)f, \1f\)", body)]


def fma(a, b, c):
    """32-bit a * b + c, rounded once (the product is exact in 64 bits; rounding the sum to 64
    bits first changes no more than the last bit now and then)."""
    return (a.astype(np.float64) * b.astype(np.float64) + c.astype(np.float64)).astype(np.float32)


def ex2_fma(x):
    """As the kernel computes it: x rounded to a whole number by adding 1.5 * 2^23."""
    f32 = np.float32
    x = np.maximum(x.astype(f32), f32(-126))
    r = (x + f32(12582912)).astype(f32)
    n = (r - f32(12582912)).astype(f32)
    f = (x - n).astype(f32)
    p = np.full_like(x, coefficients()[0])
    for c in coefficients()[1:]:
        p = fma(p, f, np.full_like(x, c))
    bits = (r.view(np.int32).astype(np.int64) << 23) + 0x3f800000
    return p * (bits & 0xffffffff).astype(np.uint32).view(f32)


def test_error_of_the_polynomial():
    """2.65e-6 of the polynomial, half a unit (2^-24) for each rounding that counts: the last
    two steps, the product with 2^n is exact; the same again for slack."""
    assert len(coefficients()) == 5
    x = np.concatenate([np.linspace(-126, 16, 2_000_003), np.arange(-126, 17),
                        np.arange(-126, 16) + 0.5]).astype(np.float32)
    want = np.exp2(x.astype(np.float64))
    error = np.abs(ex2_fma(x).astype(np.float64) / want - 1)
    assert error.max() <= 2.65e-6 + 4 * 2.0 ** -24
    assert error.max() >= 1e-6  # the figure in the source is no overstatement


def test_below_the_smallest_exponent():
    x = np.array([-127, -200, -1e30, -np.inf], dtype=np.float32)
    got = ex2_fma(x)
    assert (np.abs(got / 2.0 ** -126 - 1) < 3e-6).all()
