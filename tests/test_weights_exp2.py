"""The polynomial form of 2^x in the weights kernel, restated with numpy from the constants
in the source, against 64 bits."""

from __future__ import annotations

import re
from pathlib import Path

import numpy as np

SOURCE = (Path(__file__).resolve().parents[1] / "twilight-cpu-gpu-offloading_b200" / "csrc"
          / "paged_weights.cu")


def coefficients():
    body = SOURCE.read_text().split("void ex2_five(")[1].split("\n}\n")[0]
    return [float.fromhex(x) for x in re.findall(r"pair\((0x1\.[0-9a-f]+p[-+]\d+)f, \1f\)", body)]


def ex2_five(x):
    """As the kernel computes it: x rounded to a whole number by adding 1.5 * 2^23; products and
    sums rounded once (the product is exact in 64 bits)."""
    f32 = np.float32
    x = np.minimum(np.maximum(x.astype(f32), f32(-127)), f32(128))
    r = (x + f32(12582912)).astype(f32)
    f = (x - (r - f32(12582912))).astype(f32)
    p = np.full_like(x, coefficients()[0])
    for c in coefficients()[1:]:
        p = (p.astype(np.float64) * f.astype(np.float64) + np.float64(f32(c))).astype(f32)
    bits = (r.view(np.int32).astype(np.int64) << 23) + 0x3f800000
    with np.errstate(over="ignore"):
        return p * (bits & 0xffffffff).astype(np.uint32).view(f32)


def test_error_of_the_polynomial():
    """7.5e-8 of the polynomial, half a unit (2^-24) for each rounding that counts: the last two
    steps, the product with 2^n is exact; it stays below the special-function unit's 2^-22."""
    assert len(coefficients()) == 6
    x = np.concatenate([np.linspace(-126, 127, 2_000_003), np.arange(-126, 128),
                        np.arange(-126, 127) + 0.5]).astype(np.float32)
    error = np.abs(ex2_five(x).astype(np.float64) / np.exp2(x.astype(np.float64)) - 1)
    assert 1e-7 <= error.max() <= 7.5e-8 + 3 * 2.0 ** -24 <= 2.0 ** -21.9


def test_beyond_the_exponents():
    x = np.array([-126.6, -127, -200, -1e30, -np.inf], dtype=np.float32)
    assert (ex2_five(x) == 0).all()
    x = np.array([128, 129, 1e30, np.inf], dtype=np.float32)
    assert np.isinf(ex2_five(x)).all()
    assert np.isnan(ex2_five(np.array([np.nan], dtype=np.float32))).all()
