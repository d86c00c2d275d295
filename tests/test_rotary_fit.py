"""Where the sine and cosine coefficients of csrc/rotary.h come from (no GPU): the minimax fits are computed here by Remez
exchange and have to give the constants in the source, and the evaluation, modelled in fp32, keeps the stated error."""
import os
import re
from fractions import Fraction

import numpy as np
import pytest

SOURCE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "feather_amd", "csrc", "rotary.h")
LD = np.longdouble
PI = LD("3.14159265358979323846264338327950288")


def _constants():
    text = open(SOURCE).read()
    return {n: np.float32(v) for n, v in re.findall(r"\b(k\w+) = (-?[0-9.]+e[+-][0-9]+)f", text)}


def _solve(A, b):
    """Gaussian elimination in extended precision (numpy's solver has none)."""
    M = np.concatenate([A, b[:, None]], 1).astype(LD)
    n = len(M)
    for c in range(n):
        p = c + int(np.argmax(np.abs(M[c:, c])))
        M[[c, p]] = M[[p, c]]
        M[c] = M[c] / M[c, c]
        for r in range(n):
            if r != c:
                M[r] = M[r] - M[r, c] * M[c]
    return M[:, -1]


def _minimax(f, w, terms, top, fixed):
    """Coefficients of z^len(fixed) .. z^(terms-1) that make max |w (fixed + rest - f)| over (0, top] least."""
    k, m = len(fixed), terms - len(fixed)
    rest = lambda z: f(z) - sum((LD(c) * z ** j for j, c in enumerate(fixed)), LD(0))
    i = np.arange(m + 1)
    z = np.maximum(top / 2 * (1 - np.cos(PI * i.astype(LD) / m)), top * LD(1e-6))
    grid = (np.arange(1, 20001).astype(LD)) * (top / 20000)
    for _ in range(60):
        A = np.stack([w(z) * z ** (k + j) for j in range(m)] + [(-1.0) ** i], 1)
        c = _solve(A, w(z) * rest(z))[:m]
        e = w(grid) * (sum(c[j] * grid ** (k + j) for j in range(m)) - rest(grid))
        runs = np.split(np.arange(grid.size), np.flatnonzero(np.sign(e[1:]) != np.sign(e[:-1])) + 1)
        peaks = [r[int(np.argmax(np.abs(e[r])))] for r in runs]
        while len(peaks) > m + 1:
            peaks.pop(0 if abs(e[peaks[0]]) < abs(e[peaks[-1]]) else -1)
        assert len(peaks) == m + 1
        new = grid[peaks]
        if np.array_equal(new, z):
            break
        z = new
    return c, float(np.abs(e).max())


def _fit(f, w, terms):
    fixed, err = [], 0.0
    while len(fixed) < terms:
        c, err = _minimax(f, w, terms, (PI / 4) ** 2, fixed)
        fixed.append(np.float32(c[0]))
    return fixed, err


def test_coefficients_are_the_minimax_fits():
    r, k = np.sqrt, _constants()
    sin, e_sin = _fit(lambda z: (np.sin(r(z)) / r(z) - 1) / z, lambda z: z * r(z) / np.sin(r(z)), 3)
    cos, e_cos = _fit(lambda z: (np.cos(r(z)) - 1 + z / 2) / z ** 2, lambda z: z ** 2, 3)
    for j in range(3):
        # (the longdouble quotients near z = 0 leave the last fitted digits open: one step of fp32)
        assert abs(sin[j] - k[f"kSin{j}"]) <= np.spacing(abs(k[f"kSin{j}"])), j
        assert abs(cos[j] - k[f"kCos{j}"]) <= np.spacing(abs(k[f"kCos{j}"])), j
    assert e_sin < 2.0 ** -27.8 and e_cos < 2.0 ** -33


def test_the_parts_of_half_pi():
    """Each part is the fp32 nearest to what the parts before it leave of pi/2 (50 digits)."""
    left = Fraction("1.57079632679489661923132169163975144209858469968755")
    for j in range(3):
        part = _constants()[f"kHalfPi{j}"]
        for other in (np.nextafter(part, np.float32(-9)), np.nextafter(part, np.float32(9))):
            assert abs(left - Fraction(float(part))) < abs(left - Fraction(float(other)))
        left -= Fraction(float(part))
    assert abs(left) < 1.1e-23


@pytest.mark.parametrize("top", [0.7853, 6.3, 4096.0, 1e5])
def test_error_of_the_evaluation(top):
    """The device's operations one by one in fp32, a fused multiply-add as one rounding of the exact value."""
    k = _constants()
    fma = lambda a, b, c: (np.float64(a) * np.float64(b) + np.float64(c)).astype(np.float32)
    x = (np.random.default_rng(0).random(1000000) * top).astype(np.float32)
    n = np.rint(x * np.float32(0.636619772))
    y = fma(-n, k["kHalfPi2"], fma(-n, k["kHalfPi1"], fma(-n, k["kHalfPi0"], x)))
    z = y * y
    sp = fma(y * z, fma(z, fma(z, k["kSin2"], k["kSin1"]), k["kSin0"]), y)
    cp = fma(z, fma(z, fma(z, fma(z, k["kCos2"], k["kCos1"]), k["kCos0"]), np.float32(-0.5)), np.float32(1))
    q = n.astype(np.int64)
    s, c = np.where(q & 1, cp, sp), np.where(q & 1, sp, cp)
    s, c = np.where(q & 2, -s, s), np.where((q + 1) & 2, -c, c)
    assert np.abs(s - np.sin(x.astype(LD))).max() <= 1.25 * 2.0 ** -24
    assert np.abs(c - np.cos(x.astype(LD))).max() <= 1.25 * 2.0 ** -24
