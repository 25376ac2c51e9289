"""The integer arithmetic of the experts' kernels, restated in Python's integers and doubles and compared with the formulas it stands for."""
import math

import numpy as np
import pytest


def _divider(d, off=0):
    """(m, shift of the upper word) of norm_rows.hip's reciprocal. off: of the hardware's single-precision reciprocal, in its units."""
    l, f = (d - 1).bit_length(), np.float32
    r = (f(1) / f(d)).view(np.int32) + np.int32(off)
    r = r.view(f) * f(1 - 2.0 ** -21)
    m = int(np.ldexp(r, 31 + l))
    m += int(f((1 << (31 + l)) - m * d) * r)
    left = (1 << (31 + l)) - m * d
    assert 0 <= left < 2 * d
    return m + (left > 0) + (left > d), l - 1


def test_reciprocals_of_every_kind():
    """The smallest m with m d >= 2^(31+l), whatever the last unit of the hardware's reciprocal."""
    rng = np.random.default_rng(3)
    for d in {max(2, min(1 << 23, (1 << k) + e)) for k in range(1, 24) for e in range(-3, 4)} | set(rng.integers(2, 1 << 23, 3000).tolist()):
        for off in (-1, 0, 1):
            m, sh = _divider(d, off)
            assert m == -(-(1 << (32 + sh)) // d) and 1 << 31 <= m < 1 << 32


def test_codes_by_reciprocal():
    """sign(t) floor((254 |t| + a) / 2a) from (254 t + 257 a - [t < 0]) m >> 32 + l - 1, at every largest value up to 300, powers of two and
    their neighbours up to 2^22, random ones, and at the t around every code's border."""
    rng = np.random.default_rng(0)
    tops = set(range(1, 300)) | {min(1 << 22, max(1, (1 << k) + d)) for k in range(23) for d in (-1, 0, 1)} | set(rng.integers(1, 1 << 22, 300).tolist())
    for a in tops:
        m, sh = _divider(2 * a)
        assert 1 << 31 <= m < 1 << 32
        border = {min(a, max(0, (2 * c - 1) * a // 254 + d)) for c in range(128) for d in (-1, 0, 1)} | {0, 1, a - 1, a}
        for x in border:
            for t in (x, -x):
                u = 254 * t + 257 * a - (t < 0)
                assert 0 <= u < 1 << 31
                code = (u * m >> 32 >> sh) - 128
                want = (254 * abs(t) + a) // (2 * a)
                assert code == (want if t >= 0 else -want), (a, t)


@pytest.mark.parametrize("lo,hi", [(-128, 127), (-32768, 32767)])
def test_requant_from_the_upper_word(lo, hi):
    """clamp((acc m + 2^(s-1)) >> s) from the product's upper word, clamped before the shift by s - 32."""
    rng = np.random.default_rng(1)
    i32 = lambda v: -(1 << 31) <= v < 1 << 31                                                         # noqa: E731
    for s in range(33, 63):
        rest = s - 32
        clo, chi = max(lo << rest, -(1 << 31)), min(((hi + 1) << rest) - 1, (1 << 31) - 1)
        accs = [0, 1, -1, 1 << 30, -(1 << 30)] + rng.integers(-(1 << 30), 1 << 30, 200).tolist() + rng.integers(-5000, 5000, 50).tolist()
        ms = [0, 1, -1, (1 << 31) - 1, -(1 << 31)] + rng.integers(-(1 << 31), 1 << 31, 20).tolist()
        # products at a border of the rounding
        accs += [((2 * v + 1) << (s - 1)) // m + d for v in (lo, -1, 0, 5, hi) for m in ms if m for d in (-1, 0, 1)
                 if abs(((2 * v + 1) << (s - 1)) // m) < (1 << 30) - 1]
        for acc in accs:
            for m in ms:
                x = (acc * m >> 32) + (1 << (rest - 1))
                assert i32(x)
                assert min(max(x, clo), chi) >> rest == min(max((acc * m + (1 << (s - 1))) >> s, lo), hi), (acc, m, s)


def test_a_smaller_shift_lifted():
    """(m, s) and (m 2^(33 - s), 33) round alike."""
    rng = np.random.default_rng(2)
    for s in range(33):
        for m in (1, -3, 77, (1 << s) // 4, -((1 << s) // 4)):
            if abs(m) << (33 - s) >= 1 << 31:
                continue
            for acc in rng.integers(-(1 << 30), 1 << 30, 50).tolist() + list(range(-40, 40)):
                assert (acc * m + ((1 << s) >> 1)) >> s == (acc * (m << (33 - s)) + (1 << 32)) >> 33


def test_shares_by_doubles():
    """(e one + S / 2) / S from a quotient of doubles and one correction, at sums up to 2^41 and quotients next to whole numbers."""
    rng = np.random.default_rng(3)
    for _ in range(20000):
        one = int(rng.integers(1, 32768))
        S = int(rng.integers(1, 1 << int(rng.integers(1, 42))))
        e = int(rng.integers(0, min(S, (1 << 31) - 1) + 1))
        if rng.random() < 0.5:                                 # at a border: e one + S / 2 = v S
            e = min(max(0, (int(rng.integers(0, one + 1)) * S - S // 2) // one + int(rng.integers(-1, 2))), min(S, (1 << 31) - 1))
        num = e * one + S // 2
        q = int(float(num) / float(S))
        if q * S > num:
            q -= 1
        elif (q + 1) * S <= num:
            q += 1
        assert q == num // S
