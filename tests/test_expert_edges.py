"""Calls of the experts' operators at the ends of their arguments' ranges, and with numbers on the device that leave theirs. Every result is
an integer, so every comparison is exact."""
import subprocess
from pathlib import Path

import numpy as np
import pytest

from expert_cases import Rows, act_lut, device, flat
from oracle import experts as oe
from test_expert_ops import route_case

gpu = pytest.mark.gpu
CSRC = Path(__file__).resolve().parents[1] / "anvil-compiler_amd" / "csrc"


# ------------------------------------------------------------------------------------ multipliers and shifts

def test_lifted_multipliers_stand_for_what_they_were(tmp_path):
    """lift_shift of the kernels' header, compiled for the host, at every shift and the ends of int32: the pair it leaves is the same number, and
    m 2^-s with the same half."""
    ms = sorted({v for k in range(32) for d in (-1, 0, 1) for v in ((1 << k) + d, -(1 << k) + d) if -(1 << 31) <= v < 1 << 31})
    src = tmp_path / "lift.hip"
    src.write_text('#include <cstdio>\n#include "experts.h"\nint main() {\n  long long m;\n  int s;\n'
                   '  while (scanf("%lld %d", &m, &s) == 2) {\n    int a = (int)m, b = s;\n    anvil::lift_shift(a, b);\n    printf("%d %d\\n", a, b);\n  }\n}\n')
    exe = tmp_path / "lift"
    subprocess.run(["hipcc", "-std=c++17", "--offload-host-only", "-O1", f"-I{CSRC}", f"-I{CSRC.parents[1] / 'include'}", str(src), "-o", str(exe)],
                   check=True, capture_output=True)
    pairs = [(m, s) for m in ms for s in range(63)]
    out = subprocess.run([str(exe)], input="\n".join(f"{m} {s}" for m, s in pairs), capture_output=True, text=True, check=True).stdout.split("\n")
    for (m, s), line in zip(pairs, out):
        a, b = map(int, line.split())
        assert b >= s and a == m << (b - s) and (b == s or b == 33), (m, s, a, b)
        if 2 <= s < 33 and -(1 << 31) <= m << (33 - s) < 1 << 31:
            assert b == 33, (m, s)


ENDS = [(m, s) for m in (-(1 << 31), (1 << 31) - 1, -(1 << 30), 1 << 30) for s in (0, 1, 2, 31, 62)]


@gpu
@pytest.mark.parametrize("cols", [5, 64, 77])
@pytest.mark.parametrize("mult,shift", ENDS)
def test_sums_at_the_ends_of_the_multiplier(cols, mult, shift):
    dev, rng = device(), np.random.default_rng(cols)
    Y, slot, weight = rng.integers(-128, 128, (40, cols)), rng.integers(0, 40, (20, 2)), rng.integers(-3, 4, (20, 2))
    want = oe.combine(Y, slot, weight, mult, shift, None, 0, 0, 0, "i8")
    dY, out, ds, dw = Rows(dev, Y, "i8"), Rows(dev, np.zeros((20, cols), int), "i8"), flat(dev, slot, "i32"), flat(dev, weight, "i16")
    dev.expert_combine(dY.ptr, dY.ld, 40, ds.ptr, dw.ptr, 20, 2, cols, mult, shift, None, "i8", 0, 0, 0, 0, out.ptr, "i8", out.ld)
    dev.sync()
    assert shift > 2 or {-128, 127} <= set(np.unique(want).tolist())
    out.expect(want, f"{mult} >> {shift}")


# few rows straight from memory, tiles of 64 and of 128 rows, tiles at any alignment
SIZES = [([3, 5], 40, 64), ([130, 0, 61, 200, 64, 1, 150, 65, 63], 640, 1024), ([150] * 32, 1280, 2048), ([130, 70], 70, 50)]


@gpu
@pytest.mark.parametrize("counts,N,K", SIZES, ids=["few", "64 rows", "128 rows", "any"])
@pytest.mark.parametrize("kind,dtype", [("plain", "i8"), ("plain", "i16"), ("table", "i8"), ("gated", "i8")])
def test_products_at_the_ends_of_the_multiplier(counts, N, K, kind, dtype):
    dev, rng, E, n = device(), np.random.default_rng(K), len(counts), sum(counts)
    A, B, starts = rng.integers(-128, 128, (n, K)), rng.integers(-128, 128, (2, E, N, K), dtype=np.int8), np.r_[0, np.cumsum(counts)]
    lut = None if kind == "plain" else act_lut()
    gated = kind == "gated"
    dA, dB, dB2 = Rows(dev, A, "i8"), *(Rows(dev, b.reshape(-1, K), "i8") for b in B)
    dt, dl, out = flat(dev, starts, "i32"), flat(dev, act_lut(), "i8"), Rows(dev, np.zeros((n, N), int), dtype)
    for mult, shift in ((-(1 << 31), 0), ((1 << 31) - 1, 0), (-(1 << 31), 1), (-(1 << 31), 2), (-(1 << 31), 62)):
        each = flat(dev, np.full(E, mult), "i32")
        want = oe.gemm(np.zeros((n, N)), A, None, None, B[0], B[1] if gated else None, starts, [mult] * E, shift, [mult] * E, shift, lut, 13, 9, dtype)
        for ptr in (None, each.ptr):
            dev.expert_gemm(dA.ptr, dA.ld, n, None, None, dB.ptr, dB2.ptr if gated else None, K, N * K, dt.ptr, E, n, N, K, out.ptr, out.ld, dtype,
                            mults=ptr, mult=mult, shift=shift, mults2=ptr, mult2=mult, shift2=shift, lut=dl.ptr if lut is not None else None,
                            mult3=13, shift3=9)
            dev.sync()
            out.expect(want, f"{mult} >> {shift}")


# ------------------------------------------------------------------------------------------- the router's weights

def test_shares_by_a_reciprocal_in_single_precision():
    """The router's (e one + S / 2) / S as its kernel takes it: num and S rounded to single precision, the hardware's reciprocal with its last unit
    off either way, their product cut off, one step by the remainder. The quotient before that step is off by at most 4 roundings of 2^-23 of
    at most 32767.5, 1/64, so it is the right one or next to it. Sums up to 2^41 (1024 experts of 2^31 - 1), and quotients at whole numbers."""
    rng, f, n = np.random.default_rng(5), np.float32, 400000
    one = np.where(rng.random(n) < 0.5, 32767, rng.integers(1, 32768, n))
    S = np.maximum(1, (2.0 ** rng.uniform(0, 41, n)).astype(np.int64) + rng.integers(-2, 3, n))
    S[:200] = np.r_[np.arange(1, 101), (1 << 41) - np.arange(1024, 1124)]
    most = np.minimum(S, (1 << 31) - 1)
    e = (rng.random(n) * (most + 1)).astype(np.int64)
    near = np.clip((rng.integers(0, 1 << 15, n) % (one + 1) * S - S // 2) // one + rng.integers(-1, 2, n), 0, most)     # e one + S / 2 at a multiple of S
    e = np.where(rng.random(n) < 0.6, near, np.where(rng.random(n) < 0.1, most, e))
    num = e * one + S // 2
    assert num.max() < 1 << 47
    for off in (-1, 0, 1):
        r = ((f(1) / S.astype(f)).view(np.int32) + np.int32(off)).view(f)
        q = (num.astype(f) * r).astype(np.int64)
        assert np.abs(q - num // S).max() <= 1
        left = num - q * S
        q += np.where(left < 0, -1, np.where(left >= S, 1, 0))
        assert np.array_equal(q, num // S) and q.max() <= 32767
    assert (num % S == 0).sum() > 1000 and (num % S == S - 1).sum() > 1000


@gpu
@pytest.mark.parametrize("experts", [896, 960, 1000, 1024])
def test_route_where_one_workgroup_no_longer_holds_the_counts(experts):
    """A row of counts a wave and two more, and the pairs, in 60 KiB: up to 12 rows of 1024 experts, 13 of 960, 13 of 1000 with one choice each and
    12 with 32, 15 and 14 of 896."""
    for rows in range(11, 18):
        for top in (1, 32):
            route_case(rows, experts, top, seed=rows, live=0.9, pad=1)


# ----------------------------------------------------------------------------------- numbers out of their range

@gpu
@pytest.mark.parametrize("cols", [15, 16, 17, 64])
@pytest.mark.parametrize("R", [None, "i16"])
def test_slots_of_no_positions_are_reported(cols, R):
    """Y has no rows: a slot of -1 is none, every other one is out of range, adds nothing and is reported."""
    dev, rng = device(), np.random.default_rng(cols)
    res = None if R is None else rng.integers(-3000, 3000, (9, cols))
    want = np.zeros((9, cols), int) if R is None else oe.rq(res * 256, 1, 8)
    dR, out = None if R is None else Rows(dev, res, R), Rows(dev, np.ones((9, cols), int), R or "i8")
    dw = flat(dev, np.full((9, 5), 7), "i16")
    for at, bad in ((None, -1), (0, 0), (44, -2), (22, 2 ** 31 - 1), (7, -(2 ** 31))):
        slot = np.full(45, -1)
        if at is not None:
            slot[at] = bad
        ds = flat(dev, slot, "i32")
        dev.expert_combine(None, cols, 0, ds.ptr, dw.ptr, 9, 5, cols, 3, 4, dR and dR.ptr, R or "i8", cols, 256, 9, 8, out.ptr, R or "i8", cols)
        if at is not None:
            with pytest.raises(ValueError, match="slot"):
                dev.sync()
        dev.sync()
        out.expect(want, f"slot {bad}")


def _products(starts, rows, N, K, kind, call, seed=0, experts_mult=None, unaligned=False, oracle=True):
    """(result before, the oracle's rows of each expert alone, the device's result) of a product whose starts need not ascend; call(dev, args) runs it."""
    dev, rng, E = device(), np.random.default_rng(seed), len(starts) - 1
    A, B = rng.integers(-128, 128, (rows, K)), rng.integers(-128, 128, (2, E, N, K), dtype=np.int8)
    scale, mults, shift = rng.integers(1000, 32768, rows), rng.integers(200, 900, E), 31
    lut = None if kind == "plain" else act_lut()
    before, alone = rng.integers(-100, 100, (rows, N)), {}
    for e in range(E):
        lo, hi = starts[e], starts[e + 1]
        if oracle and 0 <= lo <= hi <= rows:
            one = slice(e, e + 1)
            alone[e] = oe.gemm(np.zeros((rows, N)), A, None, scale, B[0][one], B[1][one] if kind == "gated" else None, [lo, hi], mults[one], shift,
                               mults[one], shift, lut, 13, 9, "i8")[lo:hi]
    pad = 1 if unaligned else 0
    dA, dB, dB2 = Rows(dev, A, "i8", pad), *(Rows(dev, b.reshape(-1, K), "i8", pad) for b in B)
    out, ds, dt, dl = Rows(dev, before, "i8", 5), flat(dev, scale, "i16"), flat(dev, starts, "i32"), flat(dev, act_lut(), "i8")
    given = mults if experts_mult is None else experts_mult(mults)
    dm, dm2 = flat(dev, given, "i32"), flat(dev, mults, "i32")
    call(dev, dict(A=dA.ptr, lda=dA.ld, rows_a=rows, row=None, scale=ds.ptr, B=dB.ptr, B2=dB2.ptr if kind == "gated" else None, ldb=dB.ld, sb=N * dB.ld,
                   starts=dt.ptr, experts=E, rows=rows, N=N, K=K, Cp=out.ptr, ldc=out.ld, out_dtype="i8", mults=dm.ptr, mults2=dm2.ptr,
                   shift=shift, shift2=shift, lut=None if lut is None else dl.ptr, mult3=13, shift3=9))
    return before, alone, out


def _reported(dev, args):
    dev.expert_gemm(**args)
    with pytest.raises(ValueError, match="expert"):
        dev.sync()
    dev.sync()


def _either(starts, before, alone, out):
    """Each element is that of an expert whose rows are there, or what it was; nothing around the rows is written."""
    got, count = out.get(), np.zeros(len(before), int)
    right = np.zeros(before.shape, bool)
    for e, v in alone.items():
        at = slice(starts[e], starts[e + 1])
        count[at] += 1
        right[at] |= got[at] == v
    right[count == 0] = got[count == 0] == before[count == 0]
    assert right.all(), np.argwhere(~right)[:5]
    out.expect(got, "around the rows")
    return count


# columns, depth, alignment: few rows, tiles of 64 x 128, tiles of 64 x 64 at any alignment
FORMS = [(64, 64, False), (1024, 1024, False), (1000, 1001, True)]


@gpu
@pytest.mark.parametrize("N,K,unaligned", FORMS, ids=["few", "tiles", "any"])
@pytest.mark.parametrize("kind", ["plain", "gated"])
@pytest.mark.parametrize("starts,rows", [([0, 5, 3, 9], 9), ([0, 4, 8, 99], 9), ([-1, 4, 8, 9], 9), ([0, 10, 10, 10], 9), ([0, 100, 90, 100], 100),
                                         ([0, 300, 300, 200, 500, 2 ** 31 - 1, 500], 500), ([-(2 ** 31), 0, 40, 30, 64], 64)], ids=str)
def test_starts_out_of_range_write_what_the_other_experts_have(starts, rows, N, K, unaligned, kind):
    before, alone, out = _products(starts, rows, N, K, kind, _reported, unaligned=unaligned)
    count = _either(starts, before, alone, out)
    assert len(alone) < len(starts) - 1 and (count.max() == 2) == (starts in ([0, 5, 3, 9], [0, 100, 90, 100], [0, 300, 300, 200, 500, 2 ** 31 - 1, 500],
                                                                              [-(2 ** 31), 0, 40, 30, 64]))


@gpu
@pytest.mark.parametrize("N,K,unaligned", FORMS, ids=["few", "tiles", "any"])
@pytest.mark.parametrize("experts", [3, 9, 129, 1023])
def test_starts_that_count_more_tiles_than_a_call_has_write_nothing(experts, N, K, unaligned):
    """Up and down again: half of the experts have all rows each. 1100 rows are 17 to 35 whole tiles, and one more an expert at most."""
    rows = 1100
    starts = [0 if e % 2 == 0 else rows for e in range(experts + 1)]
    N, K = (N, K) if experts < 100 else (N // 4, K // 4)
    before, _, out = _products(starts, rows, N, K, "plain", _reported, unaligned=unaligned, oracle=False)
    out.expect(before)


@gpu
@pytest.mark.parametrize("N,K,unaligned", FORMS, ids=["few", "tiles", "any"])
@pytest.mark.parametrize("kind", ["plain", "gated"])
@pytest.mark.parametrize("bad", [32768, -32768, 2 ** 31 - 1, -(2 ** 31)])
def test_multipliers_out_of_range_leave_their_experts_rows(bad, N, K, unaligned, kind):
    starts = [0, 30, 93, 100, 190]
    before, alone, out = _products(starts, 200, N, K, kind, _reported, unaligned=unaligned, experts_mult=lambda m: np.where(np.arange(4) == 1, bad, m))
    want = before.copy()
    for e, v in alone.items():
        if e != 1:
            want[starts[e]:starts[e + 1]] = v
    out.expect(want)
