"""Calls of the experts' operators at the ends of their arguments' ranges, and with numbers on the device that leave theirs. Every result is
an integer, so every comparison is exact."""
import subprocess
from pathlib import Path

import numpy as np
import pytest

from expert_cases import Rows, act_lut, device, flat
from oracle import experts as oe

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
