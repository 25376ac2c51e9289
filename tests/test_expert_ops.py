"""The operators of an experts' feed-forward (norm with rows' own scales, router and sort, experts' products, combine) against their
numpy restatement in 64 bits. Every result is an integer, so every comparison is exact, and what lies around the results is compared too."""
import ctypes as C

import numpy as np
import pytest

from anvil_mi355x import runtime as rt
from expert_cases import Rows, act_lut, device, exp_lut, flat, roots
from oracle import experts as oe
from oracle import semantics as sem

gpu = pytest.mark.gpu
LIMIT = {"i8": 128, "i16": 32768}


# ------------------------------------------------------------------------------------- the oracle itself (CPU)

def test_codes_and_scales_stand_for_the_norm():
    """code x scale / 127 against the float norm in the table's units. With `top` a row's largest value: half a code is top / 254, the
    scale's rounding at most a half, and a table index of at least 2^8 stands for sums within half a step of its middle: 2^-9 of the
    sum, 2^-10 of its root, 2^-9 with the second order and the entry's rounding."""
    rng = np.random.default_rng(0)
    x, w = rng.integers(-3000, 3001, (50, 200)), rng.integers(1, 128, 200)
    unit, shift = 1 << 24, 15
    lut = np.rint(unit / np.sqrt(np.arange(1024) + 0.5)).astype(np.int64)
    _, codes, scale = oe.add_norm(x, None, 0, 0, 0, "i16", w, lut, 0, shift)
    want = x * w / np.sqrt((x * x).sum(1))[:, None] * (unit >> shift)
    top = np.abs(want).max(1)[:, None]
    assert scale.max() < 32767 and np.abs(codes).max() == 127
    assert np.all(np.abs(codes * scale[:, None] / 127 - want) <= top / 254 + 0.5 + top * 2.0 ** -9)


def test_codes_round_half_away_from_zero():
    for a in (1, 2, 3, 127, 254, 1000):
        x = np.arange(-a, a + 1)[None]
        _, codes, _ = oe.add_norm(x, None, 0, 0, 0, "i16", np.ones(x.size, int), roots(), 0, 0)
        want = [int(np.sign(v) * ((2 * 127 * abs(v) + a) // (2 * a))) for v in x[0].tolist()]
        assert codes[0].tolist() == want and codes[0, 0] == -127 and codes[0, -1] == 127
    assert not oe.add_norm(np.zeros((2, 5), int), None, 0, 0, 0, "i8", np.ones(5, int), roots(), 0, 0)[1].any()


def test_a_route_of_all_rows_is_a_softmax_and_a_stable_sort():
    rng = np.random.default_rng(1)
    x = rng.integers(-128, 128, (40, 9))
    lut = exp_lut(bits=14)
    expert, weight, slot, row, starts = oe.route(x, None, 9, lut, 127)
    want = sem.softmax_lut(x, lut, 127, False)
    assert np.array_equal(weight, np.take_along_axis(want, expert, 1))
    assert np.array_equal(expert, np.argsort(-x, axis=1, kind="stable"))
    assert starts.tolist() == [40 * e for e in range(10)] and np.array_equal(row, np.tile(np.arange(40), 9))
    assert np.array_equal(row[slot], np.repeat(np.arange(40), 9).reshape(40, 9))


def test_one_expert_of_every_row_is_a_qlinear():
    rng = np.random.default_rng(2)
    a, w, lut = rng.integers(-128, 128, (10, 33)), rng.integers(-128, 128, (7, 33)), act_lut()
    got = oe.gemm(np.zeros((10, 7)), a, None, None, w[None], None, [0, 10], [5], 10, None, 0, lut, 1, 0, "i8")
    assert np.array_equal(got, sem.qmatmul(a, w.T, 5, 10, lut))
    y = oe.combine(got, np.arange(10)[:, None], np.full((10, 1), 64), 1, 6, a[:, :7], 3, 2, 2, "i16")
    assert np.array_equal(y, sem.add_requant(a[:, :7], got, 3, 2, 2, "i16"))


# ------------------------------------------------------------------------------------------- refusals (CPU)

def _refused(name, struct, good, bad, error=ValueError):
    with pytest.raises(error, match=name):
        rt.library().call(name, None, C.byref(struct(*{**good, **bad}.values())))
    with pytest.raises(ValueError, match="null context"):
        rt.library().call(name, None, C.byref(struct(*good.values())))
    with pytest.raises(ValueError, match="null arguments"):
        rt.library().call(name, None, None)


MIB = 1 << 20
GOOD_NORM = dict(X=MIB, Y=2 * MIB, R=3 * MIB, x_dtype=2, y_dtype=1, r_dtype=2, ldx=64, ldy=64, ldr=64, ma=256, mb=100, shift=8, w=4 * MIB,
                 lut=5 * MIB, lut_len=1024, eps=1, lut_shift=16, H=6 * MIB, ldh=64, scale=7 * MIB, rows=4, cols=64)


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(cols=0), dict(cols=65537), dict(x_dtype=4), dict(y_dtype=0), dict(r_dtype=3),
                                 dict(Y=0), dict(R=0), dict(Y=0, R=0, r_dtype=1), dict(ldx=63), dict(ldy=1), dict(ldr=63), dict(ldh=63),
                                 dict(ldx=1 << 31), dict(lut_len=1), dict(lut_len=65537), dict(eps=-1), dict(lut_shift=32),
                                 dict(lut_shift=-1), dict(shift=32), dict(shift=-1), dict(X=0), dict(w=0), dict(lut=0), dict(H=0),
                                 dict(scale=0), dict(X=MIB + 1), dict(R=3 * MIB + 1), dict(lut=5 * MIB + 2), dict(scale=7 * MIB + 1),
                                 dict(H=MIB), dict(H=2 * MIB + 255), dict(R=MIB + 2), dict(R=2 * MIB), dict(R=MIB, ldr=65),
                                 dict(scale=3 * MIB + 500), dict(H=4 * MIB + 63), dict(scale=6 * MIB), dict(scale=5 * MIB + 4094),
                                 dict(x_dtype=1, r_dtype=2, R=MIB)], ids=str)
def test_bad_norms_are_refused(bad):
    _refused("anvil_add_norm_i8", rt.AddNorm, GOOD_NORM, bad)


def test_norm_sums_that_may_leave_int32_are_refused():
    # 2^15 ma + 2^7 mb + 2^7 <= 2^31 - 1
    top = (2 ** 31 - 1 - 128 - 128 * 100) // 32768
    for ma in (top + 1, -top - 1):
        _refused("anvil_add_norm_i8", rt.AddNorm, GOOD_NORM, dict(ma=ma), OverflowError)
    for ok in (dict(ma=top), dict(ma=-top), dict(R=MIB), dict(Y=0, R=0, ma=1 << 30), dict(H=MIB + 128, ldh=256, ldx=128),
               dict(R=2 * MIB, y_dtype=2), dict(rows=0, X=0)):
        with pytest.raises(ValueError, match="null context"):
            rt.library().call("anvil_add_norm_i8", None, C.byref(rt.AddNorm(*{**GOOD_NORM, **ok}.values())))


GOOD_ROUTE = dict(scores=MIB, ld=8, live=None, rows=16, experts=8, top=2, flags=0, lut=2 * MIB, one=127, expert=3 * MIB, weight=4 * MIB,
                  slot=5 * MIB, row=6 * MIB, starts=7 * MIB)


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(experts=0), dict(experts=1025, ld=2000), dict(top=0), dict(top=9), dict(top=33, experts=64,
                                 ld=64), dict(ld=7), dict(flags=2), dict(one=0), dict(one=32768), dict(scores=0), dict(lut=0),
                                 dict(expert=0), dict(weight=0), dict(slot=0), dict(row=0), dict(starts=0), dict(starts=0, rows=0),
                                 dict(lut=2 * MIB + 1), dict(expert=3 * MIB + 2), dict(weight=4 * MIB + 1), dict(slot=5 * MIB + 1),
                                 dict(row=6 * MIB + 2), dict(starts=7 * MIB + 2), dict(rows=1 << 29), dict(expert=MIB + 124),
                                 dict(slot=3 * MIB + 124), dict(weight=2 * MIB + 1022), dict(starts=6 * MIB), dict(live=7 * MIB),
                                 dict(row=MIB - 4)], ids=str)
def test_bad_routes_are_refused(bad):
    _refused("anvil_expert_route_i8", rt.Route, GOOD_ROUTE, bad)


GOOD_GEMM = dict(A=MIB, lda=64, row=2 * MIB, scale=3 * MIB, B=4 * MIB, B2=5 * MIB, ldb=64, sb=2048, starts=6 * MIB, rows_a=8, rows=16,
                 experts=3, N=32, K=64, mults=7 * MIB, mults2=8 * MIB, mult=1, shift=40, mult2=1, shift2=40, mult3=5, shift3=9, lut=9 * MIB,
                 C=10 * MIB, ldc=32, out_dtype=1)


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(rows=1 << 30), dict(rows_a=-1), dict(experts=0), dict(experts=1025), dict(N=0), dict(K=0),
                                 dict(N=(1 << 20) + 1, ldc=1 << 21), dict(K=65537, lda=1 << 17, ldb=1 << 17), dict(out_dtype=4),
                                 dict(out_dtype=2), dict(lut=0), dict(shift=63), dict(shift=-1), dict(shift2=63), dict(shift3=32),
                                 dict(lda=63), dict(ldb=63), dict(ldc=31), dict(lda=1 << 31), dict(sb=2047), dict(sb=-1), dict(A=0), dict(B=0),
                                 dict(starts=0), dict(C=0), dict(row=2 * MIB + 1), dict(scale=3 * MIB + 1), dict(starts=6 * MIB + 2),
                                 dict(mults=7 * MIB + 2), dict(mults2=8 * MIB + 1), dict(C=MIB), dict(C=4 * MIB + 6143),
                                 dict(C=5 * MIB), dict(C=2 * MIB + 63), dict(C=6 * MIB - 1), dict(C=9 * MIB + 255), dict(C=8 * MIB - 500),
                                 dict(rows=1 << 29, N=1 << 20, ldc=1 << 20, B2=0, mults2=0, sb=1 << 40, C=1 << 62),
                                 dict(B2=0, lut=0, out_dtype=2, C=10 * MIB + 1)], ids=str)
def test_bad_products_are_refused(bad):
    _refused("anvil_expert_gemm_i8", rt.ExpertGemm, GOOD_GEMM, bad)


def test_product_multipliers_that_may_leave_int32_are_refused():
    for bad in (dict(mults=None, mult=32768), dict(mults2=None, mult2=-32768), dict(mult3=1 << 17), dict(mult3=-(1 << 17)),
                dict(mult3=(1 << 17) - 1, shift3=31)):
        _refused("anvil_expert_gemm_i8", rt.ExpertGemm, GOOD_GEMM, bad, OverflowError)
    for ok in (dict(mults=None, mult=-32767), dict(mults=None, mult=1 << 30, mults2=None, mult2=-(1 << 31), scale=None),
               dict(mult3=(1 << 17) - 1, shift3=0), dict(mult3=-(1 << 16), shift3=30), dict(rows=0, A=0, B=0), dict(rows_a=0, A=0),
               dict(C=MIB + 64, lda=96, ldc=96), dict(experts=1, sb=0)):
        with pytest.raises(ValueError, match="null context"):
            rt.library().call("anvil_expert_gemm_i8", None, C.byref(rt.ExpertGemm(*{**GOOD_GEMM, **ok}.values())))


GOOD_COMBINE = dict(Y=MIB, ldy=64, slot=2 * MIB, weight=3 * MIB, positions=8, rows=4, top=2, cols=64, mult=3, shift=10, R=4 * MIB, ldr=64,
                    r_dtype=2, ma=256, mb=100, shift2=8, D=5 * MIB, ldd=64, d_dtype=2)


@pytest.mark.parametrize("bad", [dict(positions=-1), dict(rows=-1), dict(top=0), dict(top=33), dict(cols=0), dict(cols=(1 << 20) + 1),
                                 dict(rows=1 << 29), dict(r_dtype=4), dict(d_dtype=4), dict(R=0), dict(ldy=63), dict(ldr=63), dict(ldd=63),
                                 dict(ldd=1 << 31), dict(shift=63), dict(shift=-1), dict(shift2=32), dict(Y=0), dict(slot=0),
                                 dict(weight=0), dict(D=0), dict(slot=2 * MIB + 2), dict(weight=3 * MIB + 1), dict(R=4 * MIB + 1),
                                 dict(D=5 * MIB + 1), dict(D=MIB), dict(D=2 * MIB + 30), dict(D=3 * MIB + 14), dict(D=4 * MIB + 2),
                                 dict(D=4 * MIB, ldd=65)], ids=str)
def test_bad_combines_are_refused(bad):
    _refused("anvil_expert_combine_i8", rt.ExpertCombine, GOOD_COMBINE, bad)


def test_combine_sums_that_may_leave_int32_are_refused():
    top = (2 ** 31 - 1 - 128 - 128 * 100) // 32768
    for ma in (top + 1, -top - 1):
        _refused("anvil_expert_combine_i8", rt.ExpertCombine, GOOD_COMBINE, dict(ma=ma), OverflowError)
    for ok in (dict(ma=top), dict(D=4 * MIB), dict(R=0, d_dtype=1, ma=1 << 30), dict(rows=0, slot=0), dict(positions=0, Y=0)):
        with pytest.raises(ValueError, match="null context"):
            rt.library().call("anvil_expert_combine_i8", None, C.byref(rt.ExpertCombine(*{**GOOD_COMBINE, **ok}.values())))


def test_struct_layouts_match_the_header(tmp_path):
    import subprocess
    from pathlib import Path
    include = Path(__file__).resolve().parents[1] / "include"
    for cls, name in ((rt.AddNorm, "anvil_add_norm"), (rt.Route, "anvil_route"), (rt.ExpertGemm, "anvil_expert_gemm"),
                      (rt.ExpertCombine, "anvil_expert_combine")):
        fields = [f for f, _ in cls._fields_]
        src = tmp_path / f"{name}.c"
        src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "anvil_mi355x.h"\nint main(void) {\n'
                       f'  printf("%zu", sizeof({name}));\n' +
                       "".join(f'  printf(" %zu", offsetof({name}, {f}));\n' for f in fields) + "  return 0;\n}\n")
        subprocess.run(["gcc", "-std=c99", "-I", str(include), str(src), "-o", str(tmp_path / name)], check=True)
        got = [int(v) for v in subprocess.run([str(tmp_path / name)], capture_output=True, text=True, check=True).stdout.split()]
        assert got == [C.sizeof(cls)] + [getattr(cls, f).offset for f in fields]


def test_packed_arguments_are_the_structs():
    class Buffer:
        def __index__(self):
            return (1 << 47) + 64

    for cls, pack in ((rt.AddNorm, rt._ADD_NORM), (rt.Route, rt._ROUTE), (rt.ExpertGemm, rt._EXPERT_GEMM), (rt.ExpertCombine, rt._EXPERT_COMBINE)):
        rng, sizes = np.random.default_rng(1), [t for _, t in cls._fields_]
        values = [int(rng.integers(0, 1 << 48)) if t is C.c_void_p else int(rng.integers(-2 ** 31, 2 ** 31)) for t in sizes]
        want, data = bytes(cls(*values)), pack(*values)
        fields = [(getattr(cls, n).offset, C.sizeof(t)) for n, t in cls._fields_]                     # bytes between fields are nobody's
        assert len(data) == len(want) and all(data[o:o + n] == want[o:o + n] for o, n in fields)
        assert pack(*[np.int64(v) for v in values]) == data
        at = sizes.index(C.c_void_p)
        values[at] = Buffer()
        assert pack(*values)[fields[at][0]:][:8] == Buffer().__index__().to_bytes(8, "little")
    for bad in (dict(rows=1 << 31), dict(ma=-(2 ** 31) - 1), dict(shift=1.5), dict(X="x")):
        with pytest.raises(ValueError, match="anvil_add_norm_i8"):
            rt.library().call_packed("anvil_add_norm_i8", None, rt._ADD_NORM, *{**GOOD_NORM, **bad}.values())
    with pytest.raises(ValueError, match="null context"):
        rt.library().call_packed("anvil_add_norm_i8", None, rt._ADD_NORM, *GOOD_NORM.values())


# ------------------------------------------------------------------------------------------------- norm (GPU)

def norm_case(rows, cols, x="i16", y="i8", r="i16", seed=0, pad=0, off=0, extreme=False, place=None, lut=None, eps=3, lut_shift=15, ma=None,
              mb=None, shift=8, x_values=None):
    dev, rng = device(), np.random.default_rng(seed)
    r = x if y is None else r

    def values(dtype):
        n = LIMIT[dtype]
        a = rng.integers(-n, n, (rows, cols)) if extreme else np.clip(np.rint(rng.normal(0, n / 6, (rows, cols))), -n, n - 1).astype(int)
        return np.where(rng.random((rows, cols)) < 0.3, rng.choice([-n, n - 1], (rows, cols)), a) if extreme else a

    X, Y = values(x) if x_values is None else x_values, None if y is None else values(y)
    w = rng.integers(-128, 128, cols)
    lut = roots() if lut is None else lut
    unit = LIMIT[r] // LIMIT[x] or 1
    ma = (unit << 8 if LIMIT[x] <= LIMIT[r] else 2) if ma is None else ma
    mb = 70 if mb is None else mb
    want = oe.add_norm(X, Y, ma, mb, shift, r, w, lut, eps, lut_shift)
    dx = Rows(dev, X, x, pad, off)
    dy = None if y is None else Rows(dev, Y, y, pad, off, seed=1)
    dr = None if y is None else {"x": dx, "y": dy}.get(place) or Rows(dev, np.zeros((rows, cols), int), r, pad, off, seed=2)
    h, scale = Rows(dev, np.zeros((rows, cols), int), "i8", pad, off, seed=3), flat(dev, np.zeros(rows, int), "i16", off)
    dw, dl = flat(dev, w, "i8", off), dev.upload(lut.astype(np.int32))
    dev.add_norm(dx.ptr, x, dx.ld, dy and dy.ptr, y or "i8", dy.ld if dy else 0, ma, mb, shift, dr and dr.ptr, r, dr.ld if dr else 0, dw.ptr,
                 dl.ptr, len(lut), eps, lut_shift, h.ptr, h.ld, scale.ptr, rows, cols)
    dev.sync()
    if dr is not None:
        dr.expect(want[0], "r")
    if dr is not dx:
        dx.expect(X, "x")
    if dy is not None and dr is not dy:
        dy.expect(Y, "y")
    h.expect(want[1], "codes")
    scale.expect(want[2][None], "scale")


@gpu
@pytest.mark.parametrize("cols", [1, 2, 7, 15, 16, 24, 63, 64, 100, 127, 128, 256, 500, 512, 768, 1000, 1024, 1040, 2048, 4096, 4100, 8192, 8208,
                                  12000, 16384, 65536])
def test_norm_widths(cols):
    for rows in (1, 2, 67 if cols <= 4096 else 5):
        norm_case(rows, cols, seed=cols)
    norm_case(3, cols, "i8", "i8", "i8", seed=cols + 1)
    norm_case(3, cols, "i16", None, seed=cols + 2)


@gpu
@pytest.mark.parametrize("cols", [64, 128, 200, 256, 400, 512, 768, 1024, 1400, 2048, 4096, 6000, 8192, 16384])
def test_norm_types_at_every_width(cols):
    for n, (x, y, r) in enumerate((("i16", "i16", "i16"), ("i8", "i16", "i16"), ("i16", "i8", "i8"), ("i8", None, "i8"), ("i8", "i8", "i8"),
                                   ("i8", "i8", "i16"))):
        norm_case(11, cols, x, y, r, seed=cols + n)


@gpu
@pytest.mark.parametrize("cols", [*range(8, 34), 129, 255, 257, 263, 383, 511, 513, 519, 765, 767, 769, 1023, 1025, 2047, 2049, 2055, 4095, 4097, 8191,
                                  8193, 16383, 16377])
def test_norm_of_odd_widths(cols):
    """Every number of columns that a row's last two chunks share, beside each other's rows, in place, at any alignment."""
    rows = 37 if cols < 3000 else 3
    norm_case(rows, cols, seed=cols, place="x")
    norm_case(rows, cols, "i16", "i16", "i16", seed=cols + 1, place="y", off=3)
    norm_case(rows, cols, "i8", "i8", "i8", seed=cols + 2, place="x", off=1, pad=1)
    norm_case(rows, cols, "i16", None, seed=cols + 3, pad=5)
    norm_case(rows, cols, "i8", None, "i8", seed=cols + 4, off=7)
    norm_case(rows, cols, "i8", "i16", "i16", seed=cols + 5, extreme=True)


@gpu
@pytest.mark.parametrize("rows,cols", [(300001, 128), (140003, 512), (70001, 1024), (17003, 2056), (300001, 20), (140003, 517), (17003, 2049)])
def test_norm_of_more_rows_than_workgroups(rows, cols):
    """1000 rows over and over, in place, so that a workgroup that walks over rows has them in its registers one after the other."""
    dev, rng = device(), np.random.default_rng(cols)
    x, y, w = rng.integers(-9000, 9000, (1000, cols)), rng.integers(-128, 128, (1000, cols)), rng.integers(-128, 128, cols)
    turns = -(-rows // 1000)
    tile = lambda a, t: np.tile(a.astype(t), (turns, 1))[:rows]                                       # noqa: E731
    dx, dy, dw, dl = dev.upload(tile(x, np.int16)), dev.upload(tile(y, np.int8)), flat(dev, w, "i8"), flat(dev, roots(), "i32")
    dh, ds = dev.alloc(rows * cols), dev.alloc(2 * rows)
    dev.add_norm(dx.ptr, "i16", cols, dy.ptr, "i8", cols, 256, 900, 8, dx.ptr, "i16", cols, dw.ptr, dl.ptr, 1024, 7, 10, dh.ptr, cols, ds.ptr,
                 rows, cols)
    dev.sync()
    r, h, scale = oe.add_norm(x, y, 256, 900, 8, "i16", w, roots(), 7, 10)
    assert np.array_equal(dx.download((rows, cols), np.int16), tile(r, np.int16))
    assert np.array_equal(dh.download((rows, cols), np.int8), tile(h, np.int8))
    assert np.array_equal(ds.download((rows,), np.int16), np.tile(scale.astype(np.int16), turns)[:rows])


@gpu
@pytest.mark.parametrize("x", ["i8", "i16"])
@pytest.mark.parametrize("y", [None, "i8", "i16"])
@pytest.mark.parametrize("r", ["i8", "i16"])
def test_norm_types_and_extremes(x, y, r):
    for cols in (768, 45):
        norm_case(9, cols, x, y, r, seed=1)
        norm_case(9, cols, x, y, r, seed=2, extreme=True, ma=-200 if x == "i16" else 511, mb=-255, shift=9)
        norm_case(9, cols, x, y, r, seed=3, pad=16, off=0)
        norm_case(9, cols, x, y, r, seed=4, pad=3, off=1)
        norm_case(9, cols, x, y, r, seed=5, pad=8, off=8)


@gpu
@pytest.mark.parametrize("place", ["x", "y"])
def test_norm_in_place(place):
    for cols in (64, 768, 777, 9000):
        norm_case(5, cols, "i16", "i16", "i16", seed=cols, place=place)
        norm_case(5, cols, "i8", "i8", "i8", seed=cols, place=place, pad=2)


@gpu
def test_norm_tables_shifts_and_empty_rows():
    for n in (2, 3, 16, 1023, 1024, 4096, 65536):
        norm_case(6, 300, seed=n, lut=roots(n, 1 << 14), lut_shift=8)
    norm_case(6, 300, lut=-roots(), lut_shift=0)                   # entries below 0 count as 0
    for lut_shift in (0, 1, 20, 31):                               # scales that saturate, and that vanish
        norm_case(6, 300, lut_shift=lut_shift)
        norm_case(6, 300, lut_shift=lut_shift, lut=np.full(1024, 2 ** 31 - 1))
    for eps in (0, 1, 2 ** 31 - 1):
        norm_case(4, 40, "i16", None, eps=eps, x_values=np.zeros((4, 40), int))
        norm_case(4, 40, "i16", None, eps=eps, x_values=np.repeat([[0], [1], [-1], [32767]], 40, axis=1))
    norm_case(3, 65536, "i16", None, x_values=np.full((3, 65536), -32768))     # a sum of squares of 2^46
    norm_case(70000, 16, seed=5)
    dev = device()
    dev.add_norm(None, "i8", 4, None, "i8", 4, 0, 0, 0, None, "i8", 4, None, None, 2, 0, 0, None, 4, None, 0, 4)
    dev.sync()


# ------------------------------------------------------------------------------------------------ route (GPU)

def route_case(rows, experts, top, seed=0, live=None, every=False, lut=None, one=127, pad=0, scores=None, spread=30):
    dev, rng = device(), np.random.default_rng(seed)
    x = np.clip(np.rint(rng.normal(0, spread, (rows, experts))), -128, 127).astype(int) if scores is None else scores
    alive = None if live is None else (rng.random(rows) < live).astype(int) * rng.integers(1, 256, rows)
    lut = exp_lut() if lut is None else lut
    expert, weight, slot, row, starts = oe.route(x, alive, top, lut, one, every)
    dx, dl = Rows(dev, x, "i8", pad, off=1), dev.upload(lut.astype(np.int32))
    da = None if alive is None else dev.upload(alive.astype(np.uint8))
    pairs = np.zeros((rows, top), int)
    de, ds, dr = (flat(dev, pairs, "i32", off=1) for _ in range(3))
    dw, dt = flat(dev, pairs, "i16", off=1), flat(dev, np.zeros(experts + 1, int), "i32", off=1)
    before = np.random.default_rng(5).integers(-9, 9, rows * top)
    dr = flat(dev, before, "i32", off=1)
    dev.expert_route(dx.ptr, dx.ld, da and da.ptr, rows, experts, top, dl.ptr, one, de.ptr, dw.ptr, ds.ptr, dr.ptr, dt.ptr, every=every)
    dev.sync()
    de.expect(expert.reshape(1, -1), "experts")
    dw.expect(weight.reshape(1, -1), "weights")
    dt.expect(starts[None], "starts")
    ds.expect(slot.reshape(1, -1), "slots")
    before[:len(row)] = row
    dr.expect(before[None], "rows")


@gpu
@pytest.mark.parametrize("rows", [1, 2, 3, 63, 64, 65, 127, 128, 129, 257, 1000])
def test_route_rows(rows):
    for experts, top in ((1, 1), (2, 2), (8, 2), (61, 8), (64, 6), (65, 3), (128, 8), (257, 5), (1024, 32)):
        if rows * experts <= 100000:
            route_case(rows, experts, top, seed=rows + experts)


@gpu
@pytest.mark.parametrize("live", [0.0, 0.3, 0.9])
@pytest.mark.parametrize("every", [False, True])
def test_route_padding_and_weights(live, every):
    for rows, experts, top in ((1, 4, 2), (5, 8, 8), (300, 64, 6), (700, 130, 4)):
        for one in (1, 127, 32767):
            route_case(rows, experts, top, seed=rows, live=live, every=every, one=one, pad=3)


@gpu
def test_route_ties_and_tables():
    for experts, top in ((8, 3), (64, 32), (200, 17), (1024, 5)):
        route_case(40, experts, top, scores=np.zeros((40, experts), int))
        route_case(40, experts, top, spread=1.5)
        route_case(40, experts, top, scores=np.full((40, experts), -128))
        route_case(40, experts, top, scores=np.random.default_rng(3).choice([-128, 127], (40, experts)))
    for lut in (np.full(256, 2 ** 31 - 1), np.arange(256) - 200, np.r_[np.zeros(255, int), 1], np.r_[np.full(255, -5), 3],
                np.r_[np.full(255, 2 ** 31 - 1), 1]):
        for every in (False, True):
            route_case(50, 70, 9, lut=lut, one=32767, every=every)
    route_case(50, 70, 9, spread=500)


@gpu
def test_route_of_many_rows():
    rng = np.random.default_rng(0)
    route_case(20011, 16, 2, seed=1, live=0.95)
    route_case(9000, 40, 4, scores=np.clip(np.rint(rng.normal(0, 20, (9000, 40)) + 60 * (np.arange(40) == 7)), -128, 127).astype(int))


@gpu
def test_route_reports_rows_without_weight():
    dev = device()
    with pytest.raises(ZeroDivisionError):
        route_case(5, 8, 2, lut=np.zeros(256, int))
    dev.sync()
    with pytest.raises(ZeroDivisionError):
        route_case(500, 8, 2, lut=np.r_[np.zeros(255, int), -1])
    dev.sync()
    t = flat(dev, np.full(9, 77), "i32")
    dev.expert_route(None, 8, None, 0, 8, 2, None, 1, None, None, None, None, t.ptr)
    dev.sync()
    t.expect(np.zeros((1, 9), int))


# --------------------------------------------------------------------------------------------- products (GPU)

def product_case(counts, N, K, kind="plain", gather=True, scaled=True, dtype="i8", seed=0, behind=3, rows_a=None, pads=(0, 0, 0), off=0,
                 mults="each", mult=None, shift=None, extreme=False, call=None):
    """counts: the experts' rows. behind: rows of the result behind the last one."""
    dev, rng = device(), np.random.default_rng(seed)
    E, n = len(counts), sum(counts)
    starts = np.r_[0, np.cumsum(counts)]
    rows = n + behind
    na = (rows_a or max(1, n // 2 + 1)) if gather else max(1, rows)
    A = rng.choice([-128, 127], (na, K)) if extreme else rng.integers(-128, 128, (na, K))
    B, B2 = rng.integers(-128, 128, (2, E * N, K), dtype=np.int64 if E * N * K < 1 << 22 else np.int8)
    if extreme:
        B = rng.choice([-128, 127], (E * N, K))
        A[0], B[0] = -128, -128
    row = rng.integers(0, na, rows) if gather else None
    scale = rng.integers(-32768, 32768, na) if scaled and extreme else rng.integers(1, 32768, na) if scaled else None
    gated = kind == "gated"
    lut = None if kind == "plain" else act_lut()
    limit = 32767 if scaled else 2 ** 31 - 1
    spread = 5500 * np.sqrt(K) * (16000 if scaled else 1) / (90 if dtype == "i8" else 20000)
    if shift is None:
        shift = int(np.log2(spread)) + 14
    base = mult if mult is not None else min(limit, max(1, round(2 ** shift / spread)))
    m1, m2 = (np.clip(base + rng.integers(-(abs(base) // 4) - 1, abs(base) // 4 + 2, E), -limit, limit) if mults == "each" else np.full(E, base)
              for _ in range(2))
    before = rng.integers(-100, 100, (rows, N))
    want = oe.gemm(before, A, row, scale, B.reshape(E, N, K), B2.reshape(E, N, K) if gated else None, starts, m1, shift, m2, shift, lut, 13,
                   9, dtype)
    dA, dB, dB2 = Rows(dev, A, "i8", pads[0], off), Rows(dev, B, "i8", pads[1], off), Rows(dev, B2, "i8", pads[1], off)
    dC = Rows(dev, before, dtype, pads[2], off)
    dr, ds = None if row is None else flat(dev, row, "i32"), None if scale is None else flat(dev, scale, "i16")
    dt, d1, d2 = flat(dev, starts, "i32"), flat(dev, m1, "i32"), flat(dev, m2, "i32")
    dl = None if lut is None else flat(dev, lut, "i8")
    ptr = lambda b: b and b.ptr                                                                       # noqa: E731
    args = dict(A=dA.ptr, lda=dA.ld, rows_a=na, row=ptr(dr), scale=ptr(ds), B=dB.ptr, B2=dB2.ptr if gated else None, ldb=dB.ld, sb=N * dB.ld,
                starts=dt.ptr, experts=E, rows=rows, N=N, K=K, Cp=dC.ptr, ldc=dC.ld, out_dtype=dtype, shift=shift, shift2=shift,
                lut=ptr(dl), mult3=13, shift3=9, mult=int(base), mult2=int(base))
    if mults == "each":
        args.update(mults=d1.ptr, mults2=d2.ptr)
    run = lambda: dev.expert_gemm(**args)                                                             # noqa: E731
    if call:
        return call(dev, run, args, want, dC, (dA, dB, dB2, dr, ds, dt, d1, d2, dl))
    run()
    dev.sync()
    dC.expect(want, f"{counts} {N} {K} {kind}")


COUNTS = [[1], [0], [2, 0, 3], [64], [65, 1], [127, 128, 129], [0, 0, 5, 0], [31, 32, 33, 63], [300, 2, 40], [1] * 70, [0] * 100 + [9],
          [16, 17, 15, 1]]


@gpu
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}x{max(c)}")
@pytest.mark.parametrize("kind", ["plain", "table", "gated"])
def test_products_of_uneven_experts(counts, kind):
    product_case(counts, 128, 256, kind, seed=1)
    product_case(counts, 200, 144, kind, seed=2, scaled=False, gather=False)


@gpu
@pytest.mark.parametrize("N", [1, 15, 16, 17, 31, 32, 48, 63, 64, 65, 127, 129, 255, 256, 320, 1000])
def test_product_widths(N):
    for kind in ("plain", "gated"):
        product_case([40, 0, 7], N, 64, kind, seed=N)
        product_case([140, 3], N, 128, kind, seed=N, scaled=False)
    product_case([40, 0, 7], N, 64, dtype="i16", seed=N)
    product_case([140, 3], N, 192, dtype="i16", seed=N, gather=False)


@gpu
@pytest.mark.parametrize("K", [1, 3, 15, 16, 17, 32, 48, 64, 80, 100, 112, 128, 144, 256, 272, 384, 400, 512, 528, 640, 1000, 2048, 4097])
def test_product_depths(K):
    for kind in ("plain", "table", "gated"):
        product_case([40, 0, 70], 96, K, kind, seed=K)
        product_case([200], 160, K, kind, seed=K, gather=False, scaled=False)
        product_case([1, 3, 2], 40, K, kind, seed=K)


# Sizes that leave the few-rows kernel (640 workgroups, or 1280 where rows are at most 8 an expert) for 64 x 128 tiles, and (at least 640 tiles of
# 128 x 256, or 384 with a K of 2048 or more) for those, on 256 CUs.
FORMS = [("plain", "i8"), ("plain", "i16"), ("table", "i8"), ("gated", "i8")]


@gpu
@pytest.mark.parametrize("kind,dtype", FORMS)
@pytest.mark.parametrize("N,K", [(640, 1024), (700, 1040), (1001, 528), (1000, 16 * 41), (513, 2048), (5000, 128), (960, 1024), (736, 2048), (1300, 384)])
def test_products_by_tiles_of_64_rows(N, K, kind, dtype):
    counts = [130, 0, 61, 200, 64, 1, 150, 65, 63]
    product_case(counts, N, K, kind, dtype=dtype, seed=N)
    product_case(counts, N, K, kind, dtype=dtype, seed=K, gather=False, scaled=False, pads=(16, 32, 1), mults="one")


@gpu
@pytest.mark.parametrize("kind,dtype", FORMS)
@pytest.mark.parametrize("experts,N,K", [(90, 2048, 80), (90, 2000, 64), (85, 2049, 128), (90, 2048, 192), (80, 2300, 208), (24, 4096, 2064),
                                         (25, 4100, 2048)])
def test_products_by_tiles_of_128_rows(experts, N, K, kind, dtype):
    rng = np.random.default_rng(N)
    counts = rng.integers(0, 60, experts)
    counts[[1, 3]] = 0, 300
    counts[5:8] = 127, 128, 129
    counts[9] += max(0, (1 << 28) // (N * K) + 1 - counts.sum())
    product_case(counts.tolist(), N, K, kind, dtype=dtype, seed=K, scaled=K % 128 == 0)


@gpu
@pytest.mark.parametrize("kind,dtype", FORMS)
@pytest.mark.parametrize("K", [*range(16, 34), 47, 63, 65, 79, 127, 129, 1000, 1023, 1025, 1041, 2047, 4097])
def test_products_of_odd_depths(K, kind, dtype):
    """Every number of bytes that K's last two chunks share: few rows, tiles of 64 by 64, at any alignment."""
    product_case([3, 0, 20, 1, 40], 37, K, kind, dtype=dtype, seed=K)
    product_case([3, 0, 20, 1, 40], 37, K, kind, dtype=dtype, seed=K, off=5, pads=(1, 3, 2), gather=False, scaled=False, mults="one")
    product_case([300, 5, 0, 130], 70, K, kind, dtype=dtype, seed=K, off=1)


@gpu
@pytest.mark.parametrize("kind,dtype", FORMS)
@pytest.mark.parametrize("N,K", [(1400, 33), (1401, 129), (1409, 150)])
def test_products_of_many_rows_at_any_alignment(N, K, kind, dtype):
    """At least 2048 tiles of 128 x 64 (8 a CU)."""
    product_case([4000, 0, 129, 127, 128, 5900, 1, 2000], N, K, kind, dtype=dtype, seed=K)
    product_case([6000, 3, 6200], N, K, kind, dtype=dtype, seed=N, off=3, pads=(1, 0, 5), scaled=False, gather=False)


@gpu
@pytest.mark.parametrize("kind", ["plain", "gated"])
def test_product_strides_and_alignment(kind):
    for pads, off in (((16, 16, 16), 0), ((64, 0, 0), 16), ((0, 0, 0), 1), ((1, 0, 0), 0), ((0, 3, 0), 0), ((0, 0, 5), 0), ((0, 0, 0), 4)):
        product_case([70, 5, 130], 112, 96, kind, seed=3, pads=pads, off=off)
        if kind == "plain":
            product_case([70, 5, 130], 112, 96, kind, seed=3, pads=pads, off=off, dtype="i16")


@gpu
@pytest.mark.parametrize("mults", ["each", "one"])
def test_product_multipliers_and_shifts(mults):
    for shift, mult in ((0, 1), (1, 3), (7, -1), (14, 5), (31, 70000), (32, 2 ** 20), (40, -(2 ** 30)), (62, 2 ** 31 - 1), (20, 2 ** 20)):
        for kind in ("plain", "gated"):
            product_case([30, 80], 64, 64, kind, scaled=False, mults=mults, shift=shift, mult=mult, seed=shift)
    for shift, mult in ((0, 1), (20, 7), (31, -900), (32, 32767), (33, -32767), (45, 20000), (62, 32767)):
        for dtype in ("i8", "i16"):
            product_case([30, 80], 64, 64, mults=mults, shift=shift, mult=mult, seed=shift, extreme=True, dtype=dtype)
    product_case([3, 4], 33, 65536, mults=mults, extreme=True)                # sums of 2^30


@gpu
@pytest.mark.parametrize("rows,N,K", [(20, 64, 8192), (520, 256, 8192), (300, 70, 8190), (700, 1500, 8192), (700, 1500, 8190)],
                         ids=["few", "tiles", "any", "wide tiles", "wide, any"])
@pytest.mark.parametrize("kind", ["table", "gated"])
def test_tables_behind_the_largest_shifts(rows, N, K, kind):
    """Sums near 2^27 times multipliers near 2^31: results of a few units either way at shifts up to 58."""
    dev, rng = device(), np.random.default_rng(K)
    A, B = rng.integers(100, 128, (rows, K)), rng.integers(90, 128, (2, N, K)) * rng.choice([-1, 1], (2, N, 1))
    lut = rng.permutation(256) - 128
    dA, dB, dB2, out = Rows(dev, A, "i8"), Rows(dev, B[0], "i8"), Rows(dev, B[1], "i8"), Rows(dev, np.zeros((rows, N), int), "i8")
    dt, dl, m, start = flat(dev, [0, rows], "i32"), flat(dev, lut, "i8"), 2 ** 31 - 1, [0, rows]
    for shift in (55, 56, 57, 58):
        gated = kind == "gated"
        want = oe.gemm(np.zeros((rows, N)), A, None, None, B[:1], B[1:] if gated else None, start, [m], shift, [-m], shift, lut, 20, 3, "i8")
        assert len(np.unique(want)) > 1
        dev.expert_gemm(dA.ptr, dA.ld, rows, None, None, dB.ptr, dB2.ptr if gated else None, dB.ld, 0, dt.ptr, 1, rows, N, K, out.ptr, out.ld, "i8",
                        mult=m, shift=shift, mult2=-m, shift2=shift, lut=dl.ptr, mult3=20, shift3=3)
        dev.sync()
        out.expect(want, f"shift {shift}")


@gpu
@pytest.mark.parametrize("experts,N,K", [(9, 1024, 1024), (9, 1024, 1040), (90, 2048, 192), (90, 2048, 80)])
def test_rows_out_of_range_in_tiles_count_as_zeros(experts, N, K):
    def call(dev, run, args, want, dC, keep):
        row, want = keep[3].get()[0], want.copy()
        for p, bad in ((0, -1), (77, args["rows_a"]), (300, 2 ** 31 - 1), (301, -(2 ** 31))):
            row[p], want[p] = bad, 0
        dr = flat(dev, row, "i32")
        dev.expert_gemm(**{**args, "row": dr.ptr})
        with pytest.raises(ValueError, match="expert"):
            dev.sync()
        dev.sync()
        dC.expect(want)

    product_case([70 + 3 * e for e in range(experts)], N, K, call=call)


@gpu
def test_products_of_no_rows_at_all():
    """rows_a 0: every position's row leaves its range, and nothing of A is read."""
    def call(dev, run, args, want, dC, keep):
        for row in (args["row"], None):
            dev.expert_gemm(**{**args, "rows_a": 0, "A": None, "row": row})
            with pytest.raises(ValueError, match="expert"):
                dev.sync()
            dev.sync()
            want = want.copy()
            want[:sum(counts)] = 0
            dC.expect(want)

    for counts in ([3, 8], [130, 200, 300]):
        product_case(counts, 640, 1024, call=call)


@gpu
def test_product_of_large_strides():
    """Weights and rows past 2^32 bytes: the fourth expert lies behind 6 GiB, the last rows behind 5."""
    dev, rng = device(), np.random.default_rng(0)
    sb, lda, K, N = 2 << 30, 5 << 20, 64, 48
    A, B = rng.integers(-128, 128, (1025, K)), rng.integers(-128, 128, (4, N, K))
    big_a, big_b = dev.alloc(1024 * lda + K), dev.alloc(3 * sb + N * K)
    for i in (0, 1, 1023, 1024):
        big_a.upload(A[i].astype(np.int8), i * lda)
    for e in range(4):
        big_b.upload(B[e].astype(np.int8), e * sb)
    row = np.array([1024, 0, 1, 1023, 1024, 0, 1024, 1])
    out = Rows(dev, np.zeros((8, N), int), "i8")
    dr, dt = flat(dev, row, "i32"), flat(dev, np.array([0, 2, 4, 6, 8]), "i32")
    dev.expert_gemm(big_a.ptr, lda, 1025, dr.ptr, None, big_b.ptr, None, K, sb, dt.ptr, 4, 8, N, K, out.ptr, out.ld, "i8", mult=1, shift=12)
    dev.sync()
    out.expect(oe.gemm(np.zeros((8, N)), A, row, None, B, None, [0, 2, 4, 6, 8], [1] * 4, 12, None, 0, None, 1, 0, "i8"))


@gpu
@pytest.mark.parametrize("starts", [[0, 5, 3, 9], [0, 4, 8, 99], [-1, 4, 8, 9], [0, 10, 10, 10]], ids=str)
def test_starts_out_of_range_are_reported(starts):
    """An expert whose starts leave their range writes nothing; the others are computed."""
    def call(dev, run, args, want, dC, keep):
        dt = flat(dev, starts, "i32")
        args.update(starts=dt.ptr)
        dev.expert_gemm(**args)
        with pytest.raises(ValueError, match="expert"):
            dev.sync()
        dev.sync()

    product_case([3, 3, 3], 64, 64, behind=0, call=call)


@gpu
def test_rows_out_of_range_are_reported_and_count_as_zeros():
    def call(dev, run, args, want, dC, keep):
        row = keep[3].get()[0]
        row[2], row[70] = -1, args["rows_a"]
        dr = flat(dev, row, "i32")
        args.update(row=dr.ptr)
        dev.expert_gemm(**args)
        with pytest.raises(ValueError, match="expert"):
            dev.sync()
        dev.sync()
        want = want.copy()
        want[2] = want[70] = 0
        dC.expect(want)

    for N, K in ((64, 64), (70, 50)):
        product_case([3, 30, 60], N, K, call=call)


@gpu
def test_multipliers_out_of_range_with_scales_are_reported():
    def call(dev, run, args, want, dC, keep):
        for name, bad in (("mults", 32768), ("mults", -40000), ("mults2", 1 << 30)):
            m = keep[6].get()[0]
            m[1] = bad
            dm = flat(dev, m, "i32")
            dev.expert_gemm(**{**args, name: dm.ptr})
            with pytest.raises(ValueError, match="multiplier"):
                dev.sync()
            dev.sync()

    product_case([3, 30, 60], 64, 64, "gated", call=call)


# ---------------------------------------------------------------------------------------------- combine (GPU)

def combine_case(rows, top, cols, R="i16", D="i16", seed=0, pad=0, off=0, positions=None, place=False, mult=3, shift=15, extreme=False, dead=0.2):
    dev, rng = device(), np.random.default_rng(seed)
    positions = rows * top if positions is None else positions
    D = "i8" if R is None else D
    Y = rng.choice([-128, 127], (positions, cols)) if extreme else rng.integers(-128, 128, (positions, cols))
    slot = rng.integers(0, positions, (rows, top)) if positions else np.full((rows, top), -1)
    slot[rng.random((rows, top)) < dead] = -1
    weight = rng.choice([-32768, 32767], (rows, top)) if extreme else rng.integers(0, 32768 // top, (rows, top))
    n = LIMIT[R or "i8"]
    res = None if R is None else rng.integers(-n, n, (rows, cols))
    ma, mb, s2 = (250, 9000, 8) if D == "i16" else (50, -70, 7)
    want = oe.combine(Y, slot, weight, mult, shift, res, ma, mb, s2, D)
    dY, dR = Rows(dev, Y if positions else np.zeros((1, cols), int), "i8", pad, off), None if R is None else Rows(dev, res, R, pad, off)
    dD = dR if place else Rows(dev, np.zeros((rows, cols), int), D, pad, off, seed=1)
    ds, dw = flat(dev, slot, "i32"), flat(dev, weight, "i16")
    dev.expert_combine(dY.ptr, dY.ld, positions, ds.ptr, dw.ptr, rows, top, cols, mult, shift, dR and dR.ptr, R or "i8", dR.ld if dR else 0,
                       ma, mb, s2, dD.ptr, D, dD.ld)
    dev.sync()
    dD.expect(want, f"{rows} x {cols}, {top}, {R} -> {D}")


@gpu
@pytest.mark.parametrize("cols", [1, 5, 15, 16, 17, 64, 100, 256, 768, 1000, 1024, 4096, 10000])
def test_combine_widths(cols):
    for rows, top in ((1, 1), (1, 8), (37, 2), (5, 3), (130, 6), (2, 32)):
        combine_case(rows, top, cols, seed=cols + rows)


@gpu
@pytest.mark.parametrize("R", [None, "i8", "i16"])
@pytest.mark.parametrize("D", ["i8", "i16"])
def test_combine_types_strides_and_extremes(R, D):
    for cols in (768, 77):
        combine_case(20, 4, cols, R, D, seed=1)
        combine_case(20, 4, cols, R, D, seed=2, pad=16)
        combine_case(20, 4, cols, R, D, seed=3, pad=5, off=1)
        combine_case(20, 4, cols, R, D, seed=4, pad=8, off=8)
        combine_case(20, 32, cols, R, D, seed=5, extreme=True, dead=0, shift=20)
        combine_case(20, 2, cols, R, D, seed=6, dead=1.0)
        combine_case(20, 2, cols, R, D, seed=7, positions=0)
        for mult, shift in ((1, 0), (-1, 3), (2 ** 31 - 1, 62), (-(2 ** 31), 40), (7, 31), (7, 32), (1 << 20, 33)):
            combine_case(20, 4, cols, R, D, seed=8, mult=mult, shift=shift)


@gpu
def test_combine_in_place_and_many_rows():
    combine_case(70, 2, 256, "i16", "i16", place=True)
    combine_case(70, 2, 250, "i8", "i8", place=True, pad=2)
    for cols in range(16, 50):                                                # every number of columns behind the last sixteen
        combine_case(40, 2, cols, "i16", "i16", place=True, off=1, seed=cols)
        combine_case(40, 3, cols, "i8", "i8", place=True, off=3, pad=1, seed=cols)
        combine_case(40, 1, cols, "i8", "i16", seed=cols, off=1)
        combine_case(40, 5, cols, None, seed=cols)
    combine_case(20011, 2, 769, "i16", "i16", place=True, seed=2)
    combine_case(30001, 2, 48, seed=1)


@gpu
def test_slots_out_of_range_are_reported_and_add_nothing():
    dev = device()
    Y, D = Rows(dev, np.full((4, 32), 100), "i8"), Rows(dev, np.zeros((3, 32), int), "i8")
    slot, weight = flat(dev, [[0, 4], [-2, 1], [2, 3]], "i32"), flat(dev, [[1, 1]] * 3, "i16")
    for cols in (32, 31):
        dev.expert_combine(Y.ptr, Y.ld, 4, slot.ptr, weight.ptr, 3, 2, cols, 1, 1, None, "i8", 0, 0, 0, 0, D.ptr, "i8", D.ld)
        with pytest.raises(ValueError, match="slot"):
            dev.sync()
        dev.sync()
        assert D.get()[:, :cols].tolist() == [[50] * cols, [50] * cols, [100] * cols]


@gpu
def test_rows_past_four_gib():
    """Norm, router and weighted sums over rows 5 MiB and more apart: the last of them lie past 2^32 bytes."""
    dev, rng = device(), np.random.default_rng(0)
    n, ld, cols = 1000, 5 << 20, 64
    big = dev.alloc((n - 1) * ld + 4096)
    some = np.array([0, 1, 409, 410, 819, 820, n - 1])                        # 820 x 5 MiB is the first past 2^32

    def put(values):
        for i, v in zip(some, values):
            big.upload(v, int(i) * ld)

    def get(n, dtype):
        return np.stack([big.download((n,), dtype, int(i) * ld) for i in some]).astype(np.int64)

    big_zero = np.zeros(cols, np.int16)
    for i in range(n):
        big.upload(big_zero, i * ld)
    # the norm, in place: x + y over x
    x, y, w = np.zeros((n, cols), int), rng.integers(-128, 128, (n, cols)), rng.integers(30, 128, cols)
    x[some] = rng.integers(-9000, 9000, (len(some), cols))
    put(x[some].astype(np.int16))
    dy, dw, dl = Rows(dev, y, "i8"), flat(dev, w, "i8"), flat(dev, roots(), "i32")
    dh, ds = Rows(dev, np.zeros((n, cols), int), "i8"), flat(dev, np.zeros(n, int), "i16")
    dev.add_norm(big.ptr, "i16", ld // 2, dy.ptr, "i8", cols, 256, 900, 8, big.ptr, "i16", ld // 2, dw.ptr, dl.ptr, 1024, 7, 10, dh.ptr, cols,
                 ds.ptr, n, cols)
    dev.sync()
    r, h, scale = oe.add_norm(x, y, 256, 900, 8, "i16", w, roots(), 7, 10)
    dh.expect(h)
    ds.expect(scale[None])
    assert np.array_equal(get(cols, np.int16), r[some])
    # the router
    scores = np.zeros((n, 8), int)
    scores[some] = rng.integers(-100, 100, (len(some), 8))
    for i in range(n):
        big.upload(scores[i].astype(np.int8), i * ld)
    expert, weight, slot, row, starts = oe.route(scores, None, 2, exp_lut(), 127)
    de, dw2, dslot = (Rows(dev, np.zeros((n, 2), int), t) for t in ("i32", "i16", "i32"))
    dr, dt, de_lut = flat(dev, np.zeros(2 * n, int), "i32"), flat(dev, np.zeros(9, int), "i32"), flat(dev, exp_lut(), "i32")
    dev.expert_route(big.ptr, ld, None, n, 8, 2, de_lut.ptr, 127, de.ptr, dw2.ptr, dslot.ptr, dr.ptr, dt.ptr)
    dev.sync()
    for got, want in ((de, expert), (dw2, weight), (dslot, slot), (dr, row[None]), (dt, starts[None])):
        got.expect(want)
    # weighted sums of the rows, and then into them
    Y = rng.integers(-128, 128, (len(some), cols))
    put(Y.astype(np.int8))
    pick = rng.integers(0, len(some), (30, 2))
    d1, wt = Rows(dev, np.zeros((30, cols), int), "i8"), rng.integers(0, 128, (30, 2))
    dp, dwt = flat(dev, some[pick], "i32"), flat(dev, wt, "i16")
    dev.expert_combine(big.ptr, ld, n, dp.ptr, dwt.ptr, 30, 2, cols, 3, 9, None, "i8", 0, 0, 0, 0, d1.ptr, "i8", cols)
    dev.sync()
    d1.expect(oe.combine(Y, pick, wt, 3, 9, None, 0, 0, 0, "i8"))
    slot = rng.integers(0, 30, (n, 2))
    dp, dwt = flat(dev, slot, "i32"), flat(dev, np.tile(wt, (34, 1))[:n], "i16")
    y1 = d1.get()
    dev.expert_combine(d1.ptr, cols, 30, dp.ptr, dwt.ptr, n, 2, cols, 3, 9, None, "i8", 0, 0, 0, 0, big.ptr, "i8", ld)
    dev.sync()
    assert np.array_equal(get(cols, np.int8), oe.combine(y1, slot, np.tile(wt, (34, 1))[:n], 3, 9, None, 0, 0, 0, "i8")[some])


# ---------------------------------------------------------------------------------- a whole feed-forward (GPU)

class Layer:
    """All of it over device buffers, as a program keeps them."""

    def __init__(self, rows, experts, top, cols, width, gated, seed=0, dev=None):
        self.dev = dev or device()
        self.rng, self.shape, self.gated = np.random.default_rng(seed), (rows, experts, top, cols, width), gated
        rng, dev = self.rng, self.dev
        self.w = {"norm": rng.integers(30, 128, cols), "router": rng.integers(-60, 61, (experts, cols)),
                  "up": rng.integers(-90, 91, (experts * width, cols)), "gate": rng.integers(-90, 91, (experts * width, cols)),
                  "down": rng.integers(-90, 91, (experts * cols, width)), "each": rng.integers(12000, 20000, experts)}
        self.d = {k: flat(dev, v, "i32" if k == "each" else "i8") for k, v in self.w.items()}
        self.d.update(roots=flat(dev, roots(), "i32"), exp=flat(dev, exp_lut(), "i32"), act=flat(dev, act_lut(), "i8"),
                      one=flat(dev, [0, rows], "i32"))
        z = lambda r, c, t: Rows(dev, np.zeros((r, c), int), t)                                       # noqa: E731
        P = rows * top
        self.b = dict(x=z(rows, cols, "i16"), y=z(rows, cols, "i8"), r=z(rows, cols, "i16"), h=z(rows, cols, "i8"), scale=z(1, rows, "i16"),
                      live=z(1, rows, "i8"), scores=z(rows, experts, "i8"), expert=z(rows, top, "i32"), weight=z(rows, top, "i16"),
                      slot=z(rows, top, "i32"), row=z(1, P, "i32"), starts=z(1, experts + 1, "i32"), mid=z(P, width, "i8"),
                      out=z(P, cols, "i8"), d=z(rows, cols, "i16"))

    def inputs(self, seed, live=0.9):
        rng, (rows, _, _, cols, _) = np.random.default_rng(seed), self.shape
        self.x, self.y = rng.integers(-9000, 9000, (rows, cols)), rng.integers(-128, 128, (rows, cols))
        self.live = (rng.random(rows) < live).astype(int)
        for name, v in (("x", self.x), ("y", self.y), ("live", self.live[None])):
            self.b[name].buf.upload(v.astype(self.b[name].host.dtype))

    def run(self):
        dev, d, b, (rows, E, top, C, N) = self.dev, self.d, self.b, self.shape
        p = lambda n: b[n].ptr                                                                        # noqa: E731
        dev.add_norm(p("x"), "i16", C, p("y"), "i8", C, 256, 900, 8, p("r"), "i16", C, d["norm"].ptr, d["roots"].ptr, 1024, 7, 10, p("h"), C,
                     p("scale"), rows, C)
        dev.expert_gemm(p("h"), C, rows, None, p("scale"), d["router"].ptr, None, C, 0, d["one"].ptr, 1, rows, E, C, p("scores"), E, "i8",
                        mult=8000, shift=37)
        dev.expert_route(p("scores"), E, p("live"), rows, E, top, d["exp"].ptr, 16384, p("expert"), p("weight"), p("slot"), p("row"), p("starts"))
        dev.expert_gemm(p("h"), C, rows, p("row"), p("scale"), d["up"].ptr, d["gate"].ptr if self.gated else None, C, N * C, p("starts"), E,
                        rows * top, N, C, p("mid"), N, "i8", mults=d["each"].ptr, shift=39, mults2=d["each"].ptr, shift2=39, lut=d["act"].ptr,
                        mult3=13, shift3=9)
        dev.expert_gemm(p("mid"), N, rows * top, None, None, d["down"].ptr, None, N, C * N, p("starts"), E, rows * top, C, N, p("out"), C, "i8",
                        mults=d["each"].ptr, shift=23)
        dev.expert_combine(p("out"), C, rows * top, p("slot"), p("weight"), rows, top, C, 1, 14, p("r"), "i16", C, 256, 5000, 8, p("d"), "i16", C)

    def want(self):
        w, (rows, E, top, C, N) = self.w, self.shape
        r, h, scale = oe.add_norm(self.x, self.y, 256, 900, 8, "i16", w["norm"], roots(), 7, 10)
        scores = oe.gemm(np.zeros((rows, E)), h, None, scale, w["router"][None], None, [0, rows], [8000], 37, None, 0, None, 1, 0, "i8")
        expert, weight, slot, row, starts = oe.route(scores, self.live, top, exp_lut(), 16384)
        n = len(row)
        mid = oe.gemm(np.zeros((n, N)), h, row, scale, w["up"].reshape(E, N, C), w["gate"].reshape(E, N, C) if self.gated else None, starts,
                      w["each"], 39, w["each"], 39, act_lut(), 13, 9, "i8")
        out = oe.gemm(np.zeros((n, C)), mid, None, None, w["down"].reshape(E, C, N), None, starts, w["each"], 23, None, 0, None, 1, 0, "i8")
        d = oe.combine(out, slot, weight, 1, 14, r, 256, 5000, 8, "i16")
        return dict(r=r, h=h, scale=scale[None], scores=scores, expert=expert, weight=weight, slot=slot, starts=starts[None], d=d)

    def check(self):
        for name, v in self.want().items():
            np.testing.assert_array_equal(self.b[name].get(), v, err_msg=name)


@gpu
@pytest.mark.parametrize("shape", [(1, 4, 2, 64, 96), (7, 8, 2, 128, 64), (100, 16, 4, 192, 160), (333, 5, 3, 100, 77), (600, 8, 2, 256, 512)],
                         ids=str)
@pytest.mark.parametrize("gated", [False, True])
def test_feed_forward(shape, gated):
    layer = Layer(*shape, gated)
    layer.inputs(1)
    layer.run()
    layer.dev.sync()
    want = layer.want()
    assert shape[0] < 5 or (want["h"].any() and np.ptp(want["scores"]) > 20 and (want["d"] != want["r"]).mean() > 0.5)
    layer.check()


@gpu
def test_feed_forward_captured_and_recorded():
    """Replays with other inputs, eager calls and other sizes of the same context between them."""
    layer, other = Layer(90, 8, 2, 128, 64, True), Layer(700, 16, 2, 64, 64, False, seed=1)
    layer.inputs(1)
    layer.run()
    layer.dev.sync()
    graph = layer.dev.capture(layer.run)
    recorded = layer.dev.sequence(layer.run)
    for n, replay in enumerate([graph, recorded, graph, graph, recorded]):
        layer.inputs(10 + n, live=(1.0, 0.5, 0.0)[n % 3])
        replay.launch()
        if n % 2:
            layer.dev.sync()
        other.inputs(n)
        other.run()
        layer.check()
        other.check()


@gpu
def test_feed_forward_on_two_contexts():
    a, b = Layer(300, 8, 2, 128, 64, True), Layer(300, 8, 2, 128, 64, True, seed=3, dev=rt.Device(0))
    for n in range(3):
        a.inputs(n), b.inputs(n + 50)
        a.run(), b.run(), a.run(), b.run()
        a.dev.sync(), b.dev.sync()
        a.check(), b.check()
