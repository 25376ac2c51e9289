"""The decoding operators (4-bit paged cache, attention over it, page tables, beam selection) against their numpy
restatement in 64 bits. Every result is an integer, so every comparison is exact."""
import ctypes as C

import numpy as np
import pytest

from anvil_mi355x import runtime as rt
from decode_cases import PAGE, OnDevice, Sequences, exp_lut, fixed, starts_of
from oracle import decode as od
from oracle import semantics as sem

gpu = pytest.mark.gpu


# ------------------------------------------------------------------------------------- the oracle itself (CPU)

@pytest.mark.parametrize("dim", [16, 32, 64, 128])
def test_round4_is_within_half_a_step(dim):
    rng = np.random.default_rng(dim)
    for x in (rng.integers(-128, 128, (50, dim)), rng.integers(-3, 4, (50, dim)), np.full((2, dim), -128), np.zeros((1, dim), int)):
        codes, step = od.round4(x)
        g = x.reshape(codes.shape)
        assert codes.min() >= -7 and codes.max() <= 7 and step.min() >= 1 and step.max() <= 18
        # half a step; the two values past 7 x 18 = 126 are off by their distance to it
        assert np.all(np.abs(codes * step - g) <= np.maximum(step / 2, np.abs(g) - 126))
    small = rng.integers(-7, 8, (20, dim))
    assert np.array_equal(od.held(small), small)


@pytest.mark.parametrize("dim", [16, 32, 64, 128])
def test_a_page_packs_and_unpacks(dim):
    rng = np.random.default_rng(dim)
    k, v = rng.integers(-128, 128, (2, PAGE, dim))
    uk, uv = od.unpack_page(od.pack_page(k, v))
    assert np.array_equal(uk[:, :dim], od.held(k)) and np.array_equal(uv[:, :dim], od.held(v))
    assert not uk[:, dim:].any() and not uv[:, dim:].any()


@pytest.mark.parametrize("T", [1, 5, 40])
def test_attend_is_the_graph_chain_over_the_held_values(T):
    """The chain that the graph ops compute over the values 4 bits hold, row by row."""
    rng = np.random.default_rng(T)
    q, k, v = rng.integers(-128, 128, (3, T, 32))
    k, v = od.held(k), od.held(v)
    lut = exp_lut(bits=14)
    x = sem.qmatmul(q, k.T, 5, 14)
    want = sem.qmatmul(sem.softmax_lut(x, lut, 127, True), v, 3, 8)
    for t in range(T):
        got, zero = od.attend(q[t], k, v, t, np.ones(1, bool), 5, 14, lut, 127, 3, 8)
        assert not zero and np.array_equal(got, want[t])


def test_beam_select_is_a_log_softmax():
    """Fixed-point scores against float64 log-softmax: a table entry and its log are each off by half a unit, an index that
    lost its low bits by one part in nlogs / 2, so the error of one step stays below 2^16 (2 / 1024) + 4 units."""
    rng = np.random.default_rng(0)
    scale, n = 0.07, 2048
    logs = np.rint(np.log(np.maximum(1, np.arange(n))) * 65536).astype(np.int64)
    lut = np.rint(np.exp(np.arange(-255, 1) * scale) * (1 << 20))
    x = rng.integers(-128, 128, (6, 300))
    s, parent, token, ended, _ = od.beam_select(x, [0] * 6, None, None, 3, 2, 5, -1, lut, logs, round(np.log(2) * 65536),
                                               round(scale * 65536))
    logp = x * scale - np.log(np.exp(x * scale).sum(1, keepdims=True))
    assert np.all(np.abs(s / 65536 - logp[parent, token]) < 2 / 1024 + (4 + 255) / 65536)


# ----------------------------------------------------------------------------------------------- refusals (CPU)

def _cache(**kw):
    base = dict(pool=4096, table=4096, lens=4096, refs=4096, seqs=2, slots=4, pages=8, heads=2, dim=64, layers=1)
    base.update(kw)
    return rt.Cache(base.pop("pool"), base.pop("table"), base.pop("lens"), base.pop("refs"), **base)


def _call(name, *args):
    """An entry point without a context: its argument checks come first."""
    rt.library().call(name, None, *args)


BAD_CACHES = [dict(dim=48), dict(dim=256), dict(dim=0), dict(seqs=-1), dict(seqs=70000), dict(slots=0), dict(slots=20000),
              dict(pages=0), dict(pages=1 << 25), dict(heads=0), dict(layers=0), dict(pool=0), dict(pool=4104),
              dict(table=0), dict(lens=4097)]
ST = (C.c_int64 * 4)(128, 64, 128, 64)


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_bad_caches_are_refused(bad):
    c = C.byref(_cache(**bad))
    good = C.byref(_cache(table=1 << 20, lens=1 << 21, refs=1 << 22))
    for args in (("anvil_cache_append_i4", c, 0, 4096, 4096, None, 2, 1, ST),
                 ("anvil_cache_read_i4", c, 0, 4096, 4096, None, 2, 1, ST),
                 ("anvil_attention_cache_i4", c, 0, 4096, 4096, None, 2, 1, 4, ST, 3, 14, 4096, 127, 3, 8, 0, 0),
                 ("anvil_cache_fork", c, good, None, None, 0, 0), ("anvil_cache_fork", good, c, None, None, 0, 0),
                 ("anvil_cache_compact", c, good, 4096)):
        with pytest.raises(ValueError, match="anvil_cache|anvil_attention"):
            _call(*args)


@pytest.mark.parametrize("args", [
    (1, 4096, 4096, None, 2, 1, ST), (-1, 4096, 4096, None, 2, 1, ST),               # layer
    (0, 4096, 4096, None, 3, 1, ST), (0, 4096, 4096, None, 2, 2, ST),                # rows without starts
    (0, 4096, 4096, 4096, -1, 1, ST), (0, 4096, 4096, 4096, 2, 0, ST), (0, 4096, 4096, 4097, 2, 1, ST),
    (0, 0, 4096, None, 2, 1, ST), (0, 4104, 4096, None, 2, 1, ST), (0, 4096, 4100, None, 2, 1, ST),
    (0, 4096, 4096, None, 2, 1, None), (0, 4096, 4096, None, 2, 1, (C.c_int64 * 4)(128, 60, 128, 64))], ids=str)
def test_bad_rows_are_refused(args):
    for name in ("anvil_cache_append_i4", "anvil_cache_read_i4"):
        with pytest.raises(ValueError, match=name):
            _call(name, C.byref(_cache()), *args)


def test_a_read_into_overlapping_rows_is_refused():
    with pytest.raises(ValueError, match="stride 0"):
        _call("anvil_cache_read_i4", C.byref(_cache()), 0, 4096, 4096, None, 2, 1, (C.c_int64 * 4)(0, 64, 128, 64))


GOOD_ATTEND = dict(layer=0, Q=4096, O=4096, starts=None, rows=2, max_new=1, heads=4, strides=(C.c_int64 * 4)(256, 64, 256, 64),
                   ms=3, ss=14, lut=4096, one=127, mo=3, so=8, window=0, sinks=0)


@pytest.mark.parametrize("bad", [dict(heads=3), dict(heads=0), dict(heads=(1 << 31) - 2), dict(ss=32), dict(ss=-1), dict(so=32), dict(one=0),
                                 dict(one=32768), dict(window=-1), dict(sinks=-1), dict(lut=0), dict(lut=4098), dict(Q=4100),
                                 dict(O=4097), dict(Q=0), dict(strides=None), dict(strides=(C.c_int64 * 4)(256, 8, 256, 64)),
                                 dict(strides=(C.c_int64 * 4)(256, 64, 256, 32)),
                                 dict(strides=(C.c_int64 * 4)(256, 64, 254, 64))], ids=str)
def test_bad_attention_arguments_are_refused(bad):
    with pytest.raises(ValueError, match="anvil_attention_cache_i4"):
        _call("anvil_attention_cache_i4", C.byref(_cache()), *{**GOOD_ATTEND, **bad}.values())


def test_more_sequences_and_heads_than_a_grid_holds_are_refused():
    with pytest.raises(ValueError, match="65535 sequences"):
        _call("anvil_attention_cache_i4", C.byref(_cache(seqs=65535, heads=128)), *{**GOOD_ATTEND, "rows": 65535, "heads": 128}.values())


def test_a_score_multiplier_past_int32_is_refused():
    """128 * 126 * D * |m| + 2^(s-1) must fit int32; the largest that does passes on to the context check."""
    for dim in (16, 32, 64, 128):
        most = ((1 << 31) - 1 - (1 << 13)) // (128 * 126 * dim)
        for m in (most + 1, -most - 1, -(1 << 31)):
            with pytest.raises(OverflowError):
                _call("anvil_attention_cache_i4", C.byref(_cache(dim=dim)), *{**GOOD_ATTEND, "ms": m}.values())
        strides = (C.c_int64 * 4)(4 * dim, dim, 4 * dim, dim)
        with pytest.raises(ValueError, match="null context"):
            _call("anvil_attention_cache_i4", C.byref(_cache(dim=dim)), *{**GOOD_ATTEND, "ms": -most, "strides": strides}.values())


@pytest.mark.parametrize("change", [dict(pool=8192), dict(slots=5), dict(pages=9), dict(heads=4), dict(dim=32), dict(layers=2),
                                    dict(seqs=3), dict(refs=0), dict(table=4096), dict(lens=4100), dict(refs=4096 + 28)], ids=str)
def test_page_tables_that_do_not_fit_are_refused(change):
    a = _cache()
    apart = dict(table=1 << 20, lens=1 << 21, refs=1 << 22)
    b = _cache(**{**apart, **change})
    with pytest.raises(ValueError, match="anvil_cache_fork"):
        _call("anvil_cache_fork", C.byref(a), C.byref(b), None, None, 0, 0)
    with pytest.raises(ValueError, match="anvil_cache_compact"):
        _call("anvil_cache_compact", C.byref(a), C.byref(b), 4096)


def test_bad_step_arguments_are_refused():
    a, b = _cache(), _cache(table=1 << 20, lens=1 << 21, refs=1 << 22)
    for args in ((4097, None, 0, 0), (None, 4097, 0, 0), (None, None, -1, 0), (None, None, 4, -1)):
        with pytest.raises(ValueError, match="anvil_cache_fork"):
            _call("anvil_cache_fork", C.byref(a), C.byref(b), *args)
    big = dict(seqs=4097)
    with pytest.raises(ValueError, match="at most 4096"):
        _call("anvil_cache_fork", C.byref(_cache(**big)), C.byref(_cache(table=1 << 24, lens=1 << 25, refs=1 << 26, **big)),
              None, None, 0, 0)
    with pytest.raises(ValueError, match="anvil_cache_compact: map"):
        _call("anvil_cache_compact", C.byref(a), C.byref(b), None)
    for args in ((0, 1, 1, 64), (1, 0, 1, 64), (1, 1, 0, 64), (1, 1, 1, 40)):
        with pytest.raises(ValueError, match="anvil_cache_bytes"):
            rt.library().call("anvil_cache_bytes", *args, C.byref(C.c_longlong()))


GOOD_BEAMS = dict(logits=4096, ld=64, scores=4096, ended=None, allowed=None, groups=2, beams=3, vocab=64, keep=3, eos=-1,
                  lut=4096, logs=4096, nlogs=16, step=4, mult=5, scores_out=4144, parent=4144, token=4144, ended_out=4144)


@pytest.mark.parametrize("bad", [dict(groups=-1), dict(beams=0), dict(beams=65), dict(keep=0), dict(keep=65), dict(vocab=0),
                                 dict(ld=63), dict(nlogs=1), dict(step=-1), dict(mult=0), dict(eos=64), dict(eos=-2),
                                 dict(ended=4096), dict(logits=0), dict(scores=4100), dict(lut=4098), dict(logs=0),
                                 dict(scores_out=4100), dict(parent=4097), dict(token=0), dict(ended_out=0),
                                 dict(groups=1 << 20, beams=5), dict(scores_out=4096), dict(parent=4096 + 44), dict(token=4092),
                                 dict(ended=8192, ended_out=8197, eos=3), dict(ended_out=4096 + 47)], ids=str)
def test_bad_beams_are_refused(bad):
    with pytest.raises(ValueError, match="anvil_beam_select_i8"):
        _call("anvil_beam_select_i8", C.byref(rt.Beams(*{**GOOD_BEAMS, **bad}.values())))
    with pytest.raises(ValueError, match="null context"):
        _call("anvil_beam_select_i8", C.byref(rt.Beams(*GOOD_BEAMS.values())))
    with pytest.raises(ValueError, match="null arguments"):
        _call("anvil_beam_select_i8", None)


def test_cache_bytes():
    n = C.c_longlong()
    for layers, pages, heads, dim in ((1, 1, 1, 16), (2, 3, 4, 32), (12, 1 << 20, 8, 128)):
        rt.library().call("anvil_cache_bytes", layers, pages, heads, dim, C.byref(n))
        assert n.value == layers * pages * heads * 68 * max(32, dim)


def test_the_structs_mirror_the_header(tmp_path):
    import subprocess
    from pathlib import Path
    root = Path(__file__).resolve().parents[1]
    pairs = {"anvil_cache": rt.Cache, "anvil_beams": rt.Beams}
    lines = []
    for name, cls in pairs.items():
        lines.append(f'printf("%zu ", sizeof({name}));')
        lines += [f'printf("%zu ", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "t.c"
    src.write_text('#include <stdio.h>\n#include "anvil_mi355x.h"\nint main(void) {' + "\n".join(lines) + "return 0; }\n")
    subprocess.run(["gcc", "-I", str(root / "include"), str(src), "-o", str(tmp_path / "t")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for cls in pairs.values():
        want += [C.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]
    assert got == want


# ------------------------------------------------------------------------------------------- append and read

def _rows(seqs, news, layer, which, order="rows"):
    """The packed new rows (rows, heads, dim) of k or v."""
    src = (seqs.k if which == "k" else seqs.v)[layer]
    return np.concatenate([x[len(x) - n:] for x, n in zip(src, news)] or [np.zeros((0, seqs.heads, seqs.dim))])


LENS_NEWS = [([1], [1]), ([64], [1]), ([65, 1, 128], [1, 1, 1]), ([5, 0, 70, 200], [5, 0, 3, 0]), ([130, 64, 63], [130, 64, 63]),
             ([191, 129, 66, 2], [65, 66, 2, 1]), ([300, 300], [127, 1])]


@gpu
@pytest.mark.parametrize("lens,news", LENS_NEWS)
@pytest.mark.parametrize("dim,heads", [(16, 3), (32, 4), (64, 1), (128, 2)])
@pytest.mark.parametrize("layout", ["rows", "heads", "padded"])
def test_append_writes_its_rows_and_nothing_else(lens, news, dim, heads, layout):
    dev = rt.device(0)
    seqs = Sequences(lens, heads, dim, seed=len(lens), layers=2)
    before = np.random.default_rng(5).integers(0, 256, (2, seqs.pages, heads, 68 * od.stored_dim(dim))).astype(np.uint8)
    d = OnDevice(dev, seqs, before)
    rows = sum(news)
    starts = None if all(n == 1 for n in news) else dev.upload(starts_of(news))
    want = before.copy()
    whole = seqs.pool()
    for i, (n, new) in enumerate(zip(lens, news)):
        for j in range((n - new) // PAGE, -(-n // PAGE)):
            for h in range(heads):
                t0, t1 = max(n - new - j * PAGE, 0), min(n - j * PAGE, PAGE)
                if t1 > t0:
                    seqs.merge(want[1, seqs.table[i, j], h], whole[1, seqs.table[i, j], h], t0, t1)
    bufs = []
    for w in "kv":
        x = _rows(seqs, news, 1, w).astype(np.int8)
        if layout == "heads":
            x = np.ascontiguousarray(x.transpose(1, 0, 2))
        elif layout == "padded":
            x = np.concatenate([x, np.full((rows, heads, 32), 99, np.int8)], axis=2)
        bufs.append(dev.upload(x))
    st = {"rows": (heads * dim, dim), "heads": (dim, rows * dim), "padded": (heads * (dim + 32), dim + 32)}[layout]
    dev.cache_append(d.cache, 1, *bufs, starts, rows, max(news), (*st, *st))
    dev.sync()
    assert np.array_equal(d.read_pool(), want)
    if layout == "heads":                                        # and back, into rows with a guard behind the last
        outs = [dev.upload(np.full((rows + 2, heads, dim), 0x5A, np.int8)) for _ in "kv"]
        dev.cache_read(d.cache, 1, *outs, starts, rows, max(news), (heads * dim, dim) * 2)
        dev.sync()
        for out, w in zip(outs, "kv"):
            got = out.download((rows + 2, heads, dim), np.int8)
            assert np.array_equal(got[:rows], od.held(_rows(seqs, news, 1, w)))
            assert np.all(got[rows:] == 0x5A)


@gpu
@pytest.mark.parametrize("loud", [0, 0.4, 3, 400])
def test_append_of_quiet_and_saturated_rows(loud):
    """Rows of zeros, of the few values a step of 1 holds, and of -128 and 127."""
    dev = rt.device(0)
    seqs = Sequences([64, 7], 2, 64, loud=loud)
    d = OnDevice(dev, seqs, np.zeros((1, seqs.pages, 2, 68 * 64), np.uint8))
    news = [64, 7]
    k, v = (dev.upload(_rows(seqs, news, 0, w).astype(np.int8)) for w in "kv")
    dev.cache_append(d.cache, 0, k, v, dev.upload(starts_of(news)), 71, 64, (128, 64, 128, 64))
    dev.sync()
    assert np.array_equal(d.read_pool(), seqs.pool())


@gpu
def test_every_int8_rounds_as_defined():
    """Each value -128 .. 127 beside each loudest value 0 .. 128 of its group."""
    dev = rt.device(0)
    rows = 129 * 9
    x = np.zeros((rows, 1, 32), np.int64)
    for m in range(129):
        for part in range(9):
            vals = np.arange(part * 31 - 128, min(part * 31 - 97, 128))
            x[m * 9 + part, 0, :len(vals)] = np.clip(vals, -m, min(m, 127))
            x[m * 9 + part, 0, 31] = -m
    seqs = Sequences([rows], 1, 32)
    seqs.k[0][0], seqs.v[0][0] = x, x[::-1]
    d = OnDevice(dev, seqs, np.zeros((1, seqs.pages, 1, 68 * 32), np.uint8))
    k, v = dev.upload(x.astype(np.int8)), dev.upload(np.ascontiguousarray(x[::-1]).astype(np.int8))
    st = dev.upload(starts_of([rows]))
    dev.cache_append(d.cache, 0, k, v, st, rows, rows, (32, 32, 32, 32))
    ko, vo = dev.alloc(rows * 32), dev.alloc(rows * 32)
    dev.cache_read(d.cache, 0, ko, vo, st, rows, rows, (32, 32, 32, 32))
    dev.sync()
    assert np.array_equal(ko.download((rows, 1, 32), np.int8), od.held(x))
    assert np.array_equal(vo.download((rows, 1, 32), np.int8), od.held(x[::-1]))


# ------------------------------------------------------------------------------------------------- attention

def attention_want(seqs, news, q, heads_q, ms, ss, lut, one, mo, so, window=0, sinks=0, layer=0, held=True):
    """(rows, heads_q, dim) int8 and whether a row summed to zero."""
    hold = od.held if held else (lambda x: x)
    out, row, zero = [], 0, False
    for i, (n, new) in enumerate(zip(seqs.lens, news)):
        ks, vs = hold(seqs.k[layer][i]), hold(seqs.v[layer][i])
        have = seqs.table[i] >= 0
        for t in range(new):
            heads = []
            for h in range(heads_q):
                kv = h // (heads_q // seqs.heads)
                o, z = od.attend(q[row, h], ks[:, kv], vs[:, kv], n - new + t, have, ms, ss, lut, one, mo, so, window, sinks)
                heads.append(o)
                zero |= z
            out.append(heads)
            row += 1
    return np.array(out, dtype=np.int64).reshape(row, heads_q, seqs.dim), zero


LUTS = {"exp": exp_lut(), "steep": exp_lut(0.9, 20), "flat": np.full(256, 7), "random": np.random.default_rng(1).integers(0, 1 << 20, 256),
        "large": exp_lut(0.01, 31).clip(max=(1 << 31) - 1), "signed": np.where(np.arange(256) % 3 == 0, -5, exp_lut())}


def attention_case(lens, news, heads_q, heads, dim, seed=0, ratio=None, lut="exp", one=127, window=0, sinks=0, drop=(), loud=None,
                   order="rows"):
    dev = rt.device(0)
    seqs = Sequences(lens, heads, dim, seed=seed, loud=loud)
    rng = np.random.default_rng([seed, 9])
    rows = sum(news)
    q = rng.integers(-128, 128, (rows, heads_q, dim))
    ms, ss = fixed((0.4 if ratio is None else abs(ratio)) / np.sqrt(dim) / 40, 128 * 126 * dim)
    ms = -ms if ratio is not None and ratio < 0 else ms
    mo, so = fixed(2.0 / one, 126 * (one + max([1, *lens]) // 2))
    d = OnDevice(dev, seqs, seqs.pool(np.random.default_rng(3)))
    if len(drop):
        for i, j in drop:
            seqs.table[i, j] = -1
        d = OnDevice(dev, seqs, d.pool)
    starts = None if all(n == 1 for n in news) else dev.upload(starts_of(news))
    guard = 2
    if order == "rows":
        qb, st, shape = q, (heads_q * dim, dim, heads_q * dim, dim), (rows + guard, heads_q, dim)
    else:                                                        # heads outermost, rows padded
        qb = np.concatenate([q.transpose(1, 0, 2), np.full((heads_q, rows, 16), 77)], axis=2)
        st, shape = (dim + 16, rows * (dim + 16), dim + 4, (rows + guard) * (dim + 4)), (heads_q, rows + guard, dim + 4)
    out = dev.upload(np.full(shape, 0x5A, np.int8))
    dev.attention_cache(d.cache, 0, dev.upload(qb.astype(np.int8)), out, starts, rows, max([1, *news]), heads_q, st, ms, ss,
                        dev.upload(LUTS[lut].astype(np.int32)), one, mo, so, window, sinks)
    want, zero = attention_want(seqs, news, q, heads_q, ms, ss, LUTS[lut], one, mo, so, window, sinks)
    if zero:
        with pytest.raises(ZeroDivisionError):
            dev.sync()
    else:
        dev.sync()
    got = out.download(shape, np.int8).astype(np.int64)
    if order != "rows":
        assert np.all(got[:, :, dim:] == 0x5A)
        got = got[:, :, :dim].transpose(1, 0, 2)
    assert np.array_equal(got[:rows], want), np.argwhere(got[:rows] != want)[:5]
    assert np.all(got[rows:] == 0x5A)
    return want


DIMS = [(16, 1, 3), (32, 4, 4), (64, 12, 4), (64, 3, 3), (128, 8, 2), (128, 5, 1), (32, 40, 2)]


@gpu
@pytest.mark.parametrize("dim,heads_q,heads", DIMS)
@pytest.mark.parametrize("lens", [[1], [2, 64, 65, 3], [127, 128, 129], [200, 1, 0, 333]])
def test_attention_of_one_token_each(dim, heads_q, heads, lens):
    heads_q = heads if heads_q % heads else heads_q
    news = [1 if n else 0 for n in lens]
    want = attention_case(lens, news, heads_q, heads, dim, seed=len(lens))
    assert len(np.unique(want)) > 8 or len(lens) == 1


@gpu
@pytest.mark.parametrize("dim,heads_q,heads", DIMS)
@pytest.mark.parametrize("lens,news", [([5], [5]), ([64, 66], [64, 3]), ([150, 20, 70], [17, 20, 0]), ([130, 257], [65, 2])])
def test_attention_of_chunks(dim, heads_q, heads, lens, news):
    heads_q = heads if heads_q % heads else heads_q
    attention_case(lens, news, heads_q, heads, dim, seed=3, order="heads" if dim != 64 else "rows")


@gpu
@pytest.mark.parametrize("lut", sorted(LUTS))
@pytest.mark.parametrize("one", [1, 100, 127, 128, 910, 911, 4096, 32767])
def test_attention_tables_and_probabilities(lut, one):
    attention_case([190, 64, 1], [1, 2, 1], 4, 2, 32, seed=one, lut=lut, one=one)
    attention_case([700], [1], 4, 2, 64, seed=one, lut=lut, one=one)


@gpu
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (64, 0), (64, 4), (65, 64), (100, 70), (7, 129), (1000, 4), (130, 1000)])
@pytest.mark.parametrize("lens,news", [([300, 70, 1], [1, 1, 1]), ([300, 131], [40, 131]), ([64, 256], [1, 64])])
def test_attention_windows_and_sinks(window, sinks, lens, news):
    attention_case(lens, news, 4, 2, 64, seed=window, window=window, sinks=sinks)


@gpu
def test_attention_skips_pages_given_back():
    attention_case([300, 256, 64], [1, 1, 1], 4, 2, 64, drop=[(0, 1), (0, 2), (1, 0)])
    attention_case([300, 256, 64], [3, 70, 1], 4, 2, 32, drop=[(0, 0), (1, 1), (2, 0)])           # a row that sees nothing
    attention_case([400], [1], 2, 2, 128, window=100, sinks=3, drop=[(0, 1), (0, 2), (0, 3)])


@gpu
@pytest.mark.parametrize("ratio", [-0.4, 0, 40, -40])
def test_attention_of_flat_saturated_and_negated_scores(ratio):
    """All scores alike, all at the ends of int8, and a negative multiplier."""
    attention_case([333, 70], [1, 9], 4, 2, 64, ratio=ratio)
    attention_case([90], [1], 4, 4, 32, ratio=ratio, loud=0)


@gpu
@pytest.mark.parametrize("dim,heads_q,heads,n,new,one", [(64, 12, 12, 5000, 1, 127), (128, 8, 1, 9001, 1, 16384), (32, 2, 2, 20000, 2, 32767),
                                                         (64, 4, 2, 4097, 5, 1024), (128, 16, 2, 2500, 33, 500), (16, 24, 1, 3000, 1, 127)])
def test_attention_over_long_sequences(dim, heads_q, heads, n, new, one):
    attention_case([n, n // 3, 1], [new, 1, 1], heads_q, heads, dim, one=one)
    attention_case([n], [new], heads_q, heads, dim, one=one, window=n // 2, sinks=130)


MANY = [([2100, 70, 300, 0], [256, 70, 3, 0], 8, 8), ([2111, 129, 64, 1], [128, 128, 1, 1], 16, 4)]    # widened pages: 256 rows a cache head


@gpu
@pytest.mark.parametrize("lens,news,heads_q,heads", MANY)
@pytest.mark.parametrize("dim", [16, 32, 64, 128])
@pytest.mark.parametrize("one", [1, 127, 128, 32639, 32640])
def test_attention_of_many_rows(lens, news, heads_q, heads, dim, one):
    attention_case(lens, news, heads_q, heads, dim, seed=dim, one=one)


@gpu
@pytest.mark.parametrize("lut", ["large", "random", "signed"])
@pytest.mark.parametrize("one", [127, 4096])
def test_attention_of_many_rows_with_tables(lut, one):
    attention_case(*MANY[0], 32, seed=one, lut=lut, one=one, order="heads")
    attention_case([190, 64, 1], [9, 12, 1], 4, 2, 32, seed=one, lut=lut, one=one)


@gpu
@pytest.mark.parametrize("window,sinks", [(1, 0), (65, 0), (700, 70), (1900, 4), (64, 640)])
def test_attention_of_many_rows_through_windows(window, sinks):
    for case in MANY:                                          # windows under 32 pages take tiles of 16 rows, the others those of 32
        attention_case(*case, 64, seed=window, window=window, sinks=sinks, drop=[(0, 20), (0, 32)])


@gpu
def test_numbers_that_leave_their_range_are_reported_and_evaluate_nothing():
    dev = rt.device(0)
    seqs = Sequences([100, 50, 70], 2, 32, extra_slots=1)
    pool = seqs.pool()
    q = dev.upload(np.ones((3, 2, 32), np.int8))
    lut = dev.upload(exp_lut().astype(np.int32))
    for lens, starts, table in (([100, 5000, 70], None, None), ([100, -1, 70], None, None), ([100, 0, 70], [0, 1, 2, 3], None),
                                (None, [0, 1, 5, 3], None), (None, [0, 1, 0, 1], None), (None, [0, 1, 3, 4], None),
                                (None, [-1, 1, 1, 2], None), (None, None, (1, 0, 99)), (None, None, (1, 0, -2))):
        t = seqs.table.copy()
        if table:
            t[table[0], table[1]] = table[2]
        d = OnDevice(dev, seqs, pool, table=t, lens=lens)
        out = dev.upload(np.full((3, 2, 32), 0x5A, np.int8))
        st = None if starts is None else dev.upload(np.array(starts, np.int32))
        dev.attention_cache(d.cache, 0, q, out, st, 3, 1, 2, (64, 32, 64, 32), 3, 10, lut, 127, 1, 7)
        with pytest.raises(ValueError, match="page table, lengths"):
            dev.sync()
        if lens:
            assert np.all(out.download((3, 2, 32), np.int8)[1] == 0x5A)
        dev.cache_append(d.cache, 0, q, q, st, 3, 1, (64, 32, 64, 32))
        with pytest.raises(ValueError, match="page table, lengths"):
            dev.sync()
        dev.cache_read(d.cache, 0, dev.alloc(192), dev.alloc(192), st, 3, 1, (64, 32, 64, 32))
        with pytest.raises(ValueError, match="page table, lengths"):
            dev.sync()
        dev.sync()


@gpu
def test_empty_calls():
    dev = rt.device(0)
    seqs = Sequences([10], 2, 32)
    d = OnDevice(dev, seqs, seqs.pool())
    none = rt.Cache(d.pool, 0, 0, d.refs, seqs=0, slots=1, pages=seqs.pages, heads=2, dim=32)
    lut = dev.upload(exp_lut().astype(np.int32))
    dev.cache_append(none, 0, None, None, None, 0, 1, (64, 32, 64, 32))
    dev.attention_cache(none, 0, None, None, None, 0, 1, 2, (64, 32, 64, 32), 3, 10, lut, 127, 1, 7)
    dev.attention_cache(d.cache, 0, None, None, dev.upload(starts_of([0])), 0, 1, 2, (64, 32, 64, 32), 3, 10, lut, 127, 1, 7)
    dev.sync()


@gpu
def test_a_pool_past_4_gib():
    """Pages whose byte offsets need 33 bits, in the second of two layers."""
    dev = rt.device(0)
    seqs = Sequences([130, 64], 8, 128)
    small = seqs.pool()
    pages = 42000                                                # 8 heads x 8704 bytes a page: 2.9 GB a layer
    table = np.where(seqs.table >= 0, pages - 1 - seqs.table, -1)
    pool = dev.alloc(2 * pages * seqs.page_bytes)
    for p in range(seqs.pages):
        pool.upload(small[0, p], (2 * pages - 1 - p) * seqs.page_bytes)
    cache = rt.Cache(pool, t := dev.upload(table.astype(np.int32)), n := dev.upload(np.array(seqs.lens, np.int32)), seqs=2,
                     slots=seqs.slots, pages=pages, heads=8, dim=128, layers=2)
    q = np.random.default_rng(0).integers(-128, 128, (2, 8, 128))
    out = dev.alloc(q.size)
    dev.attention_cache(cache, 1, dev.upload(q.astype(np.int8)), out, None, 2, 1, 8, (1024, 128, 1024, 128), 5, 18,
                        dev.upload(exp_lut().astype(np.int32)), 127, 1, 7)
    dev.sync()
    want, _ = attention_want(seqs, [1, 1], q, 8, 5, 18, exp_lut(), 127, 1, 7)
    assert np.array_equal(out.download(q.shape, np.int8), want)
    del t, n


# ------------------------------------------------------------------------------------------- fork and compact

def fork_case(seqs, parent, add, window=0, sinks=0, refs=None, table=None, lens=None):
    """One step on the device against the oracle: tables, references and the pool's bytes."""
    dev = rt.device(0)
    rng = np.random.default_rng(2)
    pool = rng.integers(0, 256, (seqs.layers, seqs.pages, seqs.heads, 68 * od.stored_dim(seqs.dim))).astype(np.uint8)
    refs = seqs.refs if refs is None else refs
    table = seqs.table if table is None else table
    lens = seqs.lens if lens is None else lens
    d = OnDevice(dev, seqs, pool, table, lens, refs)
    n = len(table) if parent is None else len(parent)
    out = d.successor(n)
    up = lambda x: None if x is None else dev.upload(np.array(x, np.int32))                          # noqa: E731
    dev.cache_fork(d.cache, out.cache, up(parent), up(add), window, sinks)
    try:
        w_table, w_lens, w_refs, copies = od.fork(table, np.array(lens), refs, parent, add, window, sinks)
    except od.OutOfPages:
        with pytest.raises(MemoryError):
            dev.sync()
        w_table, w_lens, w_refs, copies = np.full((n, seqs.slots), -1), np.zeros(n), refs, []
    else:
        dev.sync()
    t, ln, r = out.tables()
    assert np.array_equal(t, w_table) and np.array_equal(ln, w_lens) and np.array_equal(r, w_refs)
    want = pool.copy()
    for a, b in copies:
        want[:, b] = pool[:, a]
    assert np.array_equal(d.read_pool(), want)
    for got, was in zip(d.tables(), (table, lens, refs)):        # the step that was is still there
        assert np.array_equal(got, was)
    return w_table, w_lens, w_refs, copies


@gpu
@pytest.mark.parametrize("add", [None, [0, 1, 70, 0], [1, 1, 1, 1], [64, 200, 0, 1]])
def test_reserve(add):
    fork_case(Sequences([64, 10, 130, 0], 2, 32, spare=12, extra_slots=4, layers=2), None, add)


@gpu
def test_fork_copies_a_shared_last_page_once_a_row_but_the_last():
    seqs = Sequences([100, 64, 20], 2, 64, spare=8, layers=3)
    _, _, refs, copies = fork_case(seqs, [0, 0, 0, 1, 1, 2], [1, 1, 1, 1, 1, 1])
    assert len(copies) == 2
    held = seqs.refs.copy()
    held[seqs.table[0, 1]] += 1                                  # a page held by something else is copied by everyone
    _, _, _, copies = fork_case(seqs, [0, 0, -1, 2], [1, 1, 1, 0], refs=held)
    assert len(copies) == 2
    _, _, refs, copies = fork_case(seqs, [0, 0, 0], [1, 0, 0])   # one of three extends
    assert len(copies) == 1


@gpu
def test_free_and_refill():
    seqs = Sequences([200, 64, 129], 1, 32, spare=0, extra_slots=2)
    _, _, refs, _ = fork_case(seqs, [-1, 1, -1], None)
    assert refs.sum() == 1
    fork_case(seqs, [-1, 1, -1], [500, 128, 7])                  # the pages given back are taken at once
    fork_case(seqs, [-1, -1], None)


@gpu
def test_too_few_pages_or_slots_leave_everything_empty():
    seqs = Sequences([100, 64], 1, 32, spare=1, extra_slots=1)
    fork_case(seqs, None, [1, 64])                               # one page is there
    fork_case(seqs, None, [64, 1])                               # two are not
    fork_case(Sequences([100], 1, 32, spare=9), None, [29])      # slots for 128 tokens
    fork_case(Sequences([100], 1, 32, spare=9), None, [28])


@gpu
@pytest.mark.parametrize("window,sinks", [(1, 0), (64, 0), (65, 1), (100, 64), (100, 65), (128, 200), (5000, 0)])
def test_a_window_gives_pages_back(window, sinks):
    seqs = Sequences([500, 64, 129, 1, 300], 1, 32, spare=9, extra_slots=2)
    table, lens, refs, _ = fork_case(seqs, [0, 1, 2, 3, 4, 4], [1, 1, 1, 1, 0, 70], window, sinks)
    # what is gone is seen by no query of the next step or a later one
    for row in range(len(table)):
        n = [500, 64, 129, 1, 300, 300][row]
        for j in range(-(-n // PAGE)):
            keys = np.arange(j * PAGE, j * PAGE + PAGE)
            assert (table[row, j] < 0) == (not (od.visible(keys, n, window, sinks) | (keys >= n)).any())


@gpu
@pytest.mark.parametrize("seed", range(12))
def test_random_steps(seed):
    """A batch through several steps: parents, extensions, pages held elsewhere, rows that come and go."""
    random_steps(seed)


@gpu
@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("more", [dict(extra_slots=2000), dict(spare=13000), dict(extra_slots=400, spare=20000)], ids=str)
def test_random_steps_of_large_tables(more, seed):
    """Tables and pools past one workgroup's."""
    random_steps(seed, **more)


def random_steps(seed, **more):
    rng = np.random.default_rng(seed)
    n, slots = int(rng.integers(1, 40)), int(rng.integers(2, 9))
    seqs = Sequences([int(x) for x in rng.integers(0, 64 * slots // 2, n)], 1, 32, seed,
                     **{**dict(spare=int(rng.integers(0, 60)), extra_slots=slots, layers=int(rng.integers(1, 3))), **more})
    table, lens, refs = seqs.table, np.array(seqs.lens, np.int32), seqs.refs.copy()
    refs[rng.integers(0, seqs.pages, 2)] += 1
    for _ in range(4):
        m = int(rng.integers(1, 50))
        parent = rng.integers(-1, len(table), m)
        add = rng.integers(0, int(rng.choice([2, 2, 100])), m)
        window = int(rng.choice([0, 0, 70]))
        t, ln, r, _ = fork_case(seqs, parent, add, window, 3 if window else 0, refs, table, lens)
        if not ln.any():
            break
        table, lens, refs = t, ln.astype(np.int32), r


@gpu
def test_many_rows_and_pages():
    """Rows and pages past one pass of the table workgroup."""
    n = 1500
    seqs = Sequences([70] * n, 1, 32, spare=3000)
    parent = np.random.default_rng(1).integers(-1, n, 4000)
    fork_case(seqs, parent, np.random.default_rng(2).integers(0, 3, 4000) * (np.random.default_rng(3).random(4000) < 0.3))


@gpu
def test_parents_and_lengths_out_of_range_are_reported():
    dev = rt.device(0)
    seqs = Sequences([100, 64], 1, 32, spare=5)
    pool = seqs.pool()
    for parent, add, lens, table in (([2, 0], [0, 0], None, None), ([-2, 0], [0, 0], None, None), ([0, 1], [-1, 0], None, None),
                                     ([0, 1], [0, 0], [100, 1000], None), ([0, 1], [1, 1], [-5, 64], None),
                                     ([0, 1], [0, 0], None, 77)):
        t = seqs.table.copy()
        if table:
            t[0, 0] = table
        d = OnDevice(dev, seqs, pool, table=t, lens=lens)
        out = d.successor()
        dev.cache_fork(d.cache, out.cache, dev.upload(np.array(parent, np.int32)), dev.upload(np.array(add, np.int32)))
        with pytest.raises(ValueError, match="parents"):
            dev.sync()
        got, ln, _ = out.tables()
        assert got.min() >= -1 and got.max() < seqs.pages and ln.min() >= 0 and ln.max() <= 128


@gpu
def test_numbers_out_of_range_in_a_large_table_are_reported():
    dev = rt.device(0)
    seqs = Sequences([100, 64], 1, 32, spare=5, extra_slots=9000)
    pool, most = seqs.pool(), 64 * seqs.slots
    for parent, add, lens, entry in (([2, 0], [0, 0], None, None), ([-2, 0], [0, 0], None, None), ([0, 1], [-1, 0], None, None),
                                     ([0, 1], [0, 0], [100, most + 1], None), ([0, 1], [1, 1], [-5, 64], None),
                                     ([0, 1], [0, 0], None, seqs.pages), ([0, 1], [0, 0], None, -2)):
        t = seqs.table.copy()
        if entry is not None:
            t[0, 0] = entry
        d = OnDevice(dev, seqs, pool, table=t, lens=lens)
        out = d.successor()
        dev.cache_fork(d.cache, out.cache, dev.upload(np.array(parent, np.int32)), dev.upload(np.array(add, np.int32)))
        with pytest.raises(ValueError, match="parents"):
            dev.sync()
        got, ln, _ = out.tables()
        assert got.min() >= -1 and got.max() < seqs.pages and ln.min() >= 0 and ln.max() <= most


@gpu
@pytest.mark.parametrize("pages,share", [(1, 1.0), (8, 0.0), (8, 0.5), (64, 1.0), (1000, 0.5), (1025, 0.1), (3000, 0.9),
                                         (4096, 0.5), (4097, 0.3), (20000, 0.02), (30000, 0.6)])
@pytest.mark.parametrize("layers,heads,dim", [(1, 1, 32), (3, 2, 64)])
def test_compact(pages, share, layers, heads, dim):
    dev = rt.device(0)
    rng = np.random.default_rng([pages, layers])
    seqs = Sequences([1], heads, dim, layers=layers)
    seqs.pages, seqs.slots = pages, 16
    used = rng.permutation(pages)[:int(pages * share)]
    rows = -(-max(1, len(used)) // 16)
    table = np.full(rows * 16, -1, np.int32)
    table[rng.permutation(rows * 16)[:len(used)]] = used
    table = table.reshape(rows, 16)
    refs = np.zeros(pages, np.int32)
    refs[used] = rng.integers(1, 4, len(used))
    pool = rng.integers(0, 256, (layers, pages, heads, 68 * dim)).astype(np.uint8)
    d = OnDevice(dev, seqs, pool, table, rng.integers(0, 1024, rows), refs)
    out = d.successor()
    moved = dev.upload(np.full(pages, 0x5A5A5A5A, np.int32))
    dev.cache_compact(d.cache, out.cache, moved)
    dev.sync()
    w_table, w_refs, w_map, moves = od.compact(table, refs)
    t, ln, r = out.tables()
    assert np.array_equal(t, w_table) and np.array_equal(r, w_refs) and np.array_equal(ln, d.tables()[1])
    assert np.array_equal(moved.download((pages,), np.int32), w_map)
    want = pool.copy()
    for a, b in moves:
        want[:, b] = pool[:, a]
    assert np.array_equal(d.read_pool(), want)


@gpu
def test_compact_reports_an_entry_that_nothing_counts():
    dev = rt.device(0)
    seqs = Sequences([100], 1, 32)
    d = OnDevice(dev, seqs, seqs.pool(), refs=np.zeros(seqs.pages))
    out = d.successor()
    dev.cache_compact(d.cache, out.cache, dev.alloc(4 * seqs.pages))
    with pytest.raises(ValueError, match="page table"):
        dev.sync()


# ------------------------------------------------------------------------------------------------------ beams

LOGS = np.rint(np.log(np.maximum(1, np.arange(2048))) * 65536).astype(np.int64)


def beams_case(groups, beams, vocab, keep, seed=0, ended=0.0, dead=0.0, allowed=None, eos=-1, spread=30, lut=None, logs=LOGS, step=45426,
               mult=5900, ld=None):
    dev = rt.device(0)
    rng = np.random.default_rng([seed, groups, beams, vocab])
    rows, ld = groups * beams, vocab if ld is None else ld
    x = np.clip(np.rint(rng.normal(0, spread, (rows, ld))), -128, 127).astype(np.int8)
    scores = -rng.integers(0, 1 << 22, rows)
    scores[rng.random(rows) < dead] = od.NO_SCORE
    done = (rng.random(rows) < ended).astype(np.uint8) * 3 if ended else None
    ok = None if allowed is None else (rng.random(vocab) < allowed).astype(np.uint8) * 2
    lut = exp_lut(0.09, 20) if lut is None else lut
    out = [dev.alloc(groups * keep * w) for w in (8, 4, 4, 1)]
    up = lambda a, t: None if a is None else dev.upload(np.asarray(a, t))                            # noqa: E731
    keepalive = [dev.upload(x), up(scores, np.int64), up(done, np.uint8), up(ok, np.uint8), up(lut, np.int32), up(logs, np.int32)]
    xb, sb, db, ab, lb, gb = keepalive
    dev.beam_select(xb, ld, sb, db, ab, groups, beams, vocab, keep, eos, lb, gb, len(logs), step, mult, *out)
    *want, zero = od.beam_select(x[:, :vocab], scores, done, ok, groups, beams, keep, eos, lut, logs, step, mult)
    if zero:
        with pytest.raises(ZeroDivisionError):
            dev.sync()
    else:
        dev.sync()
    for name, buf, w, t in zip(("scores", "parent", "token", "ended"), out, want, (np.int64, np.int32, np.int32, np.uint8)):
        got = buf.download((groups, keep), t)
        assert np.array_equal(got, w), (name, np.argwhere(got != w)[:5], got[:1], w[:1])
    return want


@gpu
@pytest.mark.parametrize("groups,beams,vocab,keep", [(1, 1, 1, 1), (1, 1, 2, 4), (3, 2, 7, 5), (2, 4, 512, 4), (1, 64, 33, 64),
                                                     (5, 3, 1000, 8), (2, 2, 16384, 3), (2, 5, 16385, 64), (1, 3, 50001, 16),
                                                     (1, 8, 65537, 2), (40, 1, 255, 1)])
def test_beams(groups, beams, vocab, keep):
    beams_case(groups, beams, vocab, keep)
    beams_case(groups, beams, vocab, keep, seed=1, ended=0.4, dead=0.3, allowed=0.6, eos=vocab // 2, ld=vocab + 5)


@gpu
@pytest.mark.parametrize("vocab", [50, 3001, 40000])
def test_beams_with_ties_everywhere(vocab):
    """One value, two values, and all logits at an end of int8: the lowest row, then the lowest token."""
    for spread in (0, 0.5, 1e9):
        beams_case(3, 4, vocab, 9, spread=spread)
        beams_case(2, 4, vocab, 9, spread=spread, allowed=0.3)


@gpu
def test_beams_without_candidates():
    for w in (beams_case(2, 3, 40, 4, dead=1.1), beams_case(2, 3, 40, 4, allowed=0.0)):
        assert np.all(w[1] == -1) and np.all(w[2] == -1) and np.all(w[0] == od.NO_SCORE)
    w = beams_case(2, 3, 40, 4, allowed=0.0, ended=1.1, eos=7)
    assert np.all(w[1][:, :3] >= 0) and np.all(w[1][:, 3] == -1)
    beams_case(2, 3, 40, 4, lut=np.zeros(256))
    beams_case(1, 2, 3, 8, allowed=0.7, seed=4)


@gpu
@pytest.mark.parametrize("n", [2, 3, 100, 2048, 5000])
def test_beams_of_any_log_table(n):
    logs = np.rint(np.log(np.maximum(1, np.arange(n))) * 65536).astype(np.int64)
    beams_case(2, 3, 900, 5, logs=logs, lut=exp_lut(0.02, 30))
    beams_case(2, 3, 900, 5, logs=logs, lut=np.random.default_rng(0).integers(-3, 3, 256).clip(max=2) | 1, mult=(1 << 31) - 1)


# ------------------------------------------------------------------------------- graphs, contexts and the workspace

class Work:
    """A call of the attention whose inputs can be changed: run() enqueues it, check() waits and compares."""

    def __init__(self, dev, lens, news, heads_q, heads, dim, seed, one=127):
        self.dev, self.news, self.heads_q, self.dim = dev, news, heads_q, dim
        self.seqs = Sequences(lens, heads, dim, seed=seed)
        self.d = OnDevice(dev, self.seqs, self.seqs.pool())
        self.rows, self.one = sum(news), one
        self.ms, self.ss = fixed(0.4 / np.sqrt(dim) / 40, 128 * 126 * dim)
        self.mo, self.so = fixed(2.0 / one, 126 * (one + max(lens) // 2))
        self.lut, self.starts = dev.upload(exp_lut().astype(np.int32)), dev.upload(starts_of(news))
        self.q, self.out = dev.alloc(self.rows * heads_q * dim), dev.alloc(self.rows * heads_q * dim)
        self.feed(seed)

    def feed(self, seed):
        q = np.random.default_rng([seed, 5]).integers(-128, 128, (self.rows, self.heads_q, self.dim))
        self.q.upload(q.astype(np.int8))
        self.want, _ = attention_want(self.seqs, self.news, q, self.heads_q, self.ms, self.ss, exp_lut(), self.one, self.mo, self.so)

    def run(self):
        w = self.heads_q * self.dim
        self.dev.attention_cache(self.d.cache, 0, self.q, self.out, self.starts, self.rows, max(self.news), self.heads_q,
                                 (w, self.dim, w, self.dim), self.ms, self.ss, self.lut, self.one, self.mo, self.so)

    def check(self):
        self.dev.sync()
        got = self.out.download(self.want.shape, np.int8)
        assert np.array_equal(got, self.want), np.argwhere(got != self.want)[:5]


class Choice:
    """The same for a selection over a vocabulary that takes the workspace."""

    def __init__(self, dev, seed, vocab=20000):
        self.dev, self.vocab = dev, vocab
        self.lut = exp_lut(0.05)
        self.logs = np.rint(np.log(np.maximum(1, np.arange(2048))) * 65536).astype(np.int64)
        self.d_lut, self.d_logs = dev.upload(self.lut.astype(np.int32)), dev.upload(self.logs.astype(np.int32))
        self.x, self.scores = dev.alloc(4 * vocab), dev.upload(np.arange(4, dtype=np.int64))
        self.out = [dev.alloc(6 * n) for n in (8, 4, 4, 1)]
        self.feed(seed)

    def feed(self, seed):
        x = np.random.default_rng([seed, 6]).integers(-128, 128, (4, self.vocab))
        self.x.upload(x.astype(np.int8))
        self.want = od.beam_select(x, np.arange(4), None, None, 2, 2, 3, -1, self.lut, self.logs, 45426, 3277)[:4]

    def run(self):
        self.dev.beam_select(self.x, self.vocab, self.scores, None, None, 2, 2, self.vocab, 3, -1, self.d_lut, self.d_logs, 2048, 45426,
                             3277, *self.out)

    def check(self):
        self.dev.sync()
        for buf, w, t in zip(self.out, self.want, (np.int64, np.int32, np.int32, np.uint8)):
            assert np.array_equal(buf.download((2, 3), t), w)


KINDS = {"tiles": lambda dev, seed: Work(dev, [200, 64], [1, 1], 4, 2, 64, seed),
         "parts": lambda dev, seed: Work(dev, [4200], [1], 4, 1, 128, seed),
         "many rows": lambda dev, seed: Work(dev, [2100, 300], [64, 1], 64, 16, 32, seed),
         "beams": Choice}


@gpu
@pytest.mark.parametrize("kind", ["capture", "sequence"])
def test_replays_with_eager_work_between(kind):
    """Two recordings share the workspace, each other call of the context takes it too, and one that needs a larger one replaces it."""
    dev = rt.Device(0)
    works = [KINDS[k](dev, i) for i, k in enumerate(("parts", "beams", "many rows", "tiles"))]
    for w in works:
        w.run()
        w.check()
    recorded = [getattr(dev, kind)(lambda: [w.run() for w in pair]) for pair in (works[:2], works[2:])]
    for seed in range(4):
        for w in works:
            w.feed(10 + seed)
        for r in recorded:
            r.launch()
        for w in works:
            w.check()
        eager = KINDS["parts" if seed % 2 else "beams"](dev, 20 + seed)
        for w in works:
            w.feed(30 + seed)
        recorded[0].launch()
        eager.run()
        recorded[1].launch()
        recorded[0].launch()
        for w in (eager, *works):
            w.check()
        if seed == 1:                                          # 3 MiB and more of scores, histograms and sums
            big = Work(dev, [20000], [8], 32, 1, 32, 3)
            big.run()
            big.check()
    del recorded
    dev.close()


@gpu
def test_a_captured_step_of_tables_rows_and_attention():
    dev = rt.Device(0)
    seqs = Sequences([63, 64, 1], 2, 32, extra_slots=1, spare=4)
    up = lambda x: dev.upload(np.ascontiguousarray(x))                                                # noqa: E731
    pool, tables = up(seqs.pool()), [up(seqs.table), up(np.array(seqs.lens, np.int32)), up(seqs.refs)]
    cache = rt.Cache(pool, *tables, seqs=3, slots=seqs.slots, pages=seqs.pages, heads=2, dim=32)
    outs = [dev.alloc(4 * seqs.table.size), dev.alloc(12), dev.alloc(4 * seqs.refs.size)]
    stepped = cache.with_tables(*outs)
    ones, lut = up(np.ones(3, np.int32)), up(exp_lut().astype(np.int32))
    k, v, q, o = (dev.alloc(3 * 64) for _ in range(4))
    st = (64, 32, 64, 32)

    def step():
        dev.cache_fork(cache, stepped, None, ones)
        dev.cache_append(stepped, 0, k, v, None, 3, 1, st)
        dev.attention_cache(stepped, 0, q, o, None, 3, 1, 2, st, 3, 10, lut, 127, 1, 7)

    rng = np.random.default_rng(2)
    step()
    dev.sync()
    g = dev.capture(step)
    for _ in range(4):
        rows = [rng.integers(-128, 128, (3, 2, 32)) for _ in range(3)]
        for buf, x in zip((k, v, q), rows):
            buf.upload(x.astype(np.int8))
        g.launch()
        dev.sync()
        want_t, want_n, want_r, _ = od.fork(seqs.table, seqs.lens, seqs.refs, None, [1, 1, 1])
        assert np.array_equal(outs[0].download(want_t.shape, np.int32), want_t)
        assert np.array_equal(outs[1].download((3,), np.int32), want_n)
        assert np.array_equal(outs[2].download(want_r.shape, np.int32), want_r)
        got = o.download((3, 2, 32), np.int8)
        for s, h in np.ndindex(3, 2):
            keys, vals = (od.held(np.concatenate([old[0][s][:, h], new[s, h][None]])) for old, new in ((seqs.k, rows[0]), (seqs.v, rows[1])))
            want, _ = od.attend(rows[2][s, h], keys, vals, seqs.lens[s], np.ones(9, bool), 3, 10, exp_lut(), 127, 1, 7)
            assert np.array_equal(got[s, h], want)
    del g
    dev.close()


@gpu
def test_two_contexts_at_once():
    """Each context has its stream and its workspace: calls from two threads, and interleaved from one."""
    import threading
    devs = [rt.Device(0), rt.Device(0)]
    works = [[KINDS[k](dev, 7 * i + j) for j, k in enumerate(KINDS)] for i, dev in enumerate(devs)]
    for pair in zip(*works):
        for _ in range(3):
            for w in pair:
                w.run()
        for w in pair:
            w.check()
    errors = []

    def loop(ws):
        try:
            for _ in range(5):
                for w in ws:
                    w.run()
                for w in ws:
                    w.check()
        except BaseException as e:                             # noqa: BLE001  (reported by the test's thread)
            errors.append(e)

    threads = [threading.Thread(target=loop, args=(ws,)) for ws in works]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    del works
    for d in devs:
        d.close()
