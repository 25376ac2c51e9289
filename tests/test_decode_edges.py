"""Edges of the decoding operators and of the decoder's bookkeeping, against the same numpy restatement in 64 bits. Every result is an
integer, so every comparison is exact."""
import numpy as np
import pytest

import anvil_mi355x
import test_decode_ops as ops
from anvil_mi355x import decode, driver, models
from anvil_mi355x import ir as g
from anvil_mi355x import runtime as rt
from decode_cases import Sequences
from host_cache import HostDevice
from test_decoder import Oracle

gpu = pytest.mark.gpu


# ------------------------------------------------------------------------------------- tables that do not rise

def _falling(seed, top):
    """A table of large entries whose last one, that of a row's largest score, is `top`: what stands at a score that no key of the row has
    is as much as 2^30 times the sum."""
    lut = np.random.default_rng(seed).integers(1 << 20, 1 << 30, 256)
    lut[255] = top
    return lut


@gpu
@pytest.mark.parametrize("one", [127, 910, 911, 32767])
@pytest.mark.parametrize("heads_q", [1, 4, 5, 8, 9, 16])
@pytest.mark.parametrize("seed", range(4))
def test_attention_tables_whose_unseen_entries_are_large(monkeypatch, seed, heads_q, one):
    """One visible key and a few, with every form of the tiles (up to 4, 8 and 16 rows, narrow and wide digits)."""
    monkeypatch.setitem(ops.LUTS, "falling", _falling(seed, 1 + seed))
    ops.attention_case([1, 1, 1, 1], [1] * 4, heads_q, 1, 32, seed=seed, lut="falling", one=one)
    ops.attention_case([3, 70, 2], [1] * 3, heads_q, 1, 64, seed=seed, lut="falling", one=one)
    ops.attention_case([64, 1], [1] * 2, heads_q, 1, 128, seed=seed, lut="falling", one=one, window=1)
    ops.attention_case([2400], [1], heads_q, 1, 32, seed=seed, lut="falling", one=one, window=2300)


@gpu
@pytest.mark.parametrize("one", [1, 127, 128, 32639, 32640])
@pytest.mark.parametrize("window", [0, 1, 2100])
def test_attention_of_many_rows_with_tables_whose_unseen_entries_are_large(monkeypatch, window, one):
    monkeypatch.setitem(ops.LUTS, "falling", _falling(window, 3))
    for case in ops.MANY:
        ops.attention_case(*case, 32, seed=one, lut="falling", one=one, window=window)


# ------------------------------------------------------------------------------- a cache's steps and their undoing

DEVICES = [pytest.param(HostDevice, id="host"), pytest.param(lambda: rt.device(0), id="device", marks=gpu)]


def _int32s(dev, *x):
    return dev.upload(np.array(x, np.int32))


def _same(got, want):
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g, w)


@pytest.mark.parametrize("device", DEVICES)
def test_a_refused_step_leaves_the_cache_as_it_was(device):
    dev = device()
    cache = decode.KVCache(dev, 1, 1, 32, 12, 4, 200)
    cache.reset(2)
    before = cache.tables()
    add = _int32s(dev, 70, 5)
    cache.step(None, add)
    after = cache.tables()
    for refused in (lambda: cache.step(None, add, rows=4), lambda: cache.step(None, add, rows=1),
                    lambda: dev.cache_fork(cache.cache, cache.cache), lambda: cache.step(None, add, rows=5)):
        with pytest.raises(ValueError):
            refused()
        assert cache.seqs == 2
        _same(cache.tables(), after)
    cache.undo()
    assert cache.seqs == 2
    _same(cache.tables(), before)


def test_a_refused_compaction_leaves_the_cache_as_it_was():
    dev = HostDevice()
    cache = decode.KVCache(dev, 1, 1, 32, 12, 4, 200)
    cache.step(_int32s(dev, 0, 1), None, rows=2)
    moved, cache.moved = cache.moved, None
    with pytest.raises(ValueError, match="map"):
        cache.compact()
    cache.moved = moved
    assert cache.seqs == 2
    cache.undo()
    assert cache.seqs == 4
    dev.sync()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("window", [0, 10])
@pytest.mark.parametrize("recorded", [False, True])
def test_a_step_that_runs_out_of_pages_is_taken_back(device, window, recorded):
    """Parents, added tokens and a window: a step that went well cannot be taken back, one that found too few pages can."""
    dev = device()
    cache = decode.KVCache(dev, 2, 1, 32, 5, 3, 256, window=window)
    cache.reset(2)
    cache.step(None, _int32s(dev, 64, 60))
    parent, one, many = _int32s(dev, 0, 1, 1), _int32s(dev, 1, 1, 1), _int32s(dev, 1, 130, 130)
    cache.step(parent, one, 3)
    dev.sync()
    before = cache.tables()
    with pytest.raises(ValueError, match="taken back"):
        cache.undo()
    _same(cache.tables(), before)
    if recorded:                                               # what KVCache.step calls, then the word that it has run
        dev.cache_fork(cache.cache, cache._cache(1 - cache._at, 3), None, many, window, 0)
        cache.stepped(3)
    else:
        cache.step(parent, many, 3)
    with pytest.raises(MemoryError):
        dev.sync()
    assert not cache.tables()[1].any()
    cache.undo()
    _same(cache.tables(), before)
    with pytest.raises(ValueError, match="taken back"):        # once
        cache.undo()
    cache.step(_int32s(dev, -1, 1, -1), None, 3)               # a row stays, and the step fits
    cache.step(None, _int32s(dev, 0, 130, 0))
    dev.sync()
    assert cache.tables()[1].tolist() == [0, 191, 0]


@pytest.mark.parametrize("device", DEVICES)
def test_a_step_that_empties_every_row_is_not_mistaken_for_a_failed_one(device):
    """Rows given back and none extended, with `add` at hand: references tell it from a step that found no pages."""
    dev = device()
    cache = decode.KVCache(dev, 1, 1, 32, 5, 2, 256)
    cache.step(None, _int32s(dev, 64, 60))
    cache.step(_int32s(dev, -1, -1), _int32s(dev, 1, 1), 2)
    dev.sync()
    assert not cache.tables()[1].any() and not cache.tables()[2].any()
    with pytest.raises(ValueError, match="taken back"):
        cache.undo()
    cache.reset()
    cache.step(_int32s(dev, -1, 1), _int32s(dev, 1, 0), 2)     # nothing was there: nothing is written or given back
    cache.undo()
    assert cache.seqs == 2


# ------------------------------------------------------------------------------------------- the decoder's buffers

class _Short(HostDevice):
    """A device with room for so many more allocations."""
    left = 1 << 30

    def alloc(self, nbytes):
        if not self.left:
            raise RuntimeError("anvil_alloc: out of memory")
        self.left -= 1
        return super().alloc(nbytes)

    def zero(self, buf, nbytes):
        buf.bytes[:nbytes] = 0


@pytest.mark.parametrize("left", range(4))
def test_buffers_that_could_not_grow_are_not_taken_for_grown(left):
    """A call that runs out of memory while it makes room must leave the next one to make it."""
    dec = object.__new__(decode.Decoder)
    dec.dev, dec._room, dec._buffers = _Short(), 0, []
    dec._values = [decode._Rows(32, "i8"), decode._Rows(48, "i16"), decode._Rows(7, "i8")]

    def holds(rows):
        return all(v.buf is not None and v.buf.nbytes >= rows * v.width * rt.ITEMSIZE[v.dtype] for v in dec._values)

    dec._make_room(5)
    assert holds(5)
    small = [v.buf for v in dec._values]
    dec.dev.left = left
    if left < len(dec._values):
        with pytest.raises(RuntimeError, match="out of memory"):
            dec._make_room(100)
    else:
        dec._make_room(100)
    dec.dev.left = 1 << 30
    dec._make_room(5)
    assert holds(5) and holds(dec._room)
    dec._make_room(100)
    assert holds(100) and holds(dec._room)
    assert all(any(b is x for x in dec._buffers) for b in small)                   # recorded launches may name them


# ------------------------------------------------------------------------------------------------- large pools

@gpu
def test_compaction_of_a_pool_of_few_large_pages():
    """4096 heads of 128 are 8704 workgroups a page and layer: with 1000 layers the launch has more threads than an int holds. Two pages,
    of which the second moves; the bytes looked at are the first and the last layer's."""
    dev = rt.Device(0)
    heads, dim, layers, pages, slots = 4096, 128, 1000, 2, 16384
    page = heads * 68 * dim
    pool = dev.alloc(dev.cache_bytes(layers, pages, heads, dim))
    rng = np.random.default_rng(0)
    first, last = (rng.integers(0, 256, page).astype(np.uint8) for _ in range(2))
    pool.upload(first, page)
    pool.upload(last, (2 * layers - 1) * page)
    table = np.full((40, slots), -1, np.int32)
    table[[0, 39], [5, slots - 1]] = 1
    lens = np.arange(40, dtype=np.int32)
    cache = rt.Cache(pool, t := dev.upload(table), n := dev.upload(lens), r := dev.upload(np.array([0, 2], np.int32)), seqs=40,
                     slots=slots, pages=pages, heads=heads, dim=dim, layers=layers)
    out = [dev.upload(np.full(x, 0x5A5A5A5A, np.int32)) for x in (table.size, 40, pages)]
    moved = dev.alloc(4 * pages)
    dev.cache_compact(cache, cache.with_tables(*out), moved)
    dev.sync()
    assert np.array_equal(out[0].download(table.shape, np.int32), np.where(table < 0, -1, 0))
    assert np.array_equal(out[1].download((40,), np.int32), lens)
    assert out[2].download((2,), np.int32).tolist() == [2, 0] and moved.download((2,), np.int32).tolist() == [-1, 0]
    assert np.array_equal(pool.download((page,), np.uint8), first)
    assert np.array_equal(pool.download((page,), np.uint8, (2 * layers - 2) * page), last)
    del t, n, r
    dev.close()


# ------------------------------------------------------------------------------------------ what can be decoded

def _attention_graph(m_s=1, s_s=9):
    """One head of 32 over 32 tokens, queries within 4 of zero by their table, so that the proof allows a large score multiplier."""
    bld = g.GraphBuilder("m")
    x, w, lut = bld.input("x", [32, 32], "i8", 0.1), bld.const("w", [32, 32], "i8"), bld.const("lut", [256], "i32")
    q = bld.qlinear("q", x, w, 1, 5, lut=bld.const("near", [256], "i8"))
    k, v = (bld.qlinear(n, x, w, 1, 5) for n in "kv")
    s = bld.qmatmul("s", q, bld.transpose("kt", k, [1, 0]), m_s, s_s)
    bld.output(bld.qmatmul("o", bld.softmax_lut("p", s, lut, 127, True), v, 1, 7))
    consts = {"w": np.eye(32, dtype=int), "near": np.arange(-128, 128) // 32, "lut": np.r_[np.zeros(250, int), 1, 2, 4, 9, 20, 40]}
    return anvil_mi355x.compile((bld.module(), consts), embedding=(np.zeros((32, 32)), np.zeros((32, 32))))


def test_a_score_multiplier_that_the_cache_cannot_take_is_refused_at_once():
    """128 * 126 * 32 * |m| + 2^(s-1) < 2^31, or the attention over the cache refuses every call."""
    most = ((1 << 31) - 1 - (1 << 8)) // (128 * 126 * 32)
    for m in (most + 1, -most - 1):
        cm = _attention_graph(m)
        assert cm.proven
        with pytest.raises(OverflowError, match="multiplier"):
            cm.decoder(rows=1)


@gpu
def test_the_largest_score_multiplier_is_taken():
    cm = _attention_graph(((1 << 31) - 1 - (1 << 8)) // (128 * 126 * 32))
    dec, dev = cm.decoder(rows=1), cm.dev
    dec.cache.step(None, _int32s(dev, 1))
    dec.forward(_int32s(dev, 0), None, 1, 1)
    dev.sync()


def _long_model(seq):
    return models.build(models.BlockSpec(n_embd=32, n_head=2, seq=seq, layers=1, vocab=40, calib_batches=1, calib_batch=1), 6, stored=False)


def test_attention_of_more_tokens_than_the_whole_sequence_kernel_takes_is_decoded():
    """That kernel's 1024 tokens are no limit of the cache: the lowering finds the chain, and the whole graph's plan still has none."""
    cm = anvil_mi355x.compile(_long_model(1040))
    assert cm.proven and not cm._attention_chains("outputs")
    dec = object.__new__(decode.Decoder)
    dec.cm, dec.T = cm, 1040
    steps, layers, heads, dim = dec._lower()
    assert (layers, heads, dim) == (1, 2, 16) and [s[0] for s in steps].count("attend") == 1


@gpu
def test_a_model_of_1040_tokens_gives_the_graphs_logits():
    b = _long_model(1040)
    cm = anvil_mi355x.compile(b)
    dec, dev = cm.decoder(rows=1), cm.dev
    seq = np.random.default_rng(3).integers(0, 40, 1040).astype(np.int32)
    want = Oracle(b).logits([seq])[0]
    for lo, n in ((0, 1030), (1030, 7), *((t, 1) for t in range(1037, 1040))):
        dec.cache.step(None, _int32s(dev, n))
        ids = dev.upload(seq[lo:lo + n])
        got = dec.forward(ids, starts := _int32s(dev, 0, n), n, n).download((n, 40), np.int8)
        dev.sync()
        np.testing.assert_array_equal(got, want[lo:lo + n])
    del starts


# -------------------------------------------------------------------------------------------- results over queries

def _attend_within(dev, at_q, at_o, strides, rows=3, heads=2, dim=32, size=4096):
    """An attention call whose queries and results lie in one buffer, at byte offsets; returns (results, expected, the other bytes
    before and after)."""
    seqs = ops.Sequences([100, 70, 9][:rows], heads, dim)
    d = ops.OnDevice(dev, seqs, seqs.pool())
    raw = np.random.default_rng(1).integers(-128, 128, size).astype(np.int8)
    buf = dev.upload(raw)
    where = lambda at, row, head: at + (row * np.arange(rows)[:, None, None] + head * np.arange(heads)[:, None] + np.arange(dim))  # noqa: E731
    q_at, o_at = where(at_q, *strides[:2]), where(at_o, *strides[2:])
    lut = dev.upload(ops.exp_lut().astype(np.int32))
    dev.attention_cache(d.cache, 0, buf.ptr + at_q, buf.ptr + at_o, None, rows, 1, heads, strides, 5, 16, lut, 127, 1, 7)
    dev.sync()
    want, _ = ops.attention_want(seqs, [1] * rows, raw[q_at].astype(np.int64), heads, 5, 16, ops.exp_lut(), 127, 1, 7)
    got = buf.download((size,), np.int8)
    rest = np.setdiff1d(np.arange(size), o_at)
    return got[o_at], want, raw[rest], got[rest]


@gpu
@pytest.mark.parametrize("at_q,at_o,strides", [(0, 192, (64, 32, 64, 32)), (256, 0, (64, 32, 64, 32)),          # one behind the other
                                               (0, 64, (128, 32, 128, 32)), (64, 0, (128, 32, 128, 32)),       # beside each other
                                               (0, 32, (128, 64, 128, 64)), (128, 32, (512, 256, 512, 64)),    # heads between heads
                                               (2048, 0, (-64, 32, 64, 32)), (0, 1024, (0, 0, 64, 32))])
def test_queries_and_results_of_one_buffer(at_q, at_o, strides):
    got, want, before, after = _attend_within(rt.device(0), at_q, at_o, strides)
    assert np.array_equal(got, want) and np.array_equal(before, after)


@gpu
@pytest.mark.parametrize("at_q,at_o,strides", [(64, 64, (512, 0, 512, 32)), (0, 0, (64, 32, 64, 32)), (0, 188, (64, 32, 64, 32)), (176, 0, (64, 32, 64, 32)),
                                               (0, 60, (128, 32, 128, 32)), (64, 4, (128, 32, 128, 32)), (0, 124, (128, 32, 128, 32)),
                                               (0, 36, (128, 64, 128, 64)), (0, 64, (128, 32, 192, 32)), (256, 0, (-64, 32, 64, 32)),
                                               (128, 0, (0, 0, 64, 32)), (0, 64, (64, 32, 64, 32)), (1024, 0, (64, 32, 1024, 32))])
def test_results_over_queries_are_refused(at_q, at_o, strides):
    """At the ends of both extents, in the rows between, and with strides that differ."""
    with pytest.raises(ValueError, match="O overlaps Q"):
        _attend_within(rt.device(0), at_q, at_o, strides)


# ------------------------------------------------------------------------------------------ calls that fail part way

class _Watched(HostDevice):
    settled = 0

    def fetch(self, items):
        def call(check=False):
            self.settled += 1
            if check:
                self.sync()
        return call


@pytest.mark.parametrize("error", [RuntimeError("anvil_alloc: out of memory"), KeyboardInterrupt()], ids=["error", "interrupt"])
def test_a_call_that_fails_part_way_leaves_no_violation_on_the_device(error):
    """Too few pages, which the call's end would report, and an error before that end: the next call on the device is not the one to
    report them, and no kernel runs any more when the call's buffers go."""
    dec = object.__new__(decode.Decoder)
    dec.dev = dev = _Watched()
    dec.cm = object.__new__(driver.CompiledModel)
    dec.cm.dev = dev
    dec.rows, dec.max_tokens, dec.vocab, dec.logits, dec.scale = 2, 300, 40, decode._Rows(40, "i8"), 0.1
    dec.cache = decode.KVCache(dev, 1, 1, 32, 3, 2, 300)
    dec._make_room = lambda rows: None

    def forward(*args):
        assert isinstance(dev.pending, MemoryError)
        raise error

    dec.forward = forward
    with pytest.raises(type(error)):
        dec.generate([[1] * 200, [2] * 100], 4)
    assert dev.settled
    dev.sync()


# ------------------------------------------------------------------------- short sequences in tables of many slots

@gpu
@pytest.mark.parametrize("slots", [150, 2100, 16000])
@pytest.mark.parametrize("lens,news,heads_q,heads,dim", [([130, 1, 0, 65], [1, 1, 0, 1], 4, 2, 64), ([3], [1], 8, 8, 32), ([700], [1], 4, 1, 128),
                                                         ([190, 70], [6, 1], 4, 4, 64), ([300, 300], [100, 1], 12, 2, 16),
                                                         ([260, 5], [256, 3], 8, 8, 32)])
def test_attention_of_short_sequences_in_tables_of_many_slots(monkeypatch, slots, lens, news, heads_q, heads, dim):
    """What a table could hold decides how a call is split: parts, tiles whose scores lie in memory, many rows, and here most of it is
    empty."""
    monkeypatch.setattr(ops, "Sequences", lambda *a, **k: Sequences(*a, **k, extra_slots=slots))
    ops.attention_case(lens, news, heads_q, heads, dim, one=127)
    ops.attention_case(lens, news, heads_q, heads, dim, one=4096, window=100, sinks=5)
    ops.attention_case(lens, news, heads_q, heads, dim, one=911, window=40000, sinks=70)


@gpu
@pytest.mark.parametrize("fails", ["alloc", "workspace"])
def test_a_call_after_an_allocation_that_failed(fails):
    """Memory that the device has not is an error of the call that asked for it, and of no later one."""
    dev = rt.Device(0)
    work = ops.KINDS["parts"](dev, 1)
    small = ops.Choice(dev, 2, vocab=300)
    with pytest.raises(RuntimeError):
        if fails == "alloc":
            dev.alloc(1 << 50)
        else:                                                  # 2^22 rows of 2^28 logits: 2^46 bytes of histograms, before any is read
            dev.beam_select(small.x, 1 << 28, small.scores, None, None, 1 << 16, 64, 1 << 28, 64, -1, small.d_lut, small.d_logs, 2048, 1, 1,
                            *[small.x.ptr + (i << 40) for i in (1, 2, 3, 4)])
    small.run()
    work.run()
    work.check()
    small.check()
    dev.close()
