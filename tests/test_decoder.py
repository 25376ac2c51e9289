"""CompiledModel.decoder: a token model token by token over the 4-bit cache, against the whole graph evaluated by the oracle with
k and v rounded to what the cache holds. Everything is exact: the logits, the selection's scores, the tokens."""
import numpy as np
import pytest

import anvil_mi355x
import helpers
from anvil_mi355x import decode, models
from anvil_mi355x import ir as g
from anvil_mi355x import runtime as rt
from oracle import decode as od
from oracle import interp

gpu = pytest.mark.gpu

SPECS = {
    "heads of 32": models.BlockSpec(n_embd=128, n_head=4, seq=128, layers=2, vocab=512, calib_batches=1, calib_batch=2),
    "heads of 16, lut op": models.BlockSpec(n_embd=64, n_head=4, seq=80, layers=1, vocab=131, gelu="op", calib_batches=1,
                                            calib_batch=2),
    "one head of 64": models.BlockSpec(n_embd=64, n_head=1, seq=70, layers=3, vocab=67, calib_batches=1, calib_batch=2),
}
_built = {}


def built(name):
    if name not in _built:
        _built[name] = models.build(SPECS[name], 5, stored=False)
    return _built[name]


class Oracle:
    """The whole graph for every token, k and v as the cache holds them."""

    def __init__(self, b, window=0, sinks=0):
        self.b, self.window, self.sinks = b, window, sinks
        self.ops = {op.sym_str: op for op in g.func_of(b.module).ops if op.results}
        H, C = b.spec.n_head, b.spec.n_embd
        self.replace = {}
        hold = lambda x, _: od.held(x.reshape(*x.shape[:-1], H, C // H)).reshape(x.shape)       # noqa: E731
        for i in range(b.spec.layers):
            self.replace[f"L{i}.k"] = self.replace[f"L{i}.v"] = hold
            if window:
                self.replace[f"L{i}.o"] = self._windowed(f"L{i}.")

    def _windowed(self, L):
        s_op, sm, o_op = (self.ops[L + n] for n in ("scores", "p", "o"))
        H = self.b.spec.n_head
        lut = self.b.consts[L + "p.exp_lut"]

        def f(o, values):
            N, _, T, d = o.shape
            q, k, v = (values[L + n].reshape(N, T, H, d).transpose(0, 2, 1, 3) for n in "qkv")
            out = np.zeros_like(o)
            for n, h, t in np.ndindex(N, H, T):
                out[n, h, t], _ = od.attend(q[n, h, t], k[n, h, :t + 1], v[n, h, :t + 1], t, np.ones(T, bool), int(s_op.M),
                                            int(s_op.s), lut, int(sm.one), int(o_op.M), int(o_op.s), self.window, self.sinks)
            return out
        return f

    def logits(self, sequences):
        """The logits (tokens, vocab) of every sequence."""
        b, T = self.b, self.b.spec.seq
        ids = np.zeros((len(sequences), T), np.int64)
        for i, s in enumerate(sequences):
            ids[i, :len(s)] = s
        x = np.clip(np.rint(models.embed(b.spec, b.params, ids) / b.scales["x"]), -128, 127).astype(np.int64)
        out = interp.run(b.module, {"x": x}, b.consts, batch=True, fast=True, replace=self.replace).outputs[0]
        return [out[i, :len(s)] for i, s in enumerate(sequences)]

    def generate(self, prompts, new_tokens, beams, eos=None, allowed=None):
        sel = decode.Selection.of(self.b.scales["logits"])
        P = len(prompts)
        seqs, scores, ended = [list(p) for p in prompts], np.zeros(P, np.int64), np.zeros(P, np.uint8)
        width = 1
        for _ in range(new_tokens):
            live = [i for i, s in enumerate(scores) if s != od.NO_SCORE]
            logits = np.zeros((len(seqs), self.b.spec.vocab), np.int64)
            for i, x in zip(live, self.logits([seqs[i] for i in live])):
                logits[i] = x[-1]
            s, parent, token, e, _ = od.beam_select(logits, scores, ended, allowed, P, width, beams, -1 if eos is None else eos,
                                                    sel.lut, sel.logs.astype(int), sel.step, sel.mult)
            seqs = [seqs[p] + [int(t)] if p >= 0 else [] for p, t in zip(parent.reshape(-1), token.reshape(-1))]
            scores, ended, width = s.reshape(-1), e.reshape(-1), beams
        tokens = [[_cut(seqs[p * beams + b][len(prompts[p]):], eos) for b in range(beams)
                   if scores[p * beams + b] != od.NO_SCORE] for p in range(P)]
        return tokens, scores.reshape(P, beams)


def _cut(tokens, eos):
    return tokens[:tokens.index(eos) + 1] if eos in tokens else tokens


def prompts_of(spec, lens, seed):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, spec.vocab, n).tolist() for n in lens]


def same(got, want):
    tokens, scores = want
    assert got.tokens == tokens
    np.testing.assert_array_equal(got.scores, np.where(scores == od.NO_SCORE, -np.inf, scores / 65536))


@gpu
@pytest.mark.parametrize("name", SPECS)
def test_prompts_then_single_tokens_give_the_graphs_logits(name):
    b = built(name)
    cm = anvil_mi355x.compile(b)
    T, V = b.spec.seq, b.spec.vocab
    dec = cm.decoder(rows=4)
    seqs = prompts_of(b.spec, [T, 1, T - 3, 65], 1)
    want = Oracle(b).logits(seqs)
    dev = cm.dev
    for cut in ([T - 4, 0, 64, 60], [1, 1, 63, 64]):
        dec.cache.reset()
        at = np.zeros(4, int)
        for new in (np.array(cut), None):                       # the prompts; then a row a sequence until each is whole
            while True:
                n = new if new is not None else (at < [len(s) for s in seqs]).astype(int)
                if not n.any():
                    break
                starts = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
                ids = np.concatenate([s[a:a + k] for s, a, k in zip(seqs, at, n)]).astype(np.int32)
                add, ids, d_starts = dev.upload(n.astype(np.int32)), dev.upload(ids), dev.upload(starts)
                dec.cache.step(None, add)
                out = dec.forward(ids, d_starts, int(starts[-1]), int(n.max())).download((int(starts[-1]), V), np.int8)
                dev.sync()
                for s in range(4):
                    np.testing.assert_array_equal(out[starts[s]:starts[s + 1]], want[s][at[s]:at[s] + n[s]])
                at += n
                if new is not None:
                    break


@gpu
@pytest.mark.parametrize("name", ["v1", "v2"])
def test_the_frozen_models_over_an_embedding(name):
    """Gated MLPs, and in v2 an i16 residual stream with wide norms: the reference's frozen models behind random token tables."""
    text, consts, _ = helpers.reference_model(name)
    m = anvil_mi355x.parse_ir(text)
    rng = np.random.default_rng(4)
    loud = 1.5 if name == "v1" else 5.0
    wte, wpe = (rng.normal(0, loud, (n, 32)).astype(np.float32) for n in (40, 16))
    cm = anvil_mi355x.compile((m, consts), embedding=(wte, wpe))
    ids = rng.integers(0, 40, (3, 16))
    lo, hi = (-128, 127) if name == "v1" else (-32768, 32767)
    x = np.clip(np.rint((wte.astype(np.float64)[ids] + wpe) / cm.scale("x")), lo, hi).astype(np.int64)
    hold = lambda v, _: od.held(v.reshape(3, 16, 2, 16)).reshape(v.shape)                       # noqa: E731
    want = interp.run(m, {"x": x}, consts, batch=True, replace={f"L{i}.{n}": hold for i in range(2) for n in "kv"}).outputs[0]
    dec, dev = cm.decoder(rows=3), cm.dev
    at = np.zeros(3, int)
    for n in ([5, 1, 12], [0, 4, 3], *[[1, 1, 0]] * 11):
        n = np.minimum(n, 16 - at)
        starts = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        rows = int(starts[-1])
        add, new, d_starts = (dev.upload(np.asarray(v, np.int32)) for v in (
            n, np.concatenate([ids[s, at[s]:at[s] + n[s]] for s in range(3)]), starts))
        dec.cache.step(None, add)
        got = dec.forward(new, d_starts, rows, int(max(n))).download((rows, 32), np.int8 if name == "v1" else np.int16)
        dev.sync()
        for s in range(3):
            np.testing.assert_array_equal(got[starts[s]:starts[s + 1]], want[s, at[s]:at[s] + n[s]])
        at += n
    assert at.tolist() == [16, 16, 15]
    if name == "v2":
        with pytest.raises(ValueError, match="int8 logits"):
            dec.generate([[1]], 1)


@gpu
@pytest.mark.parametrize("beams,new_tokens", [(1, 1), (1, 9), (2, 2), (4, 7), (3, 4)])
@pytest.mark.parametrize("name", SPECS)
def test_generate_equals_the_oracles_beam_search(name, beams, new_tokens):
    b = built(name)
    dec = anvil_mi355x.compile(b).decoder(rows=3 * beams)
    T = b.spec.seq
    prompts = prompts_of(b.spec, [1, T - new_tokens + 1, 59], 2)
    same(dec.generate(prompts, new_tokens, beams), Oracle(b).generate(prompts, new_tokens, beams))
    again = prompts_of(b.spec, [64, 3], 3)                      # another call of the same decoder: nothing is left over
    same(dec.generate(again, 6, beams), Oracle(b).generate(again, 6, beams))
    refs = dec.cache.tables()[2]
    table, lens, _ = dec.cache.tables()
    np.testing.assert_array_equal(refs, np.bincount(table[table >= 0], minlength=refs.size))


@gpu
def test_ended_beams_allowed_tokens_and_fewer_candidates_than_beams():
    b = built("heads of 16, lut op")
    V = b.spec.vocab
    dec = anvil_mi355x.compile(b).decoder(rows=12)
    prompts = prompts_of(b.spec, [5, 20], 4)
    free, _ = Oracle(b).generate(prompts, 8, 4)
    eos = free[0][1][2]                                        # a token that some beam takes in its third step
    allowed = np.arange(V) % 3 != 1
    allowed[eos] = True
    for kw in (dict(eos=eos), dict(eos=eos, allowed=allowed), dict(allowed=np.arange(V) == 7),
               dict(eos=3, allowed=np.isin(np.arange(V), [3, 7, 90])), dict(allowed=np.zeros(V, bool))):
        same(dec.generate(prompts, 8, 4, **kw), Oracle(b).generate(prompts, 8, 4, kw.get("eos"), kw.get("allowed")))


@gpu
@pytest.mark.parametrize("window,sinks", [(5, 0), (30, 2), (64, 64)])
def test_a_window_sees_its_tokens_and_gives_pages_back(window, sinks):
    spec = models.BlockSpec(n_embd=32, n_head=1, seq=200, layers=1, vocab=40, calib_batches=1, calib_batch=2)
    b = models.build(spec, 6, stored=False)
    dec = anvil_mi355x.compile(b).decoder(rows=2, window=window, sinks=sinks)
    prompts = prompts_of(spec, [170, 60], 5)
    same(dec.generate(prompts, 12, 1), Oracle(b, window, sinks).generate(prompts, 12, 1))
    table, lens, _ = dec.cache.tables()
    first = (lens - window) // 64                              # pages before it hold no token that the next query sees
    for s in range(2):
        gone = [j for j in range(first[s]) if 64 * j >= sinks and 64 * j + 63 <= lens[s] - 1 - window]
        assert (table[s, gone] == -1).all() and (s or gone or sinks)


@gpu
def test_a_step_is_taken_back_and_the_pool_compacted():
    b = built("heads of 32")
    cm = anvil_mi355x.compile(b)
    dec, dev = cm.decoder(rows=3), cm.dev
    seqs = prompts_of(b.spec, [100, 70, 90], 7)
    want = Oracle(b).logits(seqs)
    ids = lambda lo, n: dev.upload(np.concatenate([s[lo:lo + n] for s in seqs]).astype(np.int32))      # noqa: E731
    count = lambda *n: dev.upload(np.array(n, np.int32))                                               # noqa: E731
    adds, starts = count(64, 64, 64), count(0, 64, 128, 192)
    dec.cache.step(None, adds)
    dec.forward(ids(0, 64), starts, 192, 64)
    before = dec.cache.tables()
    one = count(1, 1, 1)
    dec.cache.step(None, one)
    dec.cache.undo()
    for x, y in zip(before, dec.cache.tables()):
        np.testing.assert_array_equal(x, y)
    with pytest.raises(ValueError, match="taken back"):
        dec.cache.undo()
    parent = count(-1, 1, 2)                                   # a row is freed, its pages are holes, the others move
    dec.cache.step(parent, None)
    dec.cache.compact()
    table, lens, refs = dec.cache.tables()
    assert refs[:2].tolist() == [1, 1] and not refs[2:].any() and lens.tolist() == [0, 64, 64]
    toks = [ids(64 + t, 1) for t in range(3)]
    only = count(0, 1, 1)
    for t in range(3):
        dec.cache.step(None, only)
        out = dec.forward(toks[t], None, 3, 1).download((3, b.spec.vocab), np.int8)
        dev.sync()
        for s in (1, 2):
            np.testing.assert_array_equal(out[s], want[s][64 + t])


@gpu
def test_recorded_steps_outlive_larger_calls():
    b = built("heads of 32")
    cm = anvil_mi355x.compile(b)
    dec, dev = cm.decoder(rows=2), cm.dev
    seqs = prompts_of(b.spec, [40, 40], 11)
    want = Oracle(b).logits(seqs)
    toks, ones = dev.upload(np.zeros(2, np.int32)), dev.upload(np.ones(2, np.int32))

    def step():
        dec.cache.step(None, ones)
        return dec.forward(toks, None, 2, 1)

    def feed(t):
        toks.upload(np.array([s[t] for s in seqs], np.int32))

    def check(t):
        dev.sync()
        got = logits.download((2, b.spec.vocab), np.int8)
        np.testing.assert_array_equal(got, [w[t] for w in want])

    for t in range(2):                                         # one with each set of tables
        feed(t)
        logits = step()
        check(t)
    recorded = []
    for t in range(2, 4):
        feed(t)
        recorded.append(dev.sequence(step))
        check(t)
    other = cm.decoder(rows=2)
    prompts = prompts_of(b.spec, [100, 90], 12)
    for t in range(4, 12):
        feed(t)
        recorded[t % 2].launch()
        dec.cache.stepped(2)
        check(t)
        if t == 6:                                             # larger buffers, a larger workspace
            dec._make_room(500)
            same(other.generate(prompts, 3, 1), Oracle(b).generate(prompts, 3, 1))


@gpu
def test_too_few_pages_are_reported():
    b = built("heads of 32")
    dec = anvil_mi355x.compile(b).decoder(rows=2, pages=3)
    prompts = prompts_of(b.spec, [64, 64], 8)
    assert len(dec.generate(prompts, 1).tokens) == 2
    with pytest.raises(MemoryError, match="page"):
        dec.generate(prompts, 3)
    assert len(dec.generate(prompts, 1).tokens) == 2           # the decoder goes on


@gpu
def test_the_embedding_of_new_tokens():
    dev = rt.device(0)
    rng = np.random.default_rng(9)
    V, C, positions = 11, 37, 90
    wte, wpe = rng.normal(0, 30, (V, C)).astype(np.float32), rng.normal(0, 30, (positions, C)).astype(np.float32)
    d_wte, d_wpe = dev.upload(wte), dev.upload(wpe)
    lens, n = np.array([90, 1, 0, 7], np.int32), [5, 1, 0, 7]
    starts = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    ids = rng.integers(0, V, 15).astype(np.int32)
    table = np.full((4, 2), -1, np.int32)
    d_table, d_lens, d_starts, d_ids = (dev.upload(x) for x in (table, lens, starts, ids))
    pool = dev.alloc(dev.cache_bytes(1, 1, 1, 32))
    cache = rt.Cache(pool, d_table, d_lens, seqs=4, slots=2, pages=1, heads=1, dim=32)
    pos = np.concatenate([np.arange(l - k, l) for l, k in zip(lens, n)])
    for dtype, scale in (("i8", 0.75), ("i16", 0.001)):
        want = np.rint((wte.astype(np.float64)[ids[:13]] + wpe.astype(np.float64)[pos]) / scale)
        info = np.iinfo(rt.NP_DTYPE[dtype])
        out = dev.upload(np.full((15, C), 99, rt.NP_DTYPE[dtype]))
        dev.embed_quantize_new(cache, d_ids, d_starts, 15, 7, C, d_wte, V, d_wpe, positions, scale, out, dtype)
        dev.sync()
        got = out.download((15, C), rt.NP_DTYPE[dtype])
        np.testing.assert_array_equal(got[:13], np.clip(want, info.min, info.max))
        assert (got[13:] == 99).all()
        dev.embed_quantize_new(cache, d_ids, None, 4, 1, C, d_wte, V, d_wpe, positions, scale, out, dtype)
        dev.sync()
        got = out.download((15, C), rt.NP_DTYPE[dtype])         # a row a sequence; the empty one's is left as it was
        for s in (0, 1, 3):
            one = np.rint((wte.astype(np.float64)[ids[s]] + wpe.astype(np.float64)[lens[s] - 1]) / scale)
            np.testing.assert_array_equal(got[s], np.clip(one, info.min, info.max))
        np.testing.assert_array_equal(got[2], np.clip(want, info.min, info.max)[2])
    for bad, positions_ in ((-1, positions), (V, positions), (0, 60)):
        ids2 = ids.copy()
        ids2[0] = bad
        d_bad = dev.upload(ids2)
        dev.embed_quantize_new(cache, d_bad, None, 4, 1, C, d_wte, V, d_wpe, positions_, 0.75, out, "i8")
        with pytest.raises(ValueError):
            dev.sync()
        assert not out.download((15, C), np.int8)[0].any()


def test_models_that_cannot_be_decoded_are_refused():
    b = built("heads of 16, lut op")
    cm = anvil_mi355x.compile(b)
    for kw, what in ((dict(rows=0), "rows"), (dict(rows=1, max_tokens=81), "max_tokens"), (dict(rows=1, max_tokens=0), "max_tokens"),
                     (dict(rows=1, window=-1), "window"), (dict(rows=4097), "rows")):
        with pytest.raises(ValueError, match=what):
            cm.decoder(**kw)
    cm.embedding = None
    with pytest.raises(ValueError, match="embedding"):
        cm.decoder(rows=1)
    spec = models.BlockSpec(n_embd=64, n_head=4, seq=32, layers=1, vocab=40, causal=False, calib_batches=1, calib_batch=2)
    with pytest.raises(ValueError, match="causal"):
        anvil_mi355x.compile(models.build(spec, 5, stored=False)).decoder(rows=1)
    spec = models.BlockSpec(n_embd=64, n_head=4, seq=32, layers=1, calib_batches=1, calib_batch=2)
    with pytest.raises(ValueError, match="embedding"):
        anvil_mi355x.compile(models.build(spec, 5, stored=False)).decoder(rows=1)
    with pytest.raises(ValueError, match="proof"):
        anvil_mi355x.compile((b.module, b.consts), prove=False, embedding=(b.params["wte"], b.params["wpe"])).decoder(rows=1)


def test_graphs_that_are_not_row_by_row_are_refused():
    def graph(build):
        bld = g.GraphBuilder("m")
        x = bld.input("x", [32, 32], "i8", 0.1)
        w = bld.const("w", [32, 32], "i8")
        lut = bld.const("lut", [256], "i32")
        consts = {"w": np.eye(32, dtype=int), "lut": np.r_[np.zeros(250, int), 1, 2, 4, 9, 20, 40]}
        bld.output(build(bld, x, w, lut))
        return anvil_mi355x.compile((bld.module(), consts), embedding=(np.zeros((32, 32)), np.zeros((32, 32))))

    def attention(bld, x, w, lut, q=None, causal=True):
        q = bld.qlinear("q", x, w, 1, 5) if q is None else q
        k, v = bld.qlinear("k", x, w, 1, 5), bld.qlinear("v", x, w, 1, 5)
        s = bld.qmatmul("s", q, bld.transpose("kt", k, [1, 0]), 1, 9)
        return bld.qmatmul("o", bld.softmax_lut("p", s, lut, 127, causal), v, 1, 7)

    def rows_turned(bld, x, w, lut):
        return bld.qlinear("y", bld.transpose("t", attention(bld, x, w, lut), [1, 0]), w, 1, 5)

    def queries_turned(bld, x, w, lut):
        return attention(bld, x, w, lut, bld.transpose("qt", bld.qlinear("q", x, w, 1, 5), [1, 0]))

    assert graph(attention).proven
    for build, what in ((rows_turned, "row by row"), (queries_turned, "split into heads"),
                        (lambda b, x, w, lut: attention(b, x, w, lut, causal=False), "causal"),
                        (lambda b, x, w, lut: b.qlinear("y", x, w, 1, 5), "attention chain"),
                        (lambda b, x, w, lut: b.qmatmul("y", x, b.transpose("t", x, [1, 0]), 1, 9), "computed right operand")):
        with pytest.raises(ValueError, match=what):
            graph(build).decoder(rows=1)


def test_beams_are_traced_back():
    rng = np.random.default_rng(0)
    steps, P, beams = 7, 3, 4
    parent = np.where(np.arange(steps)[:, None, None] > 0, rng.integers(0, beams, (steps, P, beams)) + beams * np.arange(P)[:, None],
                      np.arange(P)[:, None] + np.zeros((1, 1, beams), int)).astype(np.int32)
    token = rng.integers(0, 50, (steps, P, beams)).astype(np.int32)
    got = decode._trace(parent, token)
    for p, b in np.ndindex(P, beams):
        at, want = b, []
        for n in range(steps - 1, -1, -1):
            want.append(token[n, p, at])
            at = parent[n, p, at] - beams * p
        assert got[p, b].tolist() == want[::-1]
    assert decode._cut([4, 5, 6], 5) == [4, 5] and decode._cut([4, 5], None) == [4, 5] and decode._cut([4], 9) == [4]


def test_selection_tables_are_fixed_point_logs():
    s = decode.Selection.of(0.05)
    assert s.mult == round(0.05 * 65536) and s.step == 45426 and s.lut[255] == 1 << 20
    v = np.arange(1, decode.Selection.LOGS)
    assert np.abs(s.logs[1:] / 65536 - np.log(v)).max() <= 0.5 / 65536 + 1e-12
    assert abs(s.lut[254] / (1 << 20) - np.exp(-0.05)) <= 0.5 / (1 << 20)
    assert decode.Selection.of(1e-9).mult == 1
