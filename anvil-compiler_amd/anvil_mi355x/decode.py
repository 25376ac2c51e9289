"""Token by token: a compiled token model over a paged cache of 4-bit keys and values.

    dec = cm.decoder(rows=16, max_tokens=1024)                 # CompiledModel.decoder of a model with embedding tables
    out = dec.generate(prompts, 32, beams=4)                   # lists of token ids, best beam first, with their scores

The reference evaluates a whole sequence for every token (anvil/interp/graph.py:43-92). Here each op of the graph runs on the rows of
new tokens only: row-wise ops as they are, an attention chain as an append of the new keys and values, rounded to 4 bits, to the
cache and anvil_attention_cache_i4 over it. Results are those of the graph whose k and v hold the rounded values.

KVCache is the cache by itself: pages of every layer, and two sets of tables, of which a step reads one and writes the other.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import numpy as np

from . import ir as g
from . import runtime as rt

NO_SCORE = -(1 << 63)


class KVCache:
    """A pool of pages for `layers` layers of (heads, dim) keys and values, and the tables of up to `rows` sequences of up to
    `max_tokens` tokens. It starts with `rows` empty sequences. A step() takes the tables on (anvil_cache_fork): reserve, fork, free;
    undo() goes back to those before the last one. Device buffers are this object's; the calls run on the device's stream, in order."""

    def __init__(self, dev, layers, heads, dim, pages, rows, max_tokens, window=0, sinks=0):
        if rows < 1 or max_tokens < 1:
            raise ValueError(f"a cache of {rows} rows of {max_tokens} tokens")
        self.dev, self.window, self.sinks = dev, window, sinks
        slots = -(-max_tokens // rt.CACHE_PAGE)
        self.pool = dev.alloc(dev.cache_bytes(layers, pages, heads, dim))
        self._sets = []
        for _ in range(2):
            table = dev.upload(np.full((rows, slots), -1, np.int32))
            lens, refs = dev.upload(np.zeros(rows, np.int32)), dev.upload(np.zeros(pages, np.int32))
            self._sets.append((table, lens, refs))
        self._shape = dict(slots=slots, pages=pages, heads=heads, dim=dim, layers=layers)
        self._rows, self._n, self._at = rows, [rows, rows], 0
        self.moved = dev.alloc(4 * pages)                      # compact()'s map
        self._back = False                                     # the tables before the last step still hold; None: if it failed

    def _cache(self, which, seqs=None):
        return rt.Cache(self.pool, *self._sets[which], seqs=self._n[which] if seqs is None else seqs, **self._shape)

    @property
    def cache(self) -> rt.Cache:
        """The tables as they are."""
        return self._cache(self._at)

    @property
    def seqs(self) -> int:
        return self._n[self._at]

    def step(self, parent=None, add=None, rows=None):
        """The tables of the next step: row i continues row parent[i] (device int32s; None: row i) by add[i] tokens (device int32s;
        None: none). rows: how many there are, with parents. Too few free pages are reported by the device's sync() as MemoryError, and
        leave every row empty: undo() then goes back to the rows as they were, if no other step has been taken since."""
        n = self.seqs if rows is None else rows
        if not 0 <= n <= self._rows:
            raise ValueError(f"{n} rows in a cache of {self._rows}")
        self.dev.cache_fork(self.cache, self._cache(1 - self._at, n), parent, add, self.window, self.sinks)
        self.stepped(n)
        if add is None or parent is None and not self.window:
            self._back = True

    def stepped(self, rows):
        """A step that recorded kernels have taken."""
        self._at = 1 - self._at
        self._n[self._at], self._back = rows, None

    def compact(self):
        """Used pages to the pool's lowest ids; self.moved then holds each page's new id (-1: free)."""
        n = self.seqs
        self.dev.cache_compact(self.cache, self._cache(1 - self._at, n), self.moved)
        self.stepped(n)
        self._back = True

    def undo(self):
        """The tables before the last compact() or step(), as long as nothing has been appended since. A step that both gives pages
        back (parents or a window) and adds tokens may have written some of them, and cannot be taken back unless it failed: its rows
        are then empty and its references those of before, and it has written nothing (this waits for the device to see that)."""
        if self._back is None:
            (_, lens, refs), (_, _, before) = self.tables(), self._tables(1 - self._at)
            self._back = not lens.any() and np.array_equal(refs, before)
        if not self._back:
            raise ValueError("the last step cannot be taken back")
        self._at, self._back = 1 - self._at, False

    def reset(self, rows=None):
        """`rows` empty sequences (None: as many as the cache has room for)."""
        if rows is not None and not 0 <= rows <= self._rows:
            raise ValueError(f"{rows} rows in a cache of {self._rows}")
        for table, lens, refs in self._sets:
            table.upload(np.full(table.nbytes // 4, -1, np.int32))
            lens.upload(np.zeros(lens.nbytes // 4, np.int32))
            refs.upload(np.zeros(refs.nbytes // 4, np.int32))
        self._at, self._n, self._back = 0, [self._rows if rows is None else rows] * 2, False

    def tables(self):
        """(table, lens, refs) on the host."""
        return self._tables(self._at)

    def _tables(self, which):
        table, lens, refs = self._sets[which]
        n, slots = self._n[which], self._shape["slots"]
        return (table.download((n, slots), np.int32), lens.download((n,), np.int32),
                refs.download((self._shape["pages"],), np.int32))


@dataclass
class Generated:
    """tokens[p][b]: the new tokens of prompt p's b-th best beam (up to and with eos); scores[p][b]: its log probability."""
    tokens: list
    scores: np.ndarray


class _Rows:
    """A graph value as dense rows of a device buffer: one a token, an attention result's with the heads side by side."""

    def __init__(self, width, dtype):
        self.width, self.dtype, self.buf = width, dtype, None


class Decoder:
    """CompiledModel.decoder: the model over a KVCache of `rows` sequences."""

    def __init__(self, cm, rows, max_tokens=None, pages=None, window=0, sinks=0):
        if not cm.proven:
            raise ValueError("decoding needs a graph with a sound int32 proof")
        if cm.embedding is None:
            raise ValueError("decoding needs embedding tables: compile(..., embedding=(wte, wpe))")
        if len(cm.output_values) != 1:
            raise ValueError("decoding needs a graph with one output")
        self.cm = cm
        self.T = g.qt(cm.input_ops[0].result).dims[0]
        positions = cm.embedding[1].shape[0]
        max_tokens = positions if max_tokens is None else int(max_tokens)
        if not 1 <= max_tokens <= positions:
            raise ValueError(f"max_tokens {max_tokens}: the position table has {positions} rows")
        self.rows, self.max_tokens = int(rows), max_tokens
        if not 1 <= self.rows <= rt.CACHE_ROWS_MAX:
            raise ValueError(f"rows {rows} outside [1, {rt.CACHE_ROWS_MAX}]")
        if window < 0 or sinks < 0:
            raise ValueError(f"window {window}, sinks {sinks}")
        self.steps, layers, heads, dim = self._lower()
        self.vocab = cm.embedding[0].shape[0]
        cm._ensure_device()
        self.dev = cm.dev
        slots = -(-max_tokens // rt.CACHE_PAGE)
        pages = self.rows * (slots + 1) if pages is None else int(pages)
        self.cache = KVCache(self.dev, layers, heads, dim, pages, self.rows, max_tokens, window, sinks)
        self.wte, self.wpe = (self.dev.upload(t) for t in cm.embedding)
        for kind, op, *rest in self.steps:
            if kind == "experts":
                rest[-1]["starts"] = self.dev.alloc(4 * (g.qt(op.scores).dims[-1] + 1))
        self._room, self._buffers = 0, []

    # ----------------------------------------------------------------------------------------------- lowering
    def _lower(self):
        """The graph's ops as calls on rows: ([(kind, op, ...)], layers, heads, dim). What a row holds is told by the indexes that a
        chain of transposes and reshapes moves its elements by."""
        cm, T, steps, value = self.cm, self.T, [], {}
        chains = cm._attention_chains("outputs", rt.CACHE_TOKENS_MAX)
        inside = {o for c in chains.values() for o in c}
        # adds in the epilogue of the product before them, whose own result nothing else reads
        adds = {op: add for op, add in cm._residual_fusions("outputs").items()
                if len(cm.users[op.result]) == 1 and g.qt(op.a).dims[-1] % 16 == 0}
        expert_adds, scratch = cm._expert_adds("outputs"), []
        layers, shape = 0, None

        def new(v, width=None):
            t = g.qt(v)
            if width is None and (len(t.dims) != 2 or t.dims[0] != T):
                raise ValueError(f"decoding: a value of shape {t.dims} has no row for each of {T} tokens")
            value[v] = _Rows(t.dims[1] if width is None else width, t.dtype)
            return value[v]

        def view(v):
            """(the value v is a view of, v's elements as indexes into it)."""
            op, dims = v.owner, g.qt(v).dims
            if not isinstance(op, (g.TransposeOp, g.ReshapeOp)):
                return v, np.arange(math.prod(dims)).reshape(dims)
            root, idx = view(op.x)
            return root, idx.transpose(op.perm_list) if isinstance(op, g.TransposeOp) else idx.reshape(dims)

        def rows_of(v):
            """The rows of an op's operand: a value's own, or those that merge an attention result's heads."""
            root, idx = view(v)
            if root not in value:
                raise ValueError(f"decoding: {v.owner.name} {v.owner.sym_str!r} has no rows")
            want = np.arange(idx.size).reshape(T, -1)
            if root.owner in chains:
                want = want.reshape(shape[0], T, shape[1]).transpose(1, 0, 2).reshape(T, -1)
            if not np.array_equal(idx, want):
                raise ValueError(f"decoding: {root.owner.sym_str!r} is read other than row by row")
            return value[root]

        def table(v):
            """A const operand, as it is."""
            if not isinstance(v.owner, g.ConstOp):
                raise ValueError(f"decoding: the table {v.owner.sym_str!r} is no const")
            return v

        for op in cm.ops:
            if op in inside or isinstance(op, (g.TransposeOp, g.ReshapeOp)) or op.result in cm.is_const:
                continue
            if isinstance(op, g.InputOp):
                steps.append(("embed", op, new(op.result)))
            elif op in chains:
                s_op, sm = chains[op]
                *lead, n, d = g.qt(op.result).dims
                heads = math.prod(lead)
                if n != T or not sm.causal or shape not in (None, (heads, d)):
                    raise ValueError("decoding needs causal attention over the graph's tokens, with every layer's heads alike")
                shape = (heads, d)
                # what the attention over the cache takes, whose scores' products are bounded by the values that 4 bits hold
                if 128 * 126 * d * abs(int(s_op.M)) + (1 << int(s_op.s) >> 1) > 2 ** 31 - 1:
                    raise OverflowError(f"decoding: {s_op.sym_str!r}'s multiplier {int(s_op.M)} may take scores past int32")
                split = np.arange(T * heads * d).reshape(T, heads, d).transpose(1, 0, 2)
                qkv = []
                for v, want in ((s_op.a, split), (s_op.b, split.transpose(0, 2, 1)), (op.b, split)):
                    root, idx = view(v)
                    if root not in value or root.owner in chains or not np.array_equal(idx, want.reshape(idx.shape)):
                        raise ValueError(f"decoding: an operand of {op.sym_str!r}'s attention is not rows split into heads")
                    qkv.append(value[root])
                steps.append(("attend", op, s_op, sm, layers, qkv, new(op.result, heads * d)))
                layers += 1
            elif isinstance(op, (g.QLinearOp, g.QMatmulOp)):
                if len(g.qt(op.b).dims) != 2 or op.b not in cm.is_const:
                    raise ValueError(f"decoding: {op.name} {op.sym_str!r} has a computed right operand outside an attention chain")
                a, lut, add = rows_of(op.a), None if op.lut is None else table(op.lut), adds.get(op)
                if add is not None:
                    inside.add(add)
                    other = add.b if add.a is op.result else add.a
                    steps.append(("linear_add", op, a, new(add.result), lut, add, rows_of(other)))
                    continue
                call = (op, a, new(op.result), lut)
                if steps[-1][0] == "linears" and steps[-1][1][0][1] is a and len(steps[-1][1]) < rt.GEMM_GROUP_MAX:
                    steps[-1][1].append(call)              # of one input: one launch
                else:
                    steps.append(("linears", [call]))
            elif isinstance(op, g.RmsNormIntOp):
                steps.append(("norm", op, rows_of(op.x), new(op.result), table(op.w), table(op.lut)))
            elif isinstance(op, g.AddRequantOp):
                steps.append(("add", op, rows_of(op.a), rows_of(op.b), new(op.result)))
            elif isinstance(op, g.LutOp):
                steps.append(("lut", op, rows_of(op.x), new(op.result), table(op.table)))
            elif isinstance(op, g.ExpertsOp):
                add = expert_adds.get(op)
                other = None if add is None else rows_of(add.b if add.a is op.result else add.a)
                x, scores = rows_of(op.x), rows_of(op.scores)
                if add is not None:
                    inside.add(add)
                buf = {n: _Rows(*what) for n, what in cm._expert_scratch(op).items()}
                scratch.extend(buf.values())
                steps.append(("experts", op, x, scores, new(op.result if add is None else add.result), add, other, buf))
            elif isinstance(op, g.LutMulOp):
                steps.append(("lut_mul", op, rows_of(op.x), rows_of(op.y), new(op.result), table(op.table)))
            else:
                raise ValueError(f"decoding: {op.name} {op.sym_str!r} is not row-wise")
        if not layers:
            raise ValueError("decoding needs an attention chain")
        self.logits = rows_of(cm.output_values[0])
        self.scale = g.qt(cm.output_values[0]).qscale
        self._values = list(value.values()) + scratch
        return steps, layers, *shape

    def _make_room(self, rows):
        """Buffers of every value for so many rows of tokens. They start as zeros, and only results of the graph's ops follow, so
        that the rows of empty sequences, which the row-wise ops evaluate with the others, stay in the ranges of the graph's proof.
        Smaller ones that came before stay, for launches recorded with them."""
        if rows <= self._room:
            return
        room = max(rows, 2 * self._room)
        bufs = [self.dev.alloc(room * r.width * rt.ITEMSIZE[r.dtype]) for r in self._values]
        for r, buf in zip(self._values, bufs):
            self.dev.zero(buf, buf.nbytes)
            if r.buf is not None:
                self._buffers.append(r.buf)
            r.buf = buf
        self._room = room                                      # once all of them are there

    # ------------------------------------------------------------------------------------------------ forward
    def forward(self, ids, starts, rows, max_new):
        """The graph's output (rows, width), on the device until the next call, for new tokens: `ids` (device int32s), rows
        starts[s] .. starts[s + 1] - 1 those of sequence s, at most max_new each (device int32s; None: one a sequence). The cache has
        been stepped by them. Launches only, once a call of as many rows has run."""
        dev, cm, cache = self.dev, self.cm, self.cache.cache
        heads, d = cache.heads, cache.dim
        self._make_room(rows)
        const = cm._const_views
        for kind, op, *rest in self.steps:
            if kind == "embed":
                (x,) = rest
                dev.embed_quantize_new(cache, ids, starts, rows, max_new, x.width, self.wte, self.vocab, self.wpe,
                                       self.max_tokens, cm.scale(op.sym_str), x.buf, x.dtype)
            elif kind == "attend":
                s_op, sm, layer, (q, k, v), o = rest
                dev.cache_append(cache, layer, k.buf, v.buf, starts, rows, max_new, (k.width, d, v.width, d))
                dev.attention_cache(cache, layer, q.buf, o.buf, starts, rows, max_new, heads, (q.width, d, o.width, d),
                                    int(s_op.M), int(s_op.s), const[sm.lut].ptr, int(sm.one), int(op.M), int(op.s),
                                    self.cache.window, self.cache.sinks)
            elif kind == "linears":
                calls = [self._product(*call, rows, call[2].buf) for call in op]
                if len(calls) == 1:
                    dev.gemm_i8(*calls[0])
                else:
                    dev.gemm_i8_group(calls)
            elif kind == "linear_add":
                a, y, lut, add, r = rest
                *product, dtype, flags = self._product(op, a, y, lut, rows, None)
                ma, mb = (add.Mb, add.Ma) if add.a is op.result else (add.Ma, add.Mb)              # residual, product
                dev.gemm_i8_add(*product, r.buf, int(ma), int(mb), int(add.s), y.buf, [0, 0, y.width, 0, 0, y.width], flags, dtype)
            elif kind == "norm":
                x, y, w, lut = rest
                dev.rmsnorm_int(x.buf, x.dtype, const[w].ptr, const[lut].ptr, const[lut].size, int(op.M), int(op.s), op.ss_shift_int,
                                op.ss_init_int, rows, x.width, y.buf, rt.OP_UNCHECKED)
            elif kind == "add":
                a, b, y = rest
                dev.add_requant(a.buf, a.dtype, b.buf, b.dtype, int(op.Ma), int(op.Mb), int(op.s), rows * y.width, y.buf, y.dtype,
                                rt.OP_UNCHECKED)
            elif kind == "experts":
                x, scores, y, add, other, buf = rest
                at = {n: b.buf if isinstance(b, _Rows) else b for n, b in buf.items()}
                for _, call, args in cm._expert_calls(op, x.buf, scores.buf, rows, {**at, "out": y.buf}, add, other and other.buf):
                    call(*[a.ptr if hasattr(a, "ptr") else a for a in args])
            elif kind == "lut":
                x, y, lut = rest
                dev.lut_i8(x.buf, const[lut].ptr, rows * y.width, y.buf)
            else:
                x, z, y, lut = rest
                dev.lut_mul(x.buf, z.buf, const[lut].ptr, int(op.M), int(op.s), rows * y.width, y.buf, rt.OP_UNCHECKED)
        return self.logits.buf

    def _product(self, op, a, y, lut, rows, out):
        """The arguments of gemm_i8 for rows of a into `out`."""
        cm, flags = self.cm, rt.GEMM_UNCHECKED
        if cm.acc_bounds.get(op.result, 1 << 31) < 1 << 23 and abs(int(op.M)) < 1 << 23:
            flags |= rt.GEMM_MUL24
        return (a.buf, cm._bt_const(op).ptr, out, 1, 1, rows, y.width, a.width, [0, 0, a.width, 0, 0, a.width, 0, 0, y.width],
                int(op.M), int(op.s), None if lut is None else cm._const_views[lut].ptr, y.dtype, flags)

    # ----------------------------------------------------------------------------------------------- generate
    def generate(self, prompts, new_tokens, beams=1, eos=None, allowed=None) -> Generated:
        """`new_tokens` tokens after each prompt (lists of ids, of any lengths), the best of `beams` beams by their fixed-point log
        probabilities (beams=1: the most likely token each time, the lowest id of equals). eos: a beam that ends with it is done.
        allowed: vocab truth values, tokens to choose from."""
        V = self.logits.width
        prompts = [np.asarray(p) for p in prompts]
        P, rows = len(prompts), len(prompts) * beams
        if not P or rows > self.rows or not 1 <= beams <= 64:
            raise ValueError(f"{P} prompts of {beams} beams: the decoder has {self.rows} rows")
        if new_tokens < 1:
            raise ValueError(f"new_tokens {new_tokens}")
        for p in prompts:
            if p.ndim != 1 or not p.size or p.dtype.kind not in "iu":
                raise ValueError("a prompt is a list of token ids, at least one")
            if p.size + new_tokens - 1 > self.max_tokens:
                raise ValueError(f"{p.size} + {new_tokens} tokens: the decoder holds {self.max_tokens}")
            if p.min() < 0 or p.max() >= self.vocab:
                raise ValueError(f"token ids outside [0, {self.vocab})")
        if eos is not None and not 0 <= eos < V:
            raise ValueError(f"eos {eos} outside [0, {V})")
        if self.logits.dtype != "i8" or self.scale is None or V > self.vocab:
            raise ValueError(f"the graph's output is not int8 logits with a scale for {self.vocab} tokens")
        try:
            return self._generate(prompts, new_tokens, beams, eos, allowed)
        except BaseException:
            self.cm._settle()                                  # nothing runs on the call's buffers, and no violation stays behind
            raise

    def _generate(self, prompts, new_tokens, beams, eos, allowed) -> Generated:
        dev, cache, V, P = self.dev, self.cache, self.logits.width, len(prompts)
        rows = P * beams
        select = Selection.of(self.scale)
        tables = self._tables(select, allowed, V)
        starts = np.cumsum([0] + [p.size for p in prompts]).astype(np.int32)
        total = int(starts[-1])
        self._make_room(max(total, rows))
        ids, d_starts = dev.upload(np.concatenate(prompts).astype(np.int32)), dev.upload(starts)
        lens, ones = dev.upload(np.diff(starts)), dev.upload(np.ones(rows, np.int32))
        last, states = dev.alloc(P * V), [self._state(rows) for _ in range(2)]
        states[0]["scores"].upload(np.zeros(P, np.int64))
        states[0]["ended"].upload(np.zeros(P, np.uint8))
        history = {name: dev.alloc(4 * rows * new_tokens) for name in ("parent", "token")}

        def choose(src, dst, logits, beams_in):
            dev.beam_select(logits, V, src["scores"], None if eos is None else src["ended"], tables["allowed"], P, beams_in, V, beams,
                            -1 if eos is None else eos, tables["lut"], tables["logs"], select.logs.size, select.step, select.mult,
                            dst["scores"], dst["parent"], dst["token"], dst["ended"])

        def step(src, dst):
            cache.step(src["parent"], ones, rows)
            choose(src, dst, self.forward(src["token"], None, rows, 1), beams)

        cache.reset(P)
        cache.step(None, lens)
        logits = self.forward(ids, d_starts, total, int(np.diff(starts).max()))
        for i in range(P):                                     # each prompt's last token
            dev.copy_strided(logits.ptr + (int(starts[i + 1]) - 1) * V, last.ptr + i * V, 1, [V], [1])
        choose(states[0], states[1], last, 1)
        # The tables and states alternate, so two recordings serve every step; the first step continues P rows by `rows`.
        recorded = {}
        for n in range(new_tokens):
            src, dst = states[n % 2], states[1 - n % 2]
            if n in (1, 2):
                step(src, dst)
            elif n in (3, 4):
                recorded[n % 2] = dev.sequence(step, src, dst)
            elif n > 4:
                recorded[n % 2].launch()
                cache.stepped(rows)
            for name, buf in history.items():
                dev.copy_strided(dst[name].ptr, buf.ptr + 4 * rows * n, 4, [rows], [1])
        dev.sync()
        scores = states[new_tokens % 2]["scores"].download((P, beams), np.int64)
        parent, token = (history[name].download((new_tokens, P, beams), np.int32) for name in ("parent", "token"))
        alive = scores != NO_SCORE
        rows_of = _trace(parent, token)
        tokens = [[_cut(rows_of[p, b].tolist(), eos) for b in range(beams) if alive[p, b]] for p in range(P)]
        return Generated(tokens, np.where(alive, scores / (1 << Selection.BITS), -np.inf))

    def _state(self, rows):
        dev = self.dev
        return {"scores": dev.alloc(8 * rows), "parent": dev.alloc(4 * rows), "token": dev.alloc(4 * rows), "ended": dev.alloc(rows)}

    def _tables(self, select, allowed, V):
        dev = self.dev
        if allowed is not None:
            allowed = np.asarray(allowed)
            if allowed.shape != (V,):
                raise ValueError(f"allowed: {allowed.shape} truth values for a vocabulary of {V}")
            allowed = dev.upload((allowed != 0).astype(np.uint8))
        return {"lut": dev.upload(select.lut.astype(np.int32)), "logs": dev.upload(select.logs.astype(np.int32)), "allowed": allowed}


def _trace(parent, token):
    """Every beam's tokens (prompts, beams, steps), from the last selection back to the first, whose parents are the prompts. A
    selection's parents are rows of the one before."""
    steps, P, beams = token.shape
    out = np.empty((P, beams, steps), token.dtype)
    row = np.arange(P * beams)
    for n in range(steps - 1, -1, -1):
        out[:, :, n] = token[n].reshape(-1)[row].reshape(P, beams)
        row = np.maximum(parent[n].reshape(-1)[row], 0)        # -1: of a beam that is none
    return out


def _cut(tokens, eos):
    return tokens[:tokens.index(eos) + 1] if eos is not None and eos in tokens else tokens


@dataclass
class Selection:
    """The tables of anvil_beam_select_i8 for int8 logits of a scale: log probabilities with BITS fractional bits."""
    lut: np.ndarray
    logs: np.ndarray
    step: int
    mult: int
    BITS = 16
    LOGS = 2048                 # a sum's log is that of its top 11 bits or more: within 2^-10

    @classmethod
    def of(cls, scale) -> "Selection":
        one = 1 << cls.BITS
        lut = np.rint(np.exp(np.arange(-255, 1) * scale) * (1 << 20))
        logs = np.rint(np.log(np.maximum(1, np.arange(cls.LOGS))) * one)
        return cls(lut, logs, round(math.log(2) * one), max(1, round(scale * one)))
