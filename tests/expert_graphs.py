"""Graphs with experts, and a CPU stand-in for the calls that they make. Test infrastructure only."""
import numpy as np

from anvil_mi355x import ir as g
from anvil_mi355x import models
from anvil_mi355x import quantize as Q
from fake_device import NP, FakeDevice
from oracle import experts as oe


def requant(spread, acc_rms, bound):
    """(M, s) that bring accumulators of that root mean square to `spread` and keep `bound` within int32."""
    (m,), s = Q.choose_shift([spread / acc_rms], [bound])
    return m, s


class Feed:
    """An experts op's consts and constants for rows of C columns: random weights, seeded."""

    def __init__(self, prefix, C, width, columns, experts, top, gated, seed=0, one=127, rows_rms=40):
        rng = np.random.default_rng(seed)
        self.prefix, self.gated, self.top, self.one = prefix, gated, top, one
        w = lambda *shape: np.clip(np.rint(rng.normal(0, 40, shape)), -127, 127).astype(np.int64)      # noqa: E731
        x = np.arange(-128, 128) / 16
        self.consts = {"router": w(C, experts), "up": w(experts, C, width), "down": w(experts, width, columns),
                       "exp": Q.exp_table(0.06, max(top, 2), one), "act": np.clip(np.rint(x / (1 + np.exp(-x)) * 16), -128, 127).astype(np.int64)}
        if gated:
            self.consts["gate"] = w(experts, C, width)
        bound = lambda name, mag: mag * int(np.abs(self.consts[name]).sum(axis=-2).max())              # noqa: E731
        up = requant(45, rows_rms * 40 * np.sqrt(C), bound("up", 128))
        self.router = requant(30, rows_rms * 40 * np.sqrt(C), bound("router", 128))
        down = requant(45, 18 * 40 * np.sqrt(width), bound("down", 128))
        (mc,), sc = Q.choose_shift([1.2 / one], [128 * (one + top)])
        self.args = dict(m=up[0], s=up[1], md=down[0], sd=down[1], mc=mc, sc=sc)
        if gated:
            gate = requant(45, rows_rms * 40 * np.sqrt(C), bound("gate", 128))
            (mm,), sm = Q.choose_shift([1 / 45], [1 << 14])
            self.args.update(mg=gate[0], sg=gate[1], mm=mm, sm=sm)

    def values(self):
        return {f"{self.prefix}.{k}": v for k, v in self.consts.items()}

    def add(self, b, sym, x, scores=None, scale=None):
        """The op in builder b, behind a router over x unless scores are given."""
        c = {k: b.const(f"{self.prefix}.{k}", list(v.shape), "i32" if k == "exp" else "i8") for k, v in self.consts.items()
             if k != "router" or scores is None}
        if scores is None:
            scores = b.qlinear(f"{self.prefix}.scores", x, c["router"], *self.router)
        return b.experts(sym, x, scores, c["up"], c["down"], c["exp"], c["act"], self.top, self.one, gate=c.get("gate"), scale=scale, **self.args)


def layer(T, C, width, experts, top, gated, residual="i8", seed=0, lead=()):
    """(module, consts): x -> experts over x, then x + the result (residual None: the result alone)."""
    b, feed = g.GraphBuilder("experts"), Feed("f", C, width, C, experts, top, gated, seed)
    x = b.input("x", [*lead, T, C], "i8", 0.05)
    wide = b.input("wide", [*lead, T, C], "i16", 0.01) if residual == "i16 before" else None
    y = feed.add(b, "y", x)
    if residual is None:
        b.output(y)
    else:
        if residual.startswith("i16"):
            wide = wide or b.input("wide", [*lead, T, C], "i16", 0.01)
            b.output(b.add_requant("r", wide, y, 256, 900, 8, 0.01, dtype="i16"))
        elif residual == "swapped":
            b.output(b.add_requant("r", y, x, 70, 60, 6, 0.05))
        else:
            b.output(b.add_requant("r", x, y, 60, 70, 6, 0.05))
    return b.module(), feed.values()


def with_experts(built, experts, top, gated, seed=0):
    """A built model whose MLPs (fc, GELU, proj) are experts behind a router, everything else as it is."""
    b, consts, value = g.GraphBuilder("model"), dict(built.consts), {}
    for op in g.func_of(built.module).ops:
        sym = op.sym_str or ""
        part = sym.split(".")[-1]
        if isinstance(op, g.OutputOp):
            b.output(*[value[v] for v in op.values])
        elif sym.split(".", 1)[-1].startswith(("fc", "gelu", "proj.w")):
            consts.pop(sym, None)
        elif part == "proj":
            feed = Feed(sym, built.spec.n_embd, 2 * built.spec.n_embd, built.spec.n_embd, experts, top, gated, seed + len(value))
            h2 = next(v for k, v in value.items() if k.owner.sym_str == sym.replace("proj", "h2"))
            value[op.result] = feed.add(b, sym, h2, scale=g.qt(op.result).qscale)
            consts.update(feed.values())
        else:
            new = type(op)({n: value[v] for n, v in op.operand_items()}, op.props, op.result.type, op.sym)
            value[op.result] = b._add(new)
    return models.Built(built.spec, b.module(), consts, built.scales, built.params)


class ExpertDevice(FakeDevice):
    """The experts' calls over the fake heap, by the numpy restatement."""

    def _ints(self, ptr, dtype, n):
        return self.view(ptr, dtype, (n,), (1,))

    def _rows(self, ptr, dtype, rows, cols, ld):
        return self.view(ptr, dtype, (rows, cols), (ld, 1))

    def expert_route(self, scores, ld, live, rows, experts, top, lut, one, expert, weight, slot, row, starts, every=False):
        self.calls.append("expert_route")
        live = None if live is None else self._ints(live, "i8", rows)
        out = oe.route(self._rows(scores, "i8", rows, experts, ld), live, top, self._ints(lut, "i32", 256), one, every)
        for ptr, dtype, v in zip((expert, weight, slot, row, starts), ("i32", "i16", "i32", "i32", "i32"), out):
            self.store(ptr, dtype, (v.size,), (1,), v.reshape(-1))

    def expert_gemm(self, A, lda, rows_a, row, scale, B, B2, ldb, sb, starts, experts, rows, N, K, Cp, ldc, out_dtype, mults=None, mult=0, shift=0,
                    mults2=None, mult2=0, shift2=0, lut=None, mult3=1, shift3=0):
        self.calls.append("expert_gemm")
        assert lda >= K and ldb >= K and ldc >= N and (experts == 1 or sb >= N * ldb)
        w = lambda p: None if p is None else self.view(p, "i8", (experts, N, K), (sb, ldb, 1))         # noqa: E731
        ints = lambda p, dtype, n: None if p is None else self._ints(p, dtype, n)                      # noqa: E731
        each = lambda p, m: np.full(experts, m) if p is None else self._ints(p, "i32", experts)        # noqa: E731
        out = self._rows(Cp, out_dtype, rows, N, ldc)
        out[...] = oe.gemm(out, self._rows(A, "i8", rows_a, K, lda), ints(row, "i32", rows), ints(scale, "i16", rows_a), w(B), w(B2),
                           self._ints(starts, "i32", experts + 1), each(mults, mult), shift, each(mults2, mult2), shift2, ints(lut, "i8", 256),
                           mult3, shift3, out_dtype).astype(NP[out_dtype])

    def expert_combine(self, Y, ldy, positions, slot, weight, rows, top, cols, mult, shift, R, r_dtype, ldr, ma, mb, shift2, D, d_dtype, ldd):
        self.calls.append("expert_combine")
        res = None if R is None else self._rows(R, r_dtype, rows, cols, ldr)
        v = oe.combine(self._rows(Y, "i8", positions, cols, ldy), self._ints(slot, "i32", rows * top).reshape(rows, top),
                       self._ints(weight, "i16", rows * top).reshape(rows, top), mult, shift, res, ma, mb, shift2, d_dtype)
        self.store(D, d_dtype, (rows, cols), (ldd, 1), v)
