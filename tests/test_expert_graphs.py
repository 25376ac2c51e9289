"""The graph's experts op: its typing rules, its printed form, its int32 proof, compiled models against the oracle's interpreter, and token
models whose feed-forward parts are experts, decoded over the cache. Everything is exact."""
import numpy as np
import pytest

import anvil_mi355x
import expert_graphs as eg
from anvil_mi355x import ir as g
from anvil_mi355x import models
from anvil_mi355x import quantize as Q
from anvil_mi355x import runtime as rt
from oracle import experts as oe
from oracle import interp
from oracle import semantics as sem
from test_decoder import Oracle, prompts_of, same

gpu = pytest.mark.gpu


# --------------------------------------------------------------------------------------------- the op (CPU)

def _op(**change):
    """An experts op of 6 rows of 16 columns, 3 experts of width 8."""
    b = g.GraphBuilder("t")
    shapes = {"x": [6, 16], "scores": [6, 3], "up": [3, 16, 8], "down": [3, 8, 20], "exp": [256], "act": [256], "gate": None}
    args = dict(top=2, one=127, m=3, s=10, md=3, sd=10, mc=5, sc=9)
    for k, v in change.items():
        (shapes if k in shapes else args)[k] = v
    v = {k: None if s is None else (b.input if k in ("x", "scores") else b.const)(k, s, "i32" if k == "exp" else "i8") for k, s in shapes.items()}
    return b, b.experts("y", v["x"], v["scores"], v["up"], v["down"], v["exp"], v["act"], gate=v["gate"], **args)


GATE = dict(gate=[3, 16, 8], mg=3, sg=10, mm=4, sm=8)


def test_types():
    assert g.qt(_op()[1]).dims == [6, 20] and g.qt(_op(**GATE)[1]).dims == [6, 20]
    assert g.qt(_op(x=[2, 6, 16], scores=[2, 6, 3])[1]).dims == [2, 6, 20]


@pytest.mark.parametrize("change", [dict(scores=[5, 3]), dict(scores=[6, 4]), dict(up=[3, 15, 8]), dict(up=[16, 8]), dict(down=[3, 9, 20]),
                                    dict(down=[2, 8, 20]), dict(exp=[255]), dict(act=[128]), dict(top=0), dict(top=4), dict(one=0),
                                    dict(one=32768), dict(s=32), dict(sd=-1), dict(sc=40), dict(gate=[3, 16, 8]), dict(mg=1),
                                    {**GATE, "gate": [3, 16, 9]}, {**GATE, "sm": 32}, {**GATE, "mm": None}], ids=str)
def test_what_does_not_fit_is_refused(change):
    with pytest.raises(g.VerifyException):
        _op(**change)


@pytest.mark.parametrize("gated", [False, True])
def test_round_trip_of_the_printed_form(gated):
    m, _ = eg.layer(6, 16, 8, 3, 2, gated)
    text = anvil_mi355x.print_ir(m)
    assert text.count('"anvil.graph.experts"') == 1 and ("Mg = " in text) == gated
    assert anvil_mi355x.print_ir(anvil_mi355x.parse_ir(text)) == text


@pytest.mark.parametrize("gated", [False, True])
def test_the_op_is_its_formula_row_by_row(gated):
    m, consts = eg.layer(5, 12, 7, 4, 3, gated, residual=None)
    op = next(o for o in g.func_of(m).ops if isinstance(o, g.ExpertsOp))
    x = np.random.default_rng(0).integers(-128, 128, (5, 12))
    values = interp.run(m, {"x": x}, consts).values
    c = {k: consts[f"f.{k}"] for k in ("up", "down", "exp", "act", *(["gate"] if gated else []))}
    for i in range(5):
        s = values["f.scores"][i]
        order = sorted(range(4), key=lambda e: (-s[e], e))[:3]
        w = sem.softmax_lut(s[order][None], c["exp"], int(op.one), False)[0]
        acc = 0
        for wj, e in zip(w, order):
            h = sem.requant(x[i] @ c["up"][e], int(op.M), int(op.s))
            if gated:
                t = sem.lut_i8(sem.requant(x[i] @ c["gate"][e], int(op.Mg), int(op.sg)), c["act"])
                h = sem.requant(t * h, int(op.Mm), int(op.sm))
            else:
                h = sem.lut_i8(h, c["act"])
            acc = acc + wj * sem.requant(h @ c["down"][e], int(op.Md), int(op.sd))
        assert np.array_equal(values["y"][i], sem.requant(acc, int(op.Mc), int(op.sc)))
    assert np.abs(values["y"]).max() > 10


def test_the_int32_proof():
    m, consts = eg.layer(6, 16, 8, 3, 2, True)
    bounds = Q.int32_bounds(m, consts)
    assert bounds.ok and bounds.worst["y"] > 1 << 24
    op = next(o for o in g.func_of(m).ops if isinstance(o, g.ExpertsOp))
    for name in ("M", "Md", "Mc", "Mg", "Mm", "one"):
        keep = op.props[name]
        op.props[name] = 1 << 26
        with pytest.raises(OverflowError, match="y:"):
            anvil_mi355x.compile((m, consts))
        op.props[name] = keep
    for bad in (np.r_[-1, consts["f.exp"][1:]], np.r_[consts["f.exp"][:-1], 0]):
        with pytest.raises(ValueError, match="exp table"):
            anvil_mi355x.compile((m, {**consts, "f.exp": bad}))
    with pytest.raises(ValueError, match="sound int32 proof"):
        anvil_mi355x.compile((m, consts), prove=False)


def test_the_oracles_op_checks_int32():
    m, consts = eg.layer(6, 16, 8, 3, 2, False, residual=None)
    op = next(o for o in g.func_of(m).ops if isinstance(o, g.ExpertsOp))
    x = np.full((6, 16), 127)
    op.props["Mc"] = 1 << 30
    with pytest.raises(OverflowError):
        interp.run(m, {"x": x}, consts)


# ------------------------------------------------------------------------------------------ compiled models

@pytest.fixture
def fake(monkeypatch):
    dev = eg.ExpertDevice()
    monkeypatch.setattr(rt, "device", lambda index=0: dev)
    return dev


def _check(m, consts, batch, keep, lead=(), seed=0, **run):
    cm = anvil_mi355x.compile((m, consts))
    rng = np.random.default_rng(seed)
    ins = {}
    for op in cm.input_ops:
        t = g.qt(op.result)
        n = 128 if t.dtype == "i8" else 20000
        ins[op.sym_str] = rng.integers(-n, n, (batch, *t.dims))
    want = interp.run(m, ins, consts, batch=True, fast=True)
    res = cm.run(list(ins.values()), "mi355x", batch=True, quantized=True, keep=keep, **run)
    got = res.ints
    for k, v in got.items():
        np.testing.assert_array_equal(v, want.values[k], err_msg=k)
    if keep == "all":
        assert set(got) == {k for k in want.values if k not in consts}
    return cm


CASES = [(True, "i8"), (False, "swapped"), (True, None), (False, "i16"), (True, "i16 before")]


@pytest.mark.parametrize("gated,residual", CASES)
@pytest.mark.parametrize("keep", ["outputs", "all"])
def test_plans_on_the_stand_in(fake, gated, residual, keep):
    m, consts = eg.layer(9, 32, 24, 5, 2, gated, residual)
    _check(m, consts, 3, keep)
    kinds = [c if isinstance(c, str) else c[0] for c in fake.calls]
    assert [k for k in kinds if k.startswith("expert")] == ["expert_route", "expert_gemm", "expert_gemm", "expert_combine"]
    # the residual's add rides on the weighted sums where those alone are read and the residual stands before them
    assert kinds.count("add") == (1 if residual == "i16" or residual is not None and keep == "all" else 0)


def test_plan_with_a_lead_dim_and_one_expert(fake):
    m, consts = eg.layer(4, 16, 8, 1, 1, False, "i8", lead=(3,))
    _check(m, consts, 2, "all")


@gpu
@pytest.mark.parametrize("gated,residual", CASES)
@pytest.mark.parametrize("shape", [(1, 32, 24, 4, 1), (40, 64, 128, 8, 2), (33, 100, 77, 6, 3), (256, 128, 256, 16, 4)], ids=str)
def test_compiled_models(shape, gated, residual):
    T, C, width, experts, top = shape
    m, consts = eg.layer(T, C, width, experts, top, gated, residual, seed=T)
    for batch in (1, 5):
        for keep in ("outputs", "all"):
            cm = _check(m, consts, batch, keep, seed=batch)
    for n in range(3):
        _check(m, consts, 2, "outputs", seed=n, graph=True)
    res = cm.run([np.zeros((5, T, C), int)] * len(cm.input_ops), "mi355x", batch=True, quantized=True)
    assert res.stray_writes() == []


SPEC = models.BlockSpec(n_embd=64, n_head=2, seq=48, layers=2, vocab=97, calib_batches=1, calib_batch=2)


def _model(gated):
    return eg.with_experts(models.build(SPEC, 5, stored=False), 5, 2, gated)


@pytest.mark.parametrize("gated", [False, True])
def test_a_token_model_on_the_stand_in(fake, gated):
    b = _model(gated)
    ids = np.random.default_rng(1).integers(0, SPEC.vocab, (2, SPEC.seq))
    x = np.clip(np.rint(models.embed(SPEC, b.params, ids) / b.scales["x"]), -128, 127).astype(np.int64)
    cm = anvil_mi355x.compile((b.module, b.consts))
    res = cm.run(x, "mi355x", batch=True, quantized=True)
    want = interp.run(b.module, {"x": x}, b.consts, batch=True, fast=True).outputs[0]
    assert np.array_equal(res.ints["logits"], want) and np.ptp(want) > 40


@gpu
@pytest.mark.parametrize("gated", [False, True])
def test_a_token_model_and_its_decoder(gated):
    """The whole graph, eager and captured; then token by token, beams and prompts of different lengths, against the oracle."""
    b = _model(gated)
    cm = anvil_mi355x.compile((b.module, b.consts), embedding=(b.params["wte"], b.params["wpe"]))
    ids = np.random.default_rng(1).integers(0, SPEC.vocab, (3, SPEC.seq))
    x = np.clip(np.rint(models.embed(SPEC, b.params, ids) / b.scales["x"]), -128, 127).astype(np.int64)
    want = interp.run(b.module, {"x": x}, b.consts, batch=True, fast=True).outputs[0]
    for graph in (None, None, None, True, False):
        assert np.array_equal(cm.run(ids, "mi355x", tokens=True, batch=True, graph=graph).ints["logits"], want)
    oracle, dec = Oracle(b), cm.decoder(rows=6)
    prompts = prompts_of(SPEC, [1, 20, 7], 3)
    for beams in (1, 2):
        same(dec.generate(prompts, 9, beams=beams), oracle.generate(prompts, 9, beams))


@pytest.mark.parametrize("C,width", [(65552, 8), (8, 65537)])
def test_sums_longer_than_the_kernels_take_are_refused(C, width):
    b = g.GraphBuilder("long")
    x, scores, up, down = b.input("x", [1, C], "i8"), b.input("s", [1, 2], "i8"), b.const("u", [2, C, width], "i8"), b.const("d", [2, width, 4], "i8")
    with pytest.raises(g.VerifyException, match="65536"):
        b.experts("y", x, scores, up, down, b.const("e", [256], "i32"), b.const("a", [256], "i8"), 1, 127, 1, 20, 1, 20, 1, 7)


# --------------------------------------------------------------------------------- operands that are shared

def _shared():
    """One input as rows and as scores of two experts ops with the same consts, whose results meet in an add; the first is an output
    too, and its weights are a batch product's right operand as well. A third op's rows and a fourth's scores are consts."""
    E, C, width, T = 16, 16, 32, 6
    b, feed = g.GraphBuilder("shared"), eg.Feed("f", C, width, C, E, 3, True, 4)
    rng = np.random.default_rng(9)
    consts = {k: v for k, v in feed.values().items() if not k.endswith("router")}
    consts["rows"] = rng.integers(-128, 128, (T, C))
    x, each = b.input("x", [T, C], "i8", 0.05), b.input("each", [E, T, C], "i8", 0.05)
    c = {k: b.const(k, list(v.shape), "i32" if k == "f.exp" else "i8") for k, v in consts.items()}

    def part(sym, x, scores):
        return b.experts(sym, x, scores, c["f.up"], c["f.down"], c["f.exp"], c["f.act"], 3, feed.one, gate=c["f.gate"], **feed.args)

    y1 = part("y1", x, x)
    y2 = part("y2", y1, x)
    y3, y4 = part("y3", c["rows"], x), part("y4", x, c["rows"])
    m, s = eg.requant(45, 74 * 40 * np.sqrt(C), 128 * int(np.abs(consts["f.up"]).sum(axis=1).max()))
    z = b.qmatmul("z", each, c["f.up"], m, s)
    b.output(b.add_requant("both", y1, y2, 60, 70, 6, 0.05), y1, b.add_requant("third", y3, x, 60, 70, 6, 0.05), y4, z)
    return b.module(), consts


@pytest.mark.parametrize("keep", ["outputs", "all"])
def test_shared_operands_on_the_stand_in(fake, keep):
    _check(*_shared(), 3, keep)


@gpu
@pytest.mark.parametrize("keep", ["outputs", "all"])
def test_shared_operands(keep):
    cm = _check(*_shared(), 3, keep)
    assert cm.proven
