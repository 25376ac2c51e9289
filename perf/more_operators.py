"""The operators of a feed-forward part made of experts, through this backend's public entry points.

Five families, each a dict of plain values:

    norm      the residual's addition, then a root-mean-square norm whose int8 codes have a scale of their own for each row
    route     each token's best experts, their weights, and the tokens sorted by expert
    experts   the experts' products over the sorted tokens: plain, with a table behind, or a gate's table times a second product
    combine   the sorted results back in the tokens' order, weighted, and added to the residual
    layer     all of it in a row, as a program runs it: norm, scores, route, two products, combine

Everything is an integer, so outputs are compared exactly. With rq(v, m, s) = clamp((v m + 2^(s-1)) >> s) in 64 bits:

    norm      r = rq(x ma + y mb, 1, s); t = r w; a = max |t|; code = sign(t) floor((254 |t| + a) / 2a);
              scale = min(32767, (a lut[i] + 2^(s'+k-1)) >> (s' + k)), i = (eps + sum r^2) >> 2k, the least k with i < len(lut)
    route     weights floor((e one + S/2) / S), e = lut[x - largest x + 255], S their sum over the chosen (or all) experts; ties go to
              the lowest expert; an expert's tokens stay in order
    experts   rq(sum of a b, mult of the expert x scale of the row, s)
    combine   y = rq(sum of weight x row, m, s), rq(r ma + y mb, 1, s')
"""
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

ROOT = Path(__file__).resolve().parents[1]
BITS = {"i8": 8, "i16": 16}
TORCH = {"i8": torch.int8, "i16": torch.int16}
TABLE = 1024                                                 # entries of the reciprocal square roots
ONE = 16384                                                  # a weight of 1
EPS = 16


# ------------------------------------------------------------------------------------------------------ cases

def _norm(rows, cols, x="i16", y="i8", r="i16"):
    return {"family": "norm", "rows": rows, "cols": cols, "x": x, "y": y, "r": r}


def _route(rows, experts, top, masked=False, every=False):
    return {"family": "route", "rows": rows, "experts": experts, "top": top, "masked": masked, "every": every}


def _experts(rows, experts, top, cols, width, kind="gated", scaled=True, gather=True, out="i8", masked=False):
    return {"family": "experts", "rows": rows, "experts": experts, "top": top, "cols": cols, "width": width, "kind": kind,
            "scaled": scaled, "gather": gather, "out": out, "masked": masked}


def _combine(rows, experts, top, cols, residual="i16", out="i16", masked=False):
    return {"family": "combine", "rows": rows, "experts": experts, "top": top, "cols": cols, "residual": residual, "out": out,
            "masked": masked}


def _layer(rows, experts, top, cols, width, gated=True):
    return {"family": "layer", "rows": rows, "experts": experts, "top": top, "cols": cols, "width": width, "gated": gated}


def listed():
    named = [
        # one token of the GPT-2-small-shaped block: the latency of a call; the benchmark's whole batch of that block
        ("norm-token", _norm(1, 768)),
        ("norm-prompts", _norm(32768, 768)),
        # one token and a batch of prompts whose padding has no expert
        ("route-token", _route(1, 8, 2)),
        ("route-prompts", _route(32749, 64, 6, masked=True)),
        # one step of a serving batch over many small experts: their weights are what is read
        ("experts-step", _experts(64, 64, 4, 1024, 1408)),
        # the benchmark's batch over eight experts: gate and up, and back down
        ("experts-prompts", _experts(32768, 8, 2, 768, 2048)),
        ("experts-down", _experts(32768, 8, 2, 2048, 768, "plain", scaled=False, gather=False)),
        # sizes that no tile fits, a table behind the product
        ("experts-odd", _experts(3001, 11, 3, 500, 333, "table", masked=True)),
        # a serving batch's step, and the benchmark's batch
        ("combine-step", _combine(64, 64, 8, 1024, "i8", "i8")),
        ("combine-prompts", _combine(32768, 8, 2, 768)),
        # the whole part: a step of sixteen sequences, and eight prompts of the benchmark's length
        ("layer-step", _layer(16, 32, 4, 768, 1024)),
        ("layer-prompts", _layer(8192, 16, 2, 768, 2048)),
    ]
    return [dict(c, name=n) for n, c in named]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _top(rng, experts):
    return rng.randint(1, min(experts, 8))


def draw(rng):
    family = rng.choice(["norm", "route", "combine", "experts", "experts", "experts", "layer"])
    while True:
        rows, experts = _log(rng, 1, 32768), _log(rng, 2, 256)
        top, masked = _top(rng, experts), rng.random() < 0.3
        cols, width = _log(rng, 16, 8192), _log(rng, 16, 8192)
        if rng.random() < 0.7:                               # as models have them
            cols, width = (max(64, c // 64 * 64) for c in (cols, width))
        if family == "norm" and rows * cols <= 1 << 25:
            return _norm(rows, cols, rng.choice(["i8", "i16", "i16"]), rng.choice(["i8", "i8", "i16", "none"]),
                         rng.choice(["i8", "i16", "i16"]))
        if family == "route" and rows * experts <= 1 << 22:
            return _route(rows, experts, top, masked, rng.random() < 0.3)
        if family == "combine" and rows * top * cols <= 1 << 26:
            return _combine(rows, experts, top, cols, rng.choice(["none", "i8", "i16", "i16"]), rng.choice(["i8", "i16", "i16"]),
                            masked)
        if family == "experts":
            kind = rng.choice(["gated", "plain", "table"])
            twice = 2 if kind == "gated" else 1
            if rows * top * cols * width * twice <= 1 << 37 and experts * cols * width * twice <= 1 << 28 and \
                    rows * top * max(cols, width) <= 1 << 28:
                return _experts(rows, experts, top, cols, width, kind, rng.random() < 0.6, rng.random() < 0.7,
                                rng.choice(["i8", "i8", "i16"]) if kind == "plain" else "i8", masked)
        if family == "layer" and rows * top * cols * width <= 1 << 35 and experts * cols * width <= 1 << 27 and cols <= 4096:
            return _layer(rows, experts, top, cols, width, rng.random() < 0.7)


# ----------------------------------------------------------------------------------------------------- inputs

class State:
    """What a program holds: tensors and plain values by name."""

    def __init__(self, **kw):
        self.__dict__.update(kw)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, shape, spread, bits=8):
    top = (1 << bits - 1) - 1
    return (torch.randn(shape, generator=gen, device="cuda") * spread).round().clamp(-top - 1, top).to(
        torch.int8 if bits == 8 else torch.int16)


def _empty(shape, dtype):
    return torch.zeros(shape, dtype=dtype, device="cuda")


def _i32(v):
    return torch.as_tensor(np.asarray(v, dtype=np.int32)).cuda()


def _fixed(ratio, bits):
    """(multiplier, shift) of a ratio, the multiplier of so many bits."""
    s = 0
    while round(ratio * (1 << s + 1)) < 1 << bits and s < 62:
        s += 1
    return max(1, round(ratio * (1 << s))), s


def _roots(cols):
    """Reciprocal square roots such that a row's scale is 1024 times what a code of 1 stands for."""
    root = np.sqrt(np.maximum(0.5, np.arange(TABLE)))
    return np.rint((1 << 16) * 1024 * math.sqrt(cols) / 127 / root).astype(np.int64), 16


def _act():
    """An int8 table of a smooth activation, inputs and results in steps of 1 / 16."""
    x = np.arange(-128, 128) / 16
    return torch.as_tensor(np.clip(np.rint(x / (1 + np.exp(-x)) * 16), -128, 127).astype(np.int8)).cuda()


def _exp():
    return _i32(np.rint(np.exp(np.arange(-255, 1) * 0.09) * (1 << 20)))


def _scores(rows, experts, gen):
    """Router scores: some experts are more popular than others."""
    liked = torch.randn(experts, generator=torch.Generator().manual_seed(7)).cuda() * 10
    return (torch.randn((rows, experts), generator=gen, device="cuda") * 25 + liked).round().clamp(-128, 127).to(torch.int8)


def _live(case, gen):
    """Padding: rows without experts."""
    if not case.get("masked"):
        return None
    return (torch.rand(case["rows"], generator=gen, device="cuda") < 0.9).to(torch.uint8)


def _norm_state(rows, cols, x, y, r, gen):
    lut, shift = _roots(cols)
    loud = torch.ones(cols, device="cuda")
    loud[::97] = 6                                           # channels of outliers
    spread = {"i8": 24, "i16": 2500}
    X = (torch.randn((rows, cols), generator=gen, device="cuda") * (spread[x] * loud)).round().clamp(
        -(1 << BITS[x] - 1), (1 << BITS[x] - 1) - 1).to(TORCH[x])
    Y = None if y == "none" else _normal(gen, (rows, cols), 30 if y == "i8" else 3000, BITS[y])
    if y == "none":
        r = x
    scale = {"i8": 100, "i16": 1} if "i16" == r else {"i8": 1, "i16": 0.01}
    ma, mb = (max(1, round(scale[t] * (1 << 8))) for t in (x, x if y == "none" else y))
    w = (torch.randn(cols, generator=gen, device="cuda") * 16 + 64).round().clamp(-127, 127).to(torch.int8)
    return State(family="norm", X=X, Y=Y, w=w, ma=ma, mb=mb, s=8, lut=_i32(lut), eps=EPS, shift=shift, r=r,
                 R=None if Y is None else _empty((rows, cols), TORCH[r]), H=_empty((rows, cols), torch.int8),
                 scale=_empty(rows, torch.int16))


def _prepare_norm(case, seed):
    return _norm_state(case["rows"], case["cols"], case["x"], case["y"], case["r"], _gen(seed))


def _route_buffers(rows, experts, top):
    return dict(expert=_empty((rows, top), torch.int32), weight=_empty((rows, top), torch.int16), slot=_empty((rows, top), torch.int32),
                row=_empty(rows * top, torch.int32), starts=_empty(experts + 1, torch.int32))


def _prepare_route(case, seed):
    gen = _gen(seed)
    return State(family="route", scores=_scores(case["rows"], case["experts"], gen), live=_live(case, gen), top=case["top"],
                 every=case["every"], lut=_exp(), one=ONE, **_route_buffers(case["rows"], case["experts"], case["top"]))


def _routed(case, gen):
    """What a router has left behind: weights, slots, sorted rows and starts."""
    s = State(scores=_scores(case["rows"], case["experts"], gen), live=_live(case, gen), top=case["top"], every=False, lut=_exp(),
              one=ONE, **_route_buffers(case["rows"], case["experts"], case["top"]))
    return _plain_route(s)


def _weights(gen, experts, width, cols):
    return _normal(gen, (experts, width, cols), 40)


def _product(gen, experts, spread, cols, scaled, bits, gain=40):
    """Multipliers of the experts and a shift: results of that spread."""
    base = gain / (spread * 40 * math.sqrt(cols)) / (3000 if scaled else 1)
    m, s = _fixed(base, bits)
    return (m * (0.75 + 0.5 * torch.rand(experts, generator=gen, device="cuda"))).int(), s


def _prepare_experts(case, seed):
    gen = _gen(seed)
    E, C, N = case["experts"], case["cols"], case["width"]
    got = _routed(case, gen)
    pairs = case["rows"] * case["top"]
    n = case["rows"] if case["gather"] else pairs
    gated = case["kind"] == "gated"
    mults, s = _product(gen, E, 40, C, case["scaled"], 14, 4000 if case["out"] == "i16" else 40)
    s2 = _product(gen, E, 40, C, case["scaled"], 14) if gated else (None, 0)
    m3, s3 = _fixed(1 / 40, 7)
    return State(family="experts", A=_normal(gen, (n, C), 40), row=got["row"] if case["gather"] else None, starts=got["starts"],
                 scale=torch.randint(1500, 4500, (n,), generator=gen, device="cuda", dtype=torch.int16) if case["scaled"] else None,
                 B=_weights(gen, E, N, C), B2=_weights(gen, E, N, C) if gated else None, mults=mults, s=s, mults2=s2[0], s2=s2[1],
                 table=None if case["kind"] == "plain" else _act(), m3=m3, s3=s3, out=_empty((pairs, N), TORCH[case["out"]]))


def _prepare_combine(case, seed):
    gen = _gen(seed)
    got = _routed(case, gen)
    res, out = case["residual"], case["out"]
    m, s = _fixed(1.5 / ONE, 14)
    wide = {"i8": 1, "i16": 100}
    ma, mb = (1 << 8) * wide[out] // wide.get(res, 1), 300 * wide[out]
    return State(family="combine", Y=_normal(gen, (case["rows"] * case["top"], case["cols"]), 40), slot=got["slot"], weight=got["weight"],
                 m=m, s=s, R=None if res == "none" else _normal(gen, (case["rows"], case["cols"]), 24 if res == "i8" else 2500, BITS[res]),
                 ma=max(1, ma), mb=mb, s2=8, D=_empty((case["rows"], case["cols"]), torch.int8 if res == "none" else TORCH[out]))


def _prepare_layer(case, seed):
    gen = _gen(seed)
    T, E, k, C, N = case["rows"], case["experts"], case["top"], case["cols"], case["width"]
    norm = _norm_state(T, C, "i16", "i8", "i16", gen)
    gated = case["gated"]
    scores = _empty((T, E), torch.int8)
    route = State(scores=scores, live=None, top=k, every=False, lut=_exp(), one=ONE, **_route_buffers(T, E, k))
    m1, s1 = _product(gen, 1, 40, C, True, 14, 25)
    router = State(A=norm.H, row=None, starts=_i32([0, T]), scale=norm.scale, B=_weights(gen, 1, E, C), B2=None, mults=m1, s=s1,
                   mults2=None, s2=0, table=None, m3=1, s3=0, out=scores)
    mu, su = _product(gen, E, 40, C, True, 14)
    mg, sg = _product(gen, E, 40, C, True, 14) if gated else (None, 0)
    m3, s3 = _fixed(1 / 40, 7)
    up = State(A=norm.H, row=route.row, starts=route.starts, scale=norm.scale, B=_weights(gen, E, N, C),
               B2=_weights(gen, E, N, C) if gated else None, mults=mu, s=su, mults2=mg, s2=sg, table=_act(), m3=m3, s3=s3,
               out=_empty((T * k, N), torch.int8))
    md, sd = _product(gen, E, 20, N, False, 14)
    down = State(A=up.out, row=None, starts=route.starts, scale=None, B=_weights(gen, E, C, N), B2=None, mults=md, s=sd, mults2=None,
                 s2=0, table=None, m3=1, s3=0, out=_empty((T * k, C), torch.int8))
    mc, sc = _fixed(1.2 / ONE, 14)
    combine = State(Y=down.out, slot=route.slot, weight=route.weight, m=mc, s=sc, R=norm.R, ma=1 << 8, mb=30000, s2=8,
                    D=_empty((T, C), torch.int16))
    return State(family="layer", norm=norm, router=router, route=route, up=up, down=down, combine=combine)


PREPARE = {"norm": _prepare_norm, "route": _prepare_route, "experts": _prepare_experts, "combine": _prepare_combine,
           "layer": _prepare_layer}


def _framework():
    path = str(ROOT / "anvil-compiler_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from anvil_mi355x import runtime
    return runtime


def prepare(case, seed):
    s = PREPARE[case["family"]](case, seed)
    if own:
        s.dev = _framework().device(0)
        torch.cuda.synchronize()
    return s


# -------------------------------------------------------------------------------------------------- one pass

NAME = {torch.int8: "i8", torch.int16: "i16"}


def _ptr(t):
    return None if t is None else t.data_ptr()


def _own_norm(s, dev):
    rows, cols = s.X.shape
    dev.add_norm(s.X.data_ptr(), NAME[s.X.dtype], cols, _ptr(s.Y), s.r if s.Y is None else NAME[s.Y.dtype], cols, s.ma, s.mb, s.s,
                 _ptr(s.R), s.r, cols, s.w.data_ptr(), s.lut.data_ptr(), len(s.lut), s.eps, s.shift, s.H.data_ptr(), cols,
                 s.scale.data_ptr(), rows, cols)
    return {"h": s.H, "scale": s.scale} if s.Y is None else {"r": s.R, "h": s.H, "scale": s.scale}


def _own_route(s, dev):
    rows, experts = s.scores.shape
    dev.expert_route(s.scores.data_ptr(), experts, _ptr(s.live), rows, experts, s.top, s.lut.data_ptr(), s.one, s.expert.data_ptr(),
                     s.weight.data_ptr(), s.slot.data_ptr(), s.row.data_ptr(), s.starts.data_ptr(), every=s.every)
    return {"expert": s.expert, "weight": s.weight, "slot": s.slot, "row": s.row, "starts": s.starts}


def _own_experts(s, dev):
    n, C = s.A.shape
    E, N, _ = s.B.shape
    dev.expert_gemm(s.A.data_ptr(), C, n, _ptr(s.row), _ptr(s.scale), s.B.data_ptr(), _ptr(s.B2), C, N * C, s.starts.data_ptr(), E,
                    len(s.out), N, C, s.out.data_ptr(), N, NAME[s.out.dtype], mults=s.mults.data_ptr(), shift=s.s,
                    mults2=_ptr(s.mults2), shift2=s.s2, lut=_ptr(s.table), mult3=s.m3, shift3=s.s3)
    return {"out": s.out}


def _own_combine(s, dev):
    rows, cols = s.D.shape
    dev.expert_combine(s.Y.data_ptr(), cols, len(s.Y), s.slot.data_ptr(), s.weight.data_ptr(), rows, s.slot.shape[1], cols, s.m, s.s,
                       _ptr(s.R), "i8" if s.R is None else NAME[s.R.dtype], cols, s.ma, s.mb, s.s2, s.D.data_ptr(), NAME[s.D.dtype],
                       cols)
    return {"d": s.D}


def _clamp(x, dtype):
    info = torch.iinfo(dtype)
    return x.clamp(info.min, info.max).to(dtype)


def _requant(x, m, s):
    return (x * m + (1 << s >> 1)) >> s


def _plain_norm(s):
    r = s.X.int()
    if s.Y is not None:
        s.R.copy_(_clamp(_requant(r.long() * s.ma + s.Y.long() * s.mb, 1, s.s), s.R.dtype))
        r = s.R.int()
    t = r * s.w.int()
    size = t.abs()
    a = size.amax(1, keepdim=True)
    code = torch.div(254 * size + a, (2 * a).clamp(min=1), rounding_mode="floor")
    s.H.copy_(code * t.sign())
    ss = s.eps + (r * r).sum(1, dtype=torch.int64)
    bits = torch.frexp(ss.double()).exponent.long()                  # 2^(bits-1) <= ss < 2^bits
    k = (bits - TABLE.bit_length() + 2).clamp(min=0) // 2            # the least one with ss >> 2k below the table's length
    shift = s.shift + k
    v = a[:, 0].long() * s.lut.long()[ss >> 2 * k]
    s.scale.copy_(((v + ((1 << shift) >> 1)) >> shift).clamp(max=32767))
    return {"h": s.H, "scale": s.scale} if s.Y is None else {"r": s.R, "h": s.H, "scale": s.scale}


def _plain_route(s):
    rows, E = s.scores.shape
    x = s.scores.int()
    key = (x * E + torch.arange(E - 1, -1, -1, device=x.device)).topk(s.top, dim=1).values       # no two alike
    expert = E - 1 - key % E
    top = x.gather(1, expert.long())
    e = s.lut.long()[top - top[:, :1] + 255]
    total = s.lut.long()[x - top[:, :1] + 255].sum(1, keepdim=True) if s.every else e.sum(1, keepdim=True)
    weight = (e * s.one + total // 2) // total
    live = torch.ones(rows, dtype=torch.bool, device=x.device) if s.live is None else s.live != 0
    s.expert.copy_(torch.where(live[:, None], expert, -1))
    s.weight.copy_(torch.where(live[:, None], weight, 0))
    group = torch.where(live[:, None], expert, E).view(-1).long()
    order = torch.sort(group, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(len(order), device=x.device)
    s.slot.copy_(torch.where(live[:, None], place.view(rows, -1), -1))
    counts = torch.zeros(E + 1, dtype=torch.int64, device=x.device).index_add_(0, group, torch.ones_like(group))
    s.starts.zero_()
    s.starts[1:] = counts[:E].cumsum(0)
    used = torch.arange(len(order), device=x.device) < s.starts[E]
    s.row.copy_(torch.where(used, (order // s.top).int(), s.row))
    return {"expert": s.expert, "weight": s.weight, "slot": s.slot, "row": s.row, "starts": s.starts}


def _dot(a, b):
    """a @ b^T of int8 values: pieces whose sums stay below 2^24, exact in 32 bits."""
    out = 0
    for k in range(0, a.shape[1], 1024):
        out = out + (a[:, k:k + 1024].float() @ b[:, k:k + 1024].float().t()).long()
    return out


def _plain_experts(s):
    starts = s.starts.tolist()
    for e, (lo, hi) in enumerate(zip(starts, starts[1:])):
        if lo == hi:
            continue
        at = torch.arange(lo, hi, device=s.A.device) if s.row is None else s.row[lo:hi].long()
        a = s.A[at]
        scale = 1 if s.scale is None else s.scale[at].long()[:, None]
        v = _requant(_dot(a, s.B[e]), s.mults[e].long() * scale, s.s)
        if s.table is not None:
            v = s.table[v.clamp(-128, 127) + 128].long()
        if s.B2 is not None:
            u = _requant(_dot(a, s.B2[e]), s.mults2[e].long() * scale, s.s2).clamp(-128, 127)
            v = _requant(v * u, s.m3, s.s3)
        s.out[lo:hi] = _clamp(v, s.out.dtype)
    return {"out": s.out}


def _plain_combine(s):
    rows = s.Y[s.slot.clamp(min=0).long()].int()                                    # rows, top, cols
    weight = torch.where(s.slot >= 0, s.weight.int(), 0)[:, :, None]
    y = _requant((rows * weight).sum(1, dtype=torch.int64), s.m, s.s).clamp(-128, 127)
    s.D.copy_(y if s.R is None else _clamp(_requant(s.R.long() * s.ma + y * s.mb, 1, s.s2), s.D.dtype))
    return {"d": s.D}


OWN = {"norm": _own_norm, "route": _own_route, "experts": _own_experts, "combine": _own_combine}
PLAIN = {"norm": _plain_norm, "route": _plain_route, "experts": _plain_experts, "combine": _plain_combine}


def run(state):
    call = (lambda f, s: OWN[f](s, state.dev)) if own else (lambda f, s: PLAIN[f](s))
    if state.family != "layer":
        return call(state.family, state)
    out = call("norm", state.norm)
    call("experts", state.router)
    out = dict(out, **call("route", state.route))
    call("experts", state.up)
    call("experts", state.down)
    return dict(out, **call("combine", state.combine))


# ------------------------------------------------------------------------------------------- what it must do

def _used_experts(case):
    """How many experts get a token, of random scores with the case's popular ones."""
    rows = min(case["rows"], 2048)
    if case["experts"] * 8 <= rows * case["top"] / 8:
        return case["experts"]
    liked = torch.randn(case["experts"], generator=torch.Generator().manual_seed(7)).numpy() * 10
    x = np.random.default_rng(0).normal(size=(rows, case["experts"])) * 25 + liked
    return len(np.unique(np.argsort(-x, axis=1)[:, :case["top"]]))


def work(case):
    """Each input read once, each result written once: of the weights those of the experts that have a token."""
    f, T = case["family"], case["rows"]
    size = {"i8": 1, "i16": 2, "none": 0}

    def norm(C, x, y, r):
        return T * C * (size[x] + size[y] + (0 if y == "none" else size[r]) + 1) + 2 * T + C + 4 * TABLE, 8 * T * C

    def route(E, k):
        return T * E + 14 * T * k + 4 * E + 1024, 2 * T * E

    def product(pairs, rows, used, C, N, gated, out=1):
        return rows * C + used * N * C * (2 if gated else 1) + pairs * N * out, 2 * pairs * N * C * (2 if gated else 1)

    def combine(k, C, res, out):
        return T * k * (C + 6) + T * C * (size[res] + size[out]), 2 * T * k * C

    if f == "norm":
        parts = [norm(case["cols"], case["x"], case["y"], case["r"])]
    elif f == "route":
        parts = [route(case["experts"], case["top"])]
    elif f == "combine":
        parts = [combine(case["top"], case["cols"], case["residual"], "i8" if case["residual"] == "none" else case["out"])]
    elif f == "experts":
        pairs = T * case["top"]
        parts = [product(pairs, T if case["gather"] else pairs, _used_experts(case), case["cols"], case["width"], case["kind"] == "gated",
                         size[case["out"]])]
    else:
        E, k, C, N, used = case["experts"], case["top"], case["cols"], case["width"], _used_experts(case)
        parts = [norm(C, "i16", "i8", "i16"), product(T, T, 1, C, E, False), route(E, k), product(T * k, T, used, C, N, case["gated"]),
                 product(T * k, T * k, used, N, C, False), combine(k, C, "i16", "i16")]
    return {"bytes": sum(p[0] for p in parts), "flops": sum(p[1] for p in parts)}


# ------------------------------------------------------------------------------------------ the same in 64 bits

def _half_up(v, s):
    """floor(v / 2^s + 1 / 2) of whole numbers, 1/2 only where s is not 0."""
    return v if s == 0 else torch.div(torch.div(v, 1 << s - 1, rounding_mode="floor") + 1, 2, rounding_mode="floor")


def _into(v, bits):
    return torch.minimum(torch.maximum(v, torch.full_like(v, -(1 << bits - 1))), torch.full_like(v, (1 << bits - 1) - 1))


def _exact_norm(s):
    r, got = s.X.long(), {}
    if s.Y is not None:
        r = _into(_half_up(r * s.ma + s.Y.long() * s.mb, s.s), BITS[s.r])
        got["r"] = r.to(TORCH[s.r])
    t = r * s.w.long()
    a = t.abs().max(1).values
    code = torch.floor((t.abs() * 254 + a[:, None]).double() / (2 * a[:, None]).clamp(min=1).double())
    got["h"] = torch.where(t < 0, -code, code).to(torch.int8)
    lut, scale = s.lut.tolist(), []
    for total, top in zip((s.eps + (r.double() ** 2).sum(1)).long().tolist(), a.tolist()):
        k = 0
        while total >= len(lut):
            total >>= 2
            k += 1
        k += s.shift
        scale.append(min(32767, top * lut[total] + (1 << k >> 1) >> k))
    got["scale"] = torch.tensor(scale, dtype=torch.int16, device=r.device)
    return got


def _exact_route(s):
    x, lut = s.scores.cpu().numpy().astype(np.int64), s.lut.cpu().numpy().astype(np.int64)
    rows, E = x.shape
    live = np.ones(rows, bool) if s.live is None else s.live.cpu().numpy() != 0
    expert = np.argsort(-x, axis=1, kind="stable")[:, :s.top]
    mine = np.take_along_axis(x, expert, 1)
    e = lut[255 - (mine[:, :1] - mine)]
    total = (lut[255 - (mine[:, :1] - x)] if s.every else e).sum(1)[:, None]
    weight = (2 * e * s.one + 2 * (total // 2)) // (2 * total)
    expert[~live], weight[~live] = -1, 0
    slot, row, starts = np.full_like(expert, -1), s.row.cpu().numpy().copy(), [0]
    for g in range(E):
        at, choice = np.nonzero(expert == g)
        slot[at, choice] = starts[-1] + np.arange(len(at))
        row[starts[-1]:starts[-1] + len(at)] = at
        starts.append(starts[-1] + len(at))
    put = lambda v, t: torch.as_tensor(np.ascontiguousarray(v), dtype=t).to(s.scores.device)         # noqa: E731
    return {"expert": put(expert, torch.int32), "weight": put(weight, torch.int16), "slot": put(slot, torch.int32),
            "row": put(row, torch.int32), "starts": put(np.array(starts), torch.int32)}


def _exact_experts(s):
    out = s.out.clone()
    bounds = s.starts.cpu().numpy()
    for e in range(len(bounds) - 1):
        for lo in range(int(bounds[e]), int(bounds[e + 1]), 8192):
            hi = min(lo + 8192, int(bounds[e + 1]))
            at = slice(lo, hi) if s.row is None else s.row[lo:hi].long()
            a = s.A[at].double()

            def product(B, mults, shift):
                v = (a @ B[e].double().t()).long() * int(mults[e])
                return _half_up(v if s.scale is None else v * s.scale[at].long().unsqueeze(1), shift)

            v = product(s.B, s.mults, s.s)
            if s.table is not None:
                v = s.table.long()[_into(v, 8) + 128]
            if s.B2 is not None:
                v = _half_up(v * _into(product(s.B2, s.mults2, s.s2), 8) * s.m3, s.s3)
            out[lo:hi] = _into(v, 16 if out.dtype == torch.int16 else 8).to(out.dtype)
    return {"out": out}


def _exact_combine(s):
    total = torch.zeros(s.D.shape, dtype=torch.float64, device=s.D.device)
    for j in range(s.slot.shape[1]):
        have = (s.slot[:, j] >= 0).nonzero()[:, 0]
        total[have] += s.Y[s.slot[have, j].long()].double() * s.weight[have, j].double()[:, None]
    y = _into(_half_up(total.long() * s.m, s.s), 8)
    if s.R is not None:
        y = _into(_half_up(s.R.long() * s.ma + y * s.mb, s.s2), 16 if s.D.dtype == torch.int16 else 8)
    return {"d": y.to(s.D.dtype)}


EXACT = {"norm": _exact_norm, "route": _exact_route, "experts": _exact_experts, "combine": _exact_combine}


def exact(case, seed):
    s = PREPARE[case["family"]](case, seed)
    if s.family != "layer":
        return EXACT[s.family](s)
    out = dict(EXACT["norm"](s.norm))
    s.norm.H.copy_(out["h"]), s.norm.scale.copy_(out["scale"]), s.norm.R.copy_(out["r"])
    s.route.scores.copy_(EXACT["experts"](s.router)["out"])
    route = EXACT["route"](s.route)
    for name, v in route.items():
        getattr(s.route, name).copy_(v)
    s.up.out.copy_(EXACT["experts"](s.up)["out"])
    s.down.out.copy_(EXACT["experts"](s.down)["out"])
    return dict(out, **route, **EXACT["combine"](s.combine))
