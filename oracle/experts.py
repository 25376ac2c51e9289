"""ORACLE (test infrastructure only): numpy restatement, in 64 bits, of the operators of an experts' feed-forward: the residual's
addition with a norm whose rows have scales of their own, the router with the sort by expert, the experts' products, and the
weighted sums back in the rows' order. Row by row and without tiles; each value is an int64."""
import numpy as np

from . import semantics as sem


def rq(v, m, s):
    """(v * m + 2^(s-1)) >> s."""
    return (np.asarray(v, dtype=np.int64) * m + ((1 << s) >> 1)) >> s


def add_norm(x, y, ma, mb, shift, r_dtype, w, lut, eps, lut_shift):
    """(r, codes, scales) of rows x (+ y)."""
    r = np.asarray(x, dtype=np.int64)
    if y is not None:
        r = sem.clamp_dtype(rq(r * ma + np.asarray(y, dtype=np.int64) * mb, 1, shift), r_dtype)
    t = r * np.asarray(w, dtype=np.int64)
    a = np.abs(t).max(axis=1)
    codes = np.sign(t) * ((254 * np.abs(t) + a[:, None]) // np.maximum(2 * a, 1)[:, None])
    idx, k = sem.rsqrt_index(eps + (r * r).sum(axis=1), len(lut))
    v = a * np.maximum(0, np.asarray(lut, dtype=np.int64))[idx]
    s = lut_shift + k
    return r, codes, np.minimum(32767, (v + ((np.int64(1) << s) >> 1)) >> s)


def route(scores, live, top, lut, one, every=False):
    """(expert, weight, slot, row, starts); row has the used positions only. A row whose sum is 0 has weights 0."""
    scores, lut = np.asarray(scores, dtype=np.int64), np.maximum(0, np.asarray(lut, dtype=np.int64))
    n, E = scores.shape
    expert, weight, slot = (np.full((n, top), v, dtype=np.int64) for v in (-1, 0, -1))
    lists = [[] for _ in range(E)]
    for i in range(n):
        if live is not None and not live[i]:
            continue
        order = sorted(range(E), key=lambda e: (-scores[i, e], e))[:top]
        e = lut[scores[i, order] - scores[i].max() + 255]
        S = int((lut[scores[i] - scores[i].max() + 255] if every else e).sum())
        expert[i] = order
        weight[i] = [(int(v) * one + S // 2) // S for v in e] if S else 0
        for j, o in enumerate(order):
            lists[o].append((i, j))
    starts, row = [0], []
    for pairs in lists:
        for i, j in pairs:
            slot[i, j] = len(row)
            row.append(i)
        starts.append(len(row))
    return expert, weight, slot, np.array(row, dtype=np.int64), np.array(starts, dtype=np.int64)


def gemm(out, A, row, scale, B, B2, starts, mults, shift, mults2, shift2, lut, mult3, shift3, dtype):
    """The experts' products into a copy of `out`, whose other rows stay."""
    out, A = np.array(out, dtype=np.int64), np.asarray(A, dtype=np.float64)
    for e in range(len(starts) - 1):
        at = np.arange(starts[e], starts[e + 1])
        if not at.size:
            continue
        i = at if row is None else np.asarray(row)[at]
        s = 1 if scale is None else np.asarray(scale, dtype=np.int64)[i][:, None]

        def product(W, m, sh, to):                             # sums below 2^53: exact in float64
            acc = np.rint(A[i] @ np.asarray(W[e], dtype=np.float64).T).astype(np.int64)
            return sem.clamp_dtype(rq(acc, int(m[e]) * s, sh), to)

        v = product(B, mults, shift, dtype)
        if lut is not None:
            v = np.asarray(lut, dtype=np.int64)[v + 128]
        if B2 is not None:
            v = sem.clamp_i8(rq(v * product(B2, mults2, shift2, "i8"), mult3, shift3))
        out[at] = v
    return out


def combine(Y, slot, weight, mult, shift, R, ma, mb, shift2, dtype):
    acc = np.zeros((len(slot), Y.shape[1]), dtype=np.int64)
    for j in range(slot.shape[1]):
        have = slot[:, j] >= 0
        acc[have] += np.asarray(weight, dtype=np.int64)[have, j][:, None] * np.asarray(Y, dtype=np.int64)[slot[have, j]]
    y = sem.clamp_i8(rq(acc, mult, shift))
    return y if R is None else sem.clamp_dtype(rq(np.asarray(R, dtype=np.int64) * ma + y * mb, 1, shift2), dtype)


def graph_op(x, scores, up, down, exp, act, top, one, m, s, md, sd, mc, sc, gate=None, mg=0, sg=0, mm=0, sm=0, fast=False):
    """The graph's experts op on rows (..., C) with scores (..., E), every intermediate checked against int32 as the other ops' are."""
    exp = sem.check_i32(exp, "exp table")
    if exp.shape != (256,) or exp.min() < 0 or exp[-1] < 1:
        raise ValueError("the exp table needs 256 entries >= 0 and a last one >= 1")
    lead = np.broadcast_shapes(x.shape[:-1], scores.shape[:-1])    # a const is the same in every batch
    x, scores = (np.broadcast_to(v, (*lead, v.shape[-1])).reshape(-1, v.shape[-1]) for v in (x, sem.check_i8(scores, "scores")))
    expert = np.argsort(-scores, axis=1, kind="stable")[:, :top]
    mine = np.take_along_axis(scores, expert, 1)
    e = exp[mine - mine[:, :1] + 255]
    S = sem.check_i32(e.sum(axis=1, keepdims=True), "sum of exps")
    weight = sem.check_i32(e * one + S // 2, "e*one + S/2") // S
    y = np.zeros((len(x), top, down.shape[-1]), dtype=np.int64)
    for n in range(len(up)):
        row, j = np.nonzero(expert == n)
        if not row.size:
            continue
        h = sem.qmatmul(x[row], up[n], m, s, act if gate is None else None, fast=fast)
        if gate is not None:
            h = sem.swiglu_lut(sem.qmatmul(x[row], gate[n], mg, sg, fast=fast), h, act, mm, sm)
        y[row, j] = sem.qmatmul(h, down[n], md, sd, fast=fast)
    acc = sem.check_i32((weight[:, :, None] * y).sum(axis=1), "weighted sum")
    return sem.requant(acc, mc, sc).reshape(*lead, -1)
