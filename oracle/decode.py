"""ORACLE (test infrastructure only): numpy restatement of the decoding operators, row by row in int64.

The attention is the reference's chain (requant of anvil/semantics.py:146-155, the three-stage softmax of
anvil/lower/graph_to_tensor.py:352-398) over the values a 4-bit cache holds; the cache, its page tables and the beam
selection have no counterpart in the reference and are restated from their definition in include/anvil_mi355x.h.
Where lengths, windows and `one` allow it, tests compare the attention with oracle.semantics' own ops.
"""
import numpy as np

PAGE = 64
NO_SCORE = -(1 << 63)


def stored_dim(dim):
    return max(32, dim)


def round4(x):
    """The values 4 bits hold for int8 rows (..., D): groups of 32 channels (16 of a head of 16), step
    clamp(ceil(max|x| / 7), 1, 18), code clamp(floor((2 x + step) / (2 step)), -7, 7). Returns (codes, steps)."""
    x = np.asarray(x, dtype=np.int64)
    width = min(32, x.shape[-1])
    g = x.reshape(*x.shape[:-1], x.shape[-1] // width, width)
    step = np.clip(-(-np.abs(g).max(-1, keepdims=True) // 7), 1, 18)
    return np.clip((2 * g + step) // (2 * step), -7, 7), step


def held(x):
    """code x step of round4, in x's shape."""
    codes, step = round4(x)
    return (codes * step).reshape(np.shape(x))


def pack_page(k, v):
    """One head's 68 D bytes of a page from int8 rows k, v (64, D)."""
    D = stored_dim(k.shape[-1])
    NG = D // 32
    out = np.zeros(68 * D, dtype=np.uint8)
    wide = lambda x: np.concatenate([x, np.zeros((PAGE, D - x.shape[-1]), np.int64)], axis=1)       # noqa: E731
    ck, sk = round4(wide(np.asarray(k, np.int64)))
    cv, sv = round4(wide(np.asarray(v, np.int64)))
    for t in range(PAGE):
        for g in range(NG):
            out[32 * D + (t // 4 * NG + g) * 4 + t % 4] = sk[t, g, 0]
            out[66 * D + 64 * g + t] = sv[t, g, 0]
            for q in range(4):
                for i in range(4):
                    lo, hi = ck[t, g, 8 * q + i] & 15, ck[t, g, 8 * q + 4 + i] & 15
                    out[t * (D // 2) + 4 * (q * NG + g) + i] = lo | hi << 4
            for i in range(16):
                out[34 * D + (16 * g + i) * PAGE + t] = (cv[t, g, i] & 15) | (cv[t, g, 16 + i] & 15) << 4
    return out


def unpack_page(block):
    """(k, v) values (64, D) of one head's 68 D bytes."""
    b = np.asarray(block, dtype=np.int64)
    D = b.size // 68
    NG = D // 32
    sign = lambda n: (n ^ 8) - 8                                        # noqa: E731
    k, v = np.zeros((2, PAGE, D), np.int64)
    for c in range(D):
        g, r = divmod(c, 32)
        t = np.arange(PAGE)
        byte = b[t * (D // 2) + 4 * (r // 8 * NG + g) + r % 4]
        k[:, c] = sign(byte >> 4 if r % 8 >= 4 else byte & 15) * b[32 * D + (t // 4 * NG + g) * 4 + t % 4]
        byte = b[34 * D + (16 * g + r % 16) * PAGE + t]
        v[:, c] = sign(byte >> 4 if r >= 16 else byte & 15) * b[66 * D + 64 * g + t]
    return k, v


def visible(j, i, window, sinks):
    return (j <= i) & ((window == 0) | (j > i - window) | (j < sinks))


def attend(q, keys, vals, pos, seen_pages, ms, ss, lut, one, mo, so, window=0, sinks=0):
    """One query row q (D) at position pos over keys, vals (n, D) -> (int8 row as int64, softmax summed to zero).
    seen_pages: truth per 64 tokens, False where the page was given back."""
    half = lambda s: 1 << (s - 1) if s else 0                           # noqa: E731
    j = np.arange(len(keys))
    see = visible(j, pos, window, sinks) & np.asarray(seen_pages, bool)[j // PAGE]
    nothing = np.clip(np.full(len(q), half(so) >> so), -128, 127)
    if not see.any():
        return nothing, False
    x = np.clip((keys[see] @ q * ms + half(ss)) >> ss, -128, 127)
    e = np.maximum(0, np.asarray(lut, np.int64)[x - x.max() + 255])
    S = int(e.sum())
    if S == 0:
        return nothing, True
    p = (e * one + S // 2) // S
    return np.clip((p @ vals[see] * mo + half(so)) >> so, -128, 127), False


class OutOfPages(Exception):
    pass


def fork(table, lens, refs, parent=None, add=None, window=0, sinks=0):
    """(table, lens, refs, [(from, to)]) of the next step; OutOfPages where the pages or slots do not suffice."""
    table, lens = np.asarray(table), np.asarray(lens)
    parent = range(len(table)) if parent is None else parent
    slots = table.shape[1]
    add = [0] * len(parent) if add is None else add
    count = np.array(refs, dtype=np.int64)
    out = np.full((len(parent), slots), -1, dtype=np.int32)
    size = np.zeros(len(parent), dtype=np.int32)
    for p in table[table >= 0]:
        count[p] -= 1
    for i, par in enumerate(parent):
        if par < 0:
            continue
        n = size[i] = lens[par]
        if n + add[i] > slots * PAGE:
            raise OutOfPages
        for j in range(-(-int(n) // PAGE)):
            if window and j * PAGE >= sinks and j * PAGE + PAGE - 1 <= n - window:
                continue
            if table[par, j] >= 0:
                out[i, j] = table[par, j]
                count[out[i, j]] += 1
    free = [int(p) for p in np.nonzero(count == 0)[0]]
    copies = []

    def take():
        if not free:
            raise OutOfPages
        p = free.pop(0)
        count[p] = 1
        return p

    for i, par in enumerate(parent):
        n = int(size[i])
        if par < 0 or add[i] == 0:
            continue
        if n % PAGE and count[out[i, n // PAGE]] > 1:
            old = int(out[i, n // PAGE])
            count[old] -= 1
            out[i, n // PAGE] = take()
            copies.append((old, int(out[i, n // PAGE])))
        for j in range(-(-n // PAGE), -(-(n + add[i]) // PAGE)):
            out[i, j] = take()
        size[i] = n + add[i]
    return out, size, count.astype(np.int32), copies


def compact(table, refs):
    """(table, refs, map, [(from, to)])."""
    refs = np.asarray(refs)
    used = np.nonzero(refs > 0)[0]
    n = len(used)
    holes = [p for p in range(n) if refs[p] <= 0]
    moved = np.full(len(refs), -1, dtype=np.int32)
    moved[used] = used
    moves = list(zip([int(p) for p in used if p >= n], holes))
    for a, b in moves:
        moved[a] = b
    out = np.zeros_like(refs)
    out[moved[used]] = refs[used]
    table = np.asarray(table)
    return np.where(table >= 0, moved[np.maximum(table, 0)], -1).astype(np.int32), out, moved, moves


def log_fixed(v, logs, step):
    v, k = int(v), 0
    while v >= len(logs):
        v, k = v >> 1, k + 1
    return int(logs[v]) + k * step


def beam_select(logits, scores, ended, allowed, groups, beams, keep, eos, lut, logs, step, mult):
    """(scores, parent, token, ended), each (groups, keep), and whether a live row's softmax summed to zero."""
    logits = np.asarray(logits, dtype=np.int64)
    lut = np.maximum(0, np.asarray(lut, dtype=np.int64))
    out = (np.full((groups, keep), NO_SCORE, np.int64), np.full((groups, keep), -1, np.int32),
           np.full((groups, keep), -1, np.int32), np.zeros((groups, keep), np.uint8))
    zero = False
    for g in range(groups):
        found = []
        for row in range(g * beams, (g + 1) * beams):
            score = int(scores[row])
            if score == NO_SCORE:
                continue
            if ended is not None and ended[row]:
                found.append((-score, row, eos))
                continue
            x = logits[row]
            S, one = int(lut[x - x.max() + 255].sum()), int(lut[255])
            if S < 1 or one < 1:
                zero = True
                continue
            norm = log_fixed(S, logs, step) - log_fixed(one, logs, step)
            for v, xv in enumerate(x.tolist()):
                if allowed is None or allowed[v]:
                    found.append((-(score + (xv - int(x.max())) * mult - norm), row, v))
        for n, (s, row, v) in enumerate(sorted(found)[:keep]):
            out[0][g, n], out[1][g, n], out[2][g, n] = -s, row, v
            out[3][g, n] = v == eos or (ended is not None and bool(ended[row]))
    return (*out, zero)
