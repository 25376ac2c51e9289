"""The operators of token-by-token decoding that this backend is measured on, through its public entry points.

Five families, each a dict of plain values:

    attention  queries of the newest tokens of every sequence over a paged cache that holds K and V in 4 bits, causal,
               optionally with a sliding window and a few first tokens that stay visible: one token a sequence
               (decoding) or a chunk of them (a prompt taken in pieces)
    append     int8 K and V rows of new tokens rounded to 4 bits into their pages, and read back as the values they stand for
    fork       page tables of a batch: every row continues a parent's pages (copying a shared last page on write),
               is extended by the pages of its next tokens, and drops what no window sees any more
    compact    the used pages of a pool moved to its lowest ids, tables rewritten
    beams      the best continuations over beams and vocabulary from int8 logits, in fixed-point log probabilities

Everything is an integer, so outputs are compared exactly. The plain forms are torch operations on the same buffers.

A page holds 64 tokens. Of one head, for D channels in groups of 32 (each of a token's groups has a step of its own):
    K codes   64 rows of D / 2 bytes; byte 4 (q D / 32 + g) + i of a row holds channels 32 g + 8 q + i (low four bits) and
              32 g + 8 q + 4 + i (high), q and i in 0..3
    K steps   byte ((t / 4) D / 32 + g) 4 + t % 4 of token t, group g
    V codes   byte (16 g + i) 64 + t: channels 32 g + i (low) and 32 g + 16 + i (high), i in 0..15
    V steps   byte 64 g + t
Codes are signed, in [-7, 7], steps in [1, 18]; a value is code x step.
"""
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

ROOT = Path(__file__).resolve().parents[1]
PAGE = 64
NO_SCORE = -(1 << 63)
LOG_LEN, LOG_BITS = 2048, 16


# ------------------------------------------------------------------------------------------------------ cases

def _attention(seqs, heads, kv_heads, dim, longest, new=1, window=0, sinks=0, one=127, ragged=True):
    return {"family": "attention", "seqs": seqs, "heads": heads, "kv_heads": kv_heads, "dim": dim, "longest": longest,
            "new": new, "window": window, "sinks": sinks, "one": one, "ragged": ragged}


def _append(seqs, heads, dim, longest, new, ragged=True):
    return {"family": "append", "seqs": seqs, "heads": heads, "dim": dim, "longest": longest, "new": new, "ragged": ragged}


def _fork(groups, beams, longest, add, layers, heads, dim, expand=False, window=0, sinks=0):
    return {"family": "fork", "groups": groups, "beams": beams, "longest": longest, "add": add, "layers": layers,
            "heads": heads, "dim": dim, "expand": expand, "window": window, "sinks": sinks}


def _compact(pages, seqs, slots, layers, heads, dim, fill):
    return {"family": "compact", "pages": pages, "seqs": seqs, "slots": slots, "layers": layers, "heads": heads,
            "dim": dim, "fill": fill}


def _beams(groups, beams, vocab, keep, masked=False):
    return {"family": "beams", "groups": groups, "beams": beams, "vocab": vocab, "keep": keep, "masked": masked}


def listed():
    named = [
        # one short sequence of a small model: the latency of a call
        ("attend-one", _attention(1, 4, 4, 32, 128, ragged=False)),
        # the GPT-2-small-shaped block's heads, the benchmark's batch, sequences of every length up to its context
        ("attend-768", _attention(32, 12, 12, 64, 1024)),
        # one long document, shared key heads, probabilities finer than 1 / 127
        ("attend-long", _attention(1, 32, 8, 128, 131072, one=16384, ragged=False)),
        # long conversations that see their last 4096 tokens and the first few
        ("attend-window", _attention(16, 32, 8, 128, 16384, window=4096, sinks=4, one=1024)),
        # a piece of four prompts against what is cached of them, through a window
        ("attend-chunk", _attention(4, 12, 12, 64, 2048, new=512, window=1024, sinks=4)),
        # a full batch of a serving system
        ("attend-batch", _attention(64, 32, 8, 128, 8192, one=4096)),
        # one token of each sequence into the cache; whole prompts of odd lengths
        ("append-step", _append(32, 12, 64, 1024, 1)),
        ("append-prompts", _append(8, 8, 128, 2048, 2048)),
        # a beam search's step over every layer's pages
        ("fork-beams", _fork(16, 4, 1024, 1, 12, 12, 64)),
        # a pool two fifths of which were given back, put together again
        ("compact-pool", _compact(1024, 48, 16, 12, 12, 64, 0.6)),
        # the token model's vocabulary, a small batch; a large odd vocabulary with forbidden tokens
        ("beams-512", _beams(8, 4, 512, 4)),
        ("beams-wide", _beams(64, 8, 100003, 8, masked=True)),
    ]
    return [dict(c, name=n) for n, c in named]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    family = rng.choice(["attention"] * 4 + ["append", "fork", "compact", "beams"])
    if family == "attention":
        while True:
            kv, dim = rng.choice([1, 2, 4, 5, 8, 12, 16]), rng.choice([32, 64, 128])
            heads = kv * rng.choice([1, 1, 2, 3, 4, 7, 8])
            longest = _log(rng, 1, 131072)
            seqs = _log(rng, 1, 64)
            new = 1 if rng.random() < 0.7 else _log(rng, 2, 512)
            if heads <= 64 and seqs * kv * dim * longest <= 1 << 28 and seqs * heads * new * longest <= 1 << 25:
                break
        window, sinks = 0, 0
        if rng.random() < 0.4:
            window, sinks = _log(rng, 1, 8192), rng.choice([0, 1, 4, 64, 100])
        return _attention(seqs, heads, kv, dim, longest, min(new, longest), window, sinks,
                          rng.choice([127, 127, 100, 1024, 16384, 32767]), rng.random() < 0.8)
    if family == "append":
        while True:
            case = _append(_log(rng, 1, 64), rng.choice([1, 2, 4, 8, 12]), rng.choice([32, 64, 128]), _log(rng, 1, 8192),
                           _log(rng, 1, 2048), rng.random() < 0.8)
            if case["seqs"] * case["new"] <= 16384 and case["seqs"] * case["longest"] <= 1 << 17:
                return dict(case, new=min(case["new"], case["longest"]))
    if family == "fork":
        window = rng.choice([0, 0, _log(rng, 16, 2048)])
        return _fork(_log(rng, 1, 32), rng.randint(1, 8), _log(rng, 1, 2048), _log(rng, 1, 300), rng.randint(1, 8),
                     rng.choice([1, 4, 8]), rng.choice([32, 64]), rng.random() < 0.3, window,
                     rng.choice([0, 4, 70]) if window else 0)
    if family == "compact":
        pages = _log(rng, 8, 1500)
        return _compact(pages, _log(rng, 1, 64), _log(rng, 1, 32), rng.randint(1, 8), rng.choice([1, 4, 8]),
                        rng.choice([32, 64]), round(rng.uniform(0.05, 0.95), 3))
    while True:
        case = _beams(_log(rng, 1, 64), rng.randint(1, 16), _log(rng, 2, 131072), rng.randint(1, 32), rng.random() < 0.4)
        if case["groups"] * case["beams"] * case["vocab"] <= 1 << 25:
            return case


# ----------------------------------------------------------------------------------------------------- inputs

def page_bytes(dim):
    """Bytes of one head's block of a page."""
    return 68 * dim


def _offsets(dim):
    return 0, 32 * dim, 34 * dim, 66 * dim


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _pool(layers, pages, heads, dim, gen):
    """A pool of random pages: codes of a normal distribution, steps of 1 to 18."""
    codes = torch.distributions.Normal(0.0, 3.0).icdf((torch.arange(256) + 0.5) / 256).round().clamp(-7, 7).long()
    codes = (codes[torch.randperm(256, generator=torch.Generator().manual_seed(1))] & 15).to(torch.uint8).cuda()
    pool = torch.empty((layers, pages, heads, page_bytes(dim)), dtype=torch.uint8, device="cuda")
    k, ks, v, vs = _offsets(dim)
    for part, lo, hi in ((0, k, ks), (1, ks, v), (0, v, vs), (1, vs, page_bytes(dim))):
        for layer in range(layers):
            shape = (pages, heads, hi - lo)
            if part:
                pool[layer, ..., lo:hi] = torch.randint(1, 19, shape, generator=gen, device="cuda", dtype=torch.uint8)
                continue
            raw = torch.randint(0, 256, shape, generator=gen, device="cuda", dtype=torch.uint8)
            low = codes[raw.int()]
            raw = torch.randint(0, 256, shape, generator=gen, device="cuda", dtype=torch.uint8)
            pool[layer, ..., lo:hi] = low | (codes[raw.int()] << 4)
    return pool


def _i32(v):
    return torch.as_tensor(np.asarray(v, dtype=np.int32)).cuda()


def _exp_table(scale, bits):
    return np.rint(np.exp(np.arange(-255, 1) * scale) * (1 << bits)).astype(np.int64)


def _fixed(ratio, bound):
    """(multiplier, shift) of a ratio: the widest shift at which bound * multiplier + rounding fits 32 bits."""
    s = 31
    while bound * max(1, round(ratio * (1 << s))) + (1 << s >> 1) > (1 << 31) - 1:
        s -= 1
    return max(1, round(ratio * (1 << s))), s


class State:
    """What a program holds: tensors and plain values by name."""

    def __init__(self, **kw):
        self.__dict__.update(kw)


def _lengths(case, rng):
    """Cached tokens of every sequence, the new ones among them, and the new ones of each: a case's own, in an order of
    the seed's."""
    n, most, new, own_rng = case["seqs"], case["longest"], case["new"], random.Random(7)
    both = [(most, min(new, most))]
    for _ in range(n - 1):
        x = own_rng.randint(min(most, max(new, most // 8)), most) if case["ragged"] else most
        both.append((x, own_rng.randint(1, min(new, x)) if case["ragged"] else min(new, x)))
    rng.shuffle(both)
    return [x for x, _ in both], [k for _, k in both]


def _paged(lens, rng, spare):
    """A page table of rows of these lengths over shuffled pages."""
    need = [-(-x // PAGE) for x in lens]
    pages = sum(need) + spare
    order = list(range(pages))
    rng.shuffle(order)
    table = np.full((len(lens), max(need)), -1, dtype=np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, pages


def _rows(seqs, kw):
    """Device tensors of a batch's new rows."""
    starts = np.concatenate([[0], np.cumsum(kw)])
    return None if all(k == 1 for k in kw) else _i32(starts), int(starts[-1])


def _prepare_attention(case, seed):
    rng, gen = random.Random(seed), _gen(seed)
    lens, news = _lengths(case, rng)
    table, pages = _paged(lens, rng, 3)
    H, D = case["heads"], case["dim"]
    starts, rows = _rows(case["seqs"], news)
    q = (torch.randn((rows, H, D), generator=gen, device="cuda") * 40).round().clamp(-128, 127).to(torch.int8)
    span = min(max(lens), case["window"] + case["sinks"]) if case["window"] else max(lens)
    ms, ss = _fixed(30 / (40 * 24 * math.sqrt(D)), 128 * 126 * D)
    mo, so = _fixed(1.5 / case["one"], 126 * (case["one"] + span // 2))
    bits = max(4, min(20, 30 - int(math.log2(case["one"])) - int(math.log2(span))))
    return State(family="attention", pool=_pool(1, pages, case["kv_heads"], D, gen), table=_i32(table), lens=_i32(lens),
                 starts=starts, rows=rows, new=max(news), q=q, out=torch.empty_like(q), ms=ms, ss=ss, mo=mo, so=so,
                 lut=_i32(_exp_table(0.08, bits)), one=case["one"], window=case["window"], sinks=case["sinks"])


def _prepare_append(case, seed):
    rng, gen = random.Random(seed), _gen(seed)
    lens, news = _lengths(case, rng)
    table, pages = _paged(lens, rng, 3)
    H, D = case["heads"], case["dim"]
    starts, rows = _rows(case["seqs"], news)

    def values():
        """Channels of different magnitude, as projections have them."""
        loud = torch.rand((1, H, D), generator=gen, device="cuda") * 45 + 3
        x = torch.randn((rows, H, D), generator=gen, device="cuda") * loud
        return x.round().clamp(-128, 127).to(torch.int8)

    k, v = values(), values()
    return State(family="append", pool=_pool(1, pages, H, D, gen), table=_i32(table), lens=_i32(lens), starts=starts,
                 rows=rows, new=max(news), k=k, v=v, k_out=torch.empty_like(k), v_out=torch.empty_like(v))


def _fork_state(case, seed):
    """The tables of a beam search in progress (or of its prompts): each group's prompt pages are shared by its beams,
    what they wrote since is their own. The lengths are the case's, in an order of the seed's."""
    rng, own_rng = random.Random(seed), random.Random(7)
    groups, beams = case["groups"], 1 if case["expand"] else case["beams"]
    slots = -(-(case["longest"] + case["add"]) // PAGE)
    rows, lens, refs = [], [], {}
    total = 0

    def take():
        nonlocal total
        total += 1
        refs[total - 1] = 1
        return total - 1

    prompts = [(own_rng.randint(max(1, case["longest"] // 4), case["longest"]), own_rng.randint(0, 100))
               for _ in range(groups)]
    rng.shuffle(prompts)
    for n, back in prompts:
        back = min(n - 1, back) if beams > 1 else 0
        shared = [take() for _ in range((n - back) // PAGE)]
        for b in range(beams):
            if b:
                for p in shared:
                    refs[p] += 1
            rows.append(shared + [take() for _ in range(-(-n // PAGE) - len(shared))])
            lens.append(n)
    n_out = groups * case["beams"]
    spare = n_out * (-(-case["add"] // PAGE) + 2)
    order = list(range(total + spare))
    rng.shuffle(order)
    table = np.full((len(rows), slots), -1, dtype=np.int32)
    for i, r in enumerate(rows):
        table[i, :len(r)] = [order[p] for p in r]
    counts = np.zeros(total + spare, dtype=np.int32)
    for p, c in refs.items():
        counts[order[p]] = c
    parent = [i // case["beams"] * beams + (0 if case["expand"] else rng.randrange(beams)) for i in range(n_out)]
    return table, np.asarray(lens, dtype=np.int32), counts, np.asarray(parent, dtype=np.int32)


def _prepare_fork(case, seed):
    table, lens, refs, parent = _fork_state(case, seed)
    n = len(parent)
    return State(family="fork", pool=_pool(case["layers"], len(refs), case["heads"], case["dim"], _gen(seed)),
                 table=_i32(table), lens=_i32(lens), refs=_i32(refs), parent=_i32(parent), add=_i32([case["add"]] * n),
                 window=case["window"], sinks=case["sinks"],
                 table_out=torch.empty((n, table.shape[1]), dtype=torch.int32, device="cuda"),
                 lens_out=torch.empty(n, dtype=torch.int32, device="cuda"), refs_out=torch.empty_like(_i32(refs)))


def _compact_state(case, seed):
    rng = random.Random(seed)
    pages, slots = case["pages"], case["slots"]
    used = max(1, min(int(pages * case["fill"]), case["seqs"] * slots))
    ids = rng.sample(range(pages), used)
    table = np.full((case["seqs"], slots), -1, dtype=np.int32)
    lens = np.zeros(case["seqs"], dtype=np.int32)
    refs = np.zeros(pages, dtype=np.int32)
    for i, p in enumerate(ids):
        row, slot = i % case["seqs"], i // case["seqs"]
        table[row, slot] = p
        lens[row] = slot * PAGE + rng.randint(1, PAGE)
        refs[p] += 1
    return table, lens, refs


def _prepare_compact(case, seed):
    table, lens, refs = _compact_state(case, seed)
    return State(family="compact", pool=_pool(case["layers"], case["pages"], case["heads"], case["dim"], _gen(seed)),
                 table=_i32(table), lens=_i32(lens), refs=_i32(refs), table_out=torch.empty_like(_i32(table)),
                 lens_out=torch.empty_like(_i32(lens)), refs_out=torch.empty_like(_i32(refs)),
                 moved=torch.empty_like(_i32(refs)))


def _prepare_beams(case, seed):
    gen = _gen(seed)
    rows, V, k = case["groups"] * case["beams"], case["vocab"], case["keep"]
    logits = (torch.randn((rows, V), generator=gen, device="cuda") * 24 - 10).round().clamp(-128, 127).to(torch.int8)
    scores = -torch.randint(0, 40 << LOG_BITS, (rows,), generator=gen, device="cuda", dtype=torch.int64)
    scores[torch.rand(rows, generator=gen, device="cuda") < 0.05] = NO_SCORE
    ended = (torch.rand(rows, generator=gen, device="cuda") < 0.1).to(torch.uint8)
    allowed = None
    if case["masked"]:
        allowed = (torch.rand(V, generator=gen, device="cuda") < 0.9).to(torch.uint8)
    scale = 0.09
    logs = np.rint(np.log(np.maximum(1, np.arange(LOG_LEN))) * (1 << LOG_BITS))
    groups = case["groups"]
    return State(family="beams", logits=logits, scores=scores, ended=ended, allowed=allowed, groups=groups,
                 beams=case["beams"], keep=k, eos=V - 1, lut=_i32(_exp_table(scale, 20)), logs=_i32(logs),
                 step=round(math.log(2) * (1 << LOG_BITS)), mult=round(scale * (1 << LOG_BITS)),
                 scores_out=torch.empty((groups, k), dtype=torch.int64, device="cuda"),
                 parent=torch.empty((groups, k), dtype=torch.int32, device="cuda"),
                 token=torch.empty((groups, k), dtype=torch.int32, device="cuda"),
                 ended_out=torch.empty((groups, k), dtype=torch.uint8, device="cuda"))


PREPARE = {"attention": _prepare_attention, "append": _prepare_append, "fork": _prepare_fork,
           "compact": _prepare_compact, "beams": _prepare_beams}


def _framework():
    """The shared context of device 0 and the binding's module."""
    path = str(ROOT / "anvil-compiler_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from anvil_mi355x import runtime
    return runtime


def prepare(case, seed):
    s = PREPARE[case["family"]](case, seed)
    if own:
        rt = _framework()
        s.dev = rt.device(0)
        if s.family != "beams":
            dim = s.pool.shape[-1] // 68
            s.cache = rt.Cache(s.pool.data_ptr(), s.table.data_ptr(), s.lens.data_ptr(),
                               s.refs.data_ptr() if hasattr(s, "refs") else 0, seqs=s.table.shape[0],
                               slots=s.table.shape[1], pages=s.pool.shape[1], heads=s.pool.shape[2], dim=dim,
                               layers=s.pool.shape[0])
            if hasattr(s, "table_out"):
                s.cache_out = s.cache.with_tables(s.table_out.data_ptr(), s.lens_out.data_ptr(), s.refs_out.data_ptr(),
                                                  seqs=s.table_out.shape[0])
        torch.cuda.synchronize()
    return s


# -------------------------------------------------------------------------------------------------- one pass

def _ptr(t):
    return None if t is None else t.data_ptr()


def _own_attention(s):
    H, D = s.q.shape[1:]
    s.dev.attention_cache(s.cache, 0, s.q.data_ptr(), s.out.data_ptr(), _ptr(s.starts), s.rows, s.new, H,
                          (H * D, D, H * D, D), s.ms, s.ss, s.lut.data_ptr(), s.one, s.mo, s.so, s.window, s.sinks)
    return {"out": s.out}


def _own_append(s):
    H, D = s.k.shape[1:]
    strides = (H * D, D, H * D, D)
    s.dev.cache_append(s.cache, 0, s.k.data_ptr(), s.v.data_ptr(), _ptr(s.starts), s.rows, s.new, strides)
    s.dev.cache_read(s.cache, 0, s.k_out.data_ptr(), s.v_out.data_ptr(), _ptr(s.starts), s.rows, s.new, strides)
    return {"k": s.k_out, "v": s.v_out}


def _own_fork(s):
    s.dev.cache_fork(s.cache, s.cache_out, s.parent.data_ptr(), s.add.data_ptr(), s.window, s.sinks)
    return {"table": s.table_out, "lens": s.lens_out, "refs": s.refs_out, "pool": s.pool}


def _own_compact(s):
    s.dev.cache_compact(s.cache, s.cache_out, s.moved.data_ptr())
    return {"table": s.table_out, "lens": s.lens_out, "refs": s.refs_out, "moved": s.moved, "pool": s.pool}


def _own_beams(s):
    s.dev.beam_select(s.logits.data_ptr(), s.logits.shape[1], s.scores.data_ptr(), s.ended.data_ptr(), _ptr(s.allowed),
                      s.groups, s.beams, s.logits.shape[1], s.keep, s.eos, s.lut.data_ptr(), s.logs.data_ptr(),
                      len(s.logs), s.step, s.mult, s.scores_out.data_ptr(), s.parent.data_ptr(), s.token.data_ptr(),
                      s.ended_out.data_ptr())
    return {"scores": s.scores_out, "parent": s.parent, "token": s.token, "ended": s.ended_out}


OWN = {"attention": _own_attention, "append": _own_append, "fork": _own_fork, "compact": _own_compact,
       "beams": _own_beams}


def _signed(b):
    """Signed values of four-bit codes."""
    return ((b & 15) ^ 8) - 8


def _unpack(blocks, dtype=torch.float32):
    """K and V values (..., 64, D) of head blocks (..., 68 D bytes)."""
    lead, D = blocks.shape[:-1], blocks.shape[-1] // 68
    NG = D // 32
    k, ks, v, vs = _offsets(D)
    b = blocks[..., k:ks].to(torch.int8).view(*lead, PAGE, 4, NG, 1, 4)              # token, q, group, i
    codes = _signed(torch.cat([b, b >> 4], dim=-2)).permute(*range(len(lead)), -5, -3, -4, -2, -1)
    steps = blocks[..., ks:v].view(*lead, PAGE // 4, NG, 4).transpose(-1, -2).reshape(*lead, PAGE, NG, 1)
    keys = (codes.reshape(*lead, PAGE, NG, 32).to(dtype) * steps.to(dtype)).view(*lead, PAGE, D)
    b = blocks[..., v:vs].to(torch.int8).view(*lead, NG, 1, 16, PAGE)
    codes = _signed(torch.cat([b, b >> 4], dim=-3)).view(*lead, NG, 32, PAGE)
    steps = blocks[..., vs:].view(*lead, NG, 1, PAGE)
    return keys, (codes.to(dtype) * steps.to(dtype)).view(*lead, D, PAGE).transpose(-1, -2)


def _positions(s):
    """(sequence, position) of every new row."""
    dev = s.lens.device
    if s.starts is None:
        return torch.arange(s.rows, device=dev), s.lens.long() - 1
    n = (s.starts[1:] - s.starts[:-1]).long()
    seq = torch.repeat_interleave(torch.arange(len(n), device=dev), n, output_size=s.rows)
    return seq, s.lens.long()[seq] - s.starts[1:].long()[seq] + torch.arange(s.rows, device=dev)


def _plain_attention(s):
    rows, H, D = s.q.shape
    n, P = s.table.shape
    Hkv = s.pool.shape[2]
    G = H // Hkv
    seq, pos = _positions(s)
    row = torch.arange(rows, device=s.q.device)
    first = row if s.starts is None else s.starts.long()[seq]
    keys, vals = _unpack(s.pool[0, s.table.clamp(min=0).long()])                    # n, P, Hkv, 64, D
    keys = keys.transpose(1, 2).reshape(n, Hkv, P * PAGE, D)
    vals = vals.transpose(1, 2).reshape(n, Hkv, P * PAGE, D)
    q = torch.zeros((n, s.new, H, D), device=s.q.device)                            # queries of a sequence, padded
    q[seq, row - first] = s.q.float()
    at = torch.full((n, s.new), -1, dtype=torch.int64, device=s.q.device)
    at[seq, row - first] = pos
    q = q.view(n, s.new, Hkv, G, D).transpose(1, 2).reshape(n, Hkv, s.new * G, D)
    acc = (q @ keys.transpose(-1, -2).contiguous()).long()                          # sums below 2^24: exact
    x = ((acc * s.ms + (1 << s.ss >> 1)) >> s.ss).clamp(-128, 127).view(n, Hkv, s.new, G, P * PAGE)
    del acc
    j, i = torch.arange(P * PAGE, device=s.q.device), at[:, None, :, None, None]
    seen = j <= i
    if s.window:
        seen = seen & ((j > i - s.window) | (j < s.sinks))
    top = torch.where(seen, x, -128).amax(-1, keepdim=True)
    e = torch.where(seen, s.lut.long()[(x - top + 255).clamp(max=255)], 0)
    del x
    total = e.sum(-1, keepdim=True)
    p = (e * s.one + total // 2) // total.clamp(min=1)
    del e
    o = (p.double().view(n, Hkv, s.new * G, P * PAGE) @ vals.double()).long()
    o = ((o * s.mo + (1 << s.so >> 1)) >> s.so).clamp(-128, 127)
    o = o.view(n, Hkv, s.new, G, D).transpose(1, 2).reshape(n, s.new, H, D)
    return {"out": o[seq, row - first].to(torch.int8)}


def _round4(x):
    """Codes and steps of int8 rows (rows, H, D): (rows, H, D / 32, 32) and (rows, H, D / 32, 1)."""
    x = x.int().view(*x.shape[:-1], -1, 32)
    step = ((x.abs().amax(-1, keepdim=True) + 6) // 7).clamp(1, 18)
    return torch.div(2 * x + step, 2 * step, rounding_mode="floor").clamp(-7, 7), step


def _plain_append(s):
    rows, H, D = s.k.shape
    NG = D // 32
    seq, pos = _positions(s)
    page, t = s.table.long()[seq, pos // PAGE], pos % PAGE
    ok, oks, ov, ovs = _offsets(D)
    dev = s.k.device
    codes, steps = _round4(s.k)
    codes = (codes & 15).view(rows, H, NG, 4, 2, 4)
    b = (codes[..., 0, :] | codes[..., 1, :] << 4).permute(0, 1, 3, 2, 4).reshape(rows, H, D // 2)
    blocks = s.pool[0]
    head = torch.arange(H, device=dev)[None, :, None]
    page, t = page[:, None, None], t[:, None, None]
    g = torch.arange(NG, device=dev)
    blocks[page, head, ok + t * (D // 2) + torch.arange(D // 2, device=dev)] = b.to(torch.uint8)
    blocks[page, head, oks + (t // 4 * NG + g) * 4 + t % 4] = steps[..., 0].to(torch.uint8)
    codes, steps = _round4(s.v)
    codes = (codes & 15).view(rows, H, NG, 2, 16)
    b = (codes[..., 0, :] | codes[..., 1, :] << 4).reshape(rows, H, D // 2)
    blocks[page, head, ov + torch.arange(D // 2, device=dev) * PAGE + t] = b.to(torch.uint8)
    blocks[page, head, ovs + g * PAGE + t] = steps[..., 0].to(torch.uint8)
    # and back: the rows' bytes of the pages
    b = blocks[page, head, ok + t * (D // 2) + torch.arange(D // 2, device=dev)].to(torch.int8).view(rows, H, 4, NG, 1, 4)
    codes = _signed(torch.cat([b, b >> 4], dim=-2)).permute(0, 1, 3, 2, 4, 5).reshape(rows, H, NG, 32)
    k = codes.int() * blocks[page, head, oks + (t // 4 * NG + g) * 4 + t % 4].int()[..., None]
    b = blocks[page, head, ov + torch.arange(D // 2, device=dev) * PAGE + t].to(torch.int8).view(rows, H, NG, 1, 16)
    codes = _signed(torch.cat([b, b >> 4], dim=-2)).reshape(rows, H, NG, 32)
    v = codes.int() * blocks[page, head, ovs + g * PAGE + t].int()[..., None]
    return {"k": k.view(rows, H, D).to(torch.int8), "v": v.view(rows, H, D).to(torch.int8)}


def _plain_fork(s):
    dev, P, pages = s.table.device, s.table.shape[1], s.pool.shape[1]
    have = s.parent >= 0
    par = s.parent.clamp(min=0).long()
    len0 = torch.where(have, s.lens.long()[par], 0)
    add = torch.where(have, s.add.long(), 0)
    slot = torch.arange(P, device=dev)
    used = (len0 + PAGE - 1) // PAGE
    kept = slot < used[:, None]
    if s.window:
        kept &= ~((slot * PAGE >= s.sinks) & (slot * PAGE + PAGE - 1 <= len0[:, None] - s.window))
    table = torch.where(kept, s.table.long()[par], -1)
    count = torch.zeros(pages + 1, dtype=torch.int64, device=dev)
    count[:pages] = s.refs
    old = s.table.long().reshape(-1)
    count.index_add_(0, torch.where(old >= 0, old, pages), torch.full_like(old, -1))
    now = table.reshape(-1)
    count.index_add_(0, torch.where(now >= 0, now, pages), torch.ones_like(now))
    # of the rows that write into a shared last page all but the last sharer copy it
    part = (add > 0) & (len0 % PAGE != 0)
    last = torch.where(part, table.gather(1, (len0 // PAGE).clamp(max=P - 1)[:, None])[:, 0], pages)
    earlier = torch.tril(last[:, None] == last[None, :], -1).sum(1)
    copies = part & (count[last] - earlier > 1)
    # new pages, lowest free ids first, in the order of the rows and their slots
    want = (slot >= used[:, None]) & (slot < (len0 + add + PAGE - 1)[:, None] // PAGE)
    want |= copies[:, None] & (slot == (len0 // PAGE)[:, None])
    free = torch.sort((count[:pages] > 0).to(torch.int8), stable=True).indices
    flat = want.reshape(-1)
    new = free[(flat.cumsum(0) - 1).clamp(0, pages - 1)].view_as(want)
    table_out = torch.where(want, new, table)
    count.index_add_(0, torch.where(copies, last, pages), torch.full_like(last, -1))
    count.index_add_(0, torch.where(want, new, pages).reshape(-1), torch.ones_like(now))
    at = copies.nonzero()[:, 0]
    s.pool[:, table_out[at, (len0 // PAGE)[at]]] = s.pool[:, last[at]]
    return {"table": table_out.int(), "lens": (len0 + add).int(), "refs": count[:pages].int(), "pool": s.pool}


def _plain_compact(s):
    used = s.refs > 0
    n = used.sum()
    ids = torch.arange(len(used), device=used.device)
    src = (used & (ids >= n)).nonzero()[:, 0]
    dst = (~used & (ids < n)).nonzero()[:, 0]
    moved = torch.where(used, ids, -1)
    moved[src] = dst
    s.pool[:, dst] = s.pool[:, src]
    table = torch.where(s.table >= 0, moved[s.table.clamp(min=0).long()], -1)
    refs = torch.zeros_like(s.refs)
    refs.index_add_(0, moved.clamp(min=0), torch.where(used, s.refs, 0))
    return {"table": table.int(), "lens": s.lens.clone(), "refs": refs, "moved": moved.int(), "pool": s.pool}


def _log_fixed(s, v):
    """Fixed-point logarithm of positive whole numbers: halved until they index the table."""
    bits = torch.frexp(v.double()).exponent.long()                   # 2^(bits-1) <= v < 2^bits
    k = (bits - (LOG_LEN.bit_length() - 1)).clamp(min=0)
    return s.logs.long()[v >> k] + k * s.step


def _plain_beams(s):
    rows, V = s.logits.shape
    x = s.logits.int()
    top = x.amax(1, keepdim=True)
    total = s.lut[x - top + 255].sum(1, dtype=torch.int64)
    norm = _log_fixed(s, total) - _log_fixed(s, s.lut[255:].long())
    base = s.scores - top[:, 0].long() * s.mult - norm
    cand = base[:, None] + x.long() * s.mult
    out = torch.zeros((rows, V), dtype=torch.bool, device=x.device)
    if s.allowed is not None:
        out |= s.allowed == 0
    ended = s.ended.bool()
    out[ended] = True
    cand = torch.where(out, NO_SCORE, cand)
    cand[:, s.eos] = torch.where(ended, s.scores, cand[:, s.eos])
    cand[s.scores == NO_SCORE] = NO_SCORE
    flat = cand.view(s.groups, s.beams * V)
    size = s.beams * V
    order = torch.arange(size - 1, -1, -1, device=x.device)
    key = torch.where(flat == NO_SCORE, NO_SCORE, flat * size + order)               # no two alike
    got = key.topk(min(s.keep, size), dim=1).values
    if got.shape[1] < s.keep:
        got = torch.nn.functional.pad(got, (0, s.keep - got.shape[1]), value=NO_SCORE)
    none = got == NO_SCORE
    at = size - 1 - got % size
    row = torch.arange(s.groups, device=x.device)[:, None] * s.beams + at // V
    token = torch.where(none, -1, at % V)
    done = torch.where(none, 0, ended[row.clamp(max=rows - 1)] | (token == s.eos)).to(torch.uint8)
    return {"scores": torch.where(none, NO_SCORE, torch.div(got, size, rounding_mode="floor")),
            "parent": torch.where(none, -1, row).int(), "token": token.int(), "ended": done}


PLAIN = {"attention": _plain_attention, "append": _plain_append, "fork": _plain_fork, "compact": _plain_compact,
         "beams": _plain_beams}


def run(state):
    return (OWN if own else PLAIN)[state.family](state)


# ------------------------------------------------------------------------------------------- what it must do

def work(case):
    """Each input read once, each result written once: of a cache the keys that some query sees, of a pool the pages that
    are copied or moved (read and written)."""
    f = case["family"]
    if f == "attention":
        lens, news = _lengths(case, random.Random(0))
        D, H, Hkv = case["dim"], case["heads"], case["kv_heads"]
        keys = pairs = 0
        for n, new in zip(lens, news):
            w, first = case["window"] or n, n - new
            low = max(0, first - w + 1)
            keys += n - low + min(low, case["sinks"] if case["window"] else 0)
            for i in (range(first, n) if new <= 64 else range(first, n, 16)):
                lo = max(0, i - w + 1)
                pairs += (i + 1 - lo + min(lo, case["sinks"] if case["window"] else 0)) * (1 if new <= 64 else 16)
        return {"bytes": keys * Hkv * page_bytes(D) / PAGE + 2 * sum(news) * H * D, "flops": 4 * pairs * H * D}
    if f == "append":
        n = sum(_lengths(case, random.Random(0))[1]) * case["heads"] * case["dim"]
        return {"bytes": n * 2 * (2 + 68 / 64), "flops": n * 2 * 6}
    if f == "fork":
        table, lens, refs, parent = _fork_state(case, 0)
        out = _fork_exact(table, lens, refs, parent, [case["add"]] * len(parent), case["window"], case["sinks"])
        page = case["layers"] * case["heads"] * page_bytes(case["dim"])
        return {"bytes": 4 * (table.size + out[0].size + 2 * refs.size + 4 * len(parent)) + 2 * page * len(out[3]),
                "flops": 4 * table.size}
    if f == "compact":
        table, _, refs = _compact_state(case, 0)
        n = int((refs > 0).sum())
        page = case["layers"] * case["heads"] * page_bytes(case["dim"])
        return {"bytes": 4 * (2 * table.size + 3 * refs.size) + 2 * page * int((refs[n:] > 0).sum()),
                "flops": 4 * refs.size}
    rows = case["groups"] * case["beams"]
    return {"bytes": rows * (case["vocab"] + 9) + case["vocab"] * case["masked"] + case["groups"] * case["keep"] * 17,
            "flops": 4 * rows * case["vocab"]}


# ------------------------------------------------------------------------------------------ the same in 64 bits

def _exact_attention(s):
    rows, H, D = s.q.shape
    n, P = s.table.shape
    Hkv = s.pool.shape[2]
    lens = s.lens.tolist()
    starts = list(range(n + 1)) if s.starts is None else s.starts.tolist()
    out = torch.zeros((rows, H, D), dtype=torch.int8, device=s.q.device)
    lut = s.lut.long()
    for i in range(n):
        lo, hi = starts[i], starts[i + 1]
        used = -(-lens[i] // PAGE)
        blocks = s.pool[0, s.table[i, :used].long()].long().movedim(2, 0).contiguous()             # 68 D, used, Hkv
        flat = blocks.view(68 * D, used * Hkv)
        keys, vals = [], []
        NG = D // 32
        t = torch.arange(PAGE, device=s.q.device)
        for c in range(D):
            g, r = c // 32, c % 32
            b = flat[t * (D // 2) + 4 * (r // 8 * NG + g) + r % 4]
            b = b // 16 if r % 8 >= 4 else b % 16
            keys.append(((b - 16 * (b > 7)) * flat[32 * D + (t // 4 * NG + g) * 4 + t % 4]).double())
            b = flat[34 * D + (16 * g + r % 16) * PAGE + t]
            b = b // 16 if r >= 16 else b % 16
            vals.append(((b - 16 * (b > 7)) * flat[66 * D + g * PAGE + t]).double())
        del blocks, flat
        keys = torch.stack(keys).view(D, PAGE, used, Hkv).permute(3, 0, 2, 1).reshape(Hkv, D, used * PAGE)
        vals = torch.stack(vals).view(D, PAGE, used, Hkv).permute(3, 2, 1, 0).reshape(Hkv, used * PAGE, D)
        at = torch.arange(lens[i] - (hi - lo), lens[i], device=s.q.device)[:, None]
        j = torch.arange(used * PAGE, device=s.q.device)[None, :]
        hidden = j > at
        if s.window:
            hidden |= (j <= at - s.window) & (j >= s.sinks)
        for h in range(H):
            kv = h // (H // Hkv)
            x = torch.floor((s.q[lo:hi, h].double() @ keys[kv] * s.ms + (0.5 * (1 << s.ss) if s.ss else 0)) / (1 << s.ss))
            x = x.clamp(-128, 127).long()
            x[hidden] = -1000
            top = x.max(1, keepdim=True).values
            e = torch.where(hidden, 0, lut[(x - top + 255).clamp(0, 255)])
            total = e.sum(1, keepdim=True)
            p = torch.div(e * s.one + torch.div(total, 2, rounding_mode="floor"), total, rounding_mode="floor")
            acc = (p.double() @ vals[kv]).long()
            out[lo:hi, h] = torch.div(acc * s.mo + (1 << s.so) // 2, 1 << s.so, rounding_mode="floor").clamp(-128, 127)
    return {"out": out}


def _exact_append(s):
    got = {}
    for name, x in (("k", s.k), ("v", s.v)):
        rows, H, D = x.shape
        x = x.double().view(rows, H, D // 32, 32)
        a = x.abs().max(-1, keepdim=True).values
        step = torch.ceil(a / 7).clamp(1, 18)
        code = torch.floor((2 * x + step).long().double() / (2 * step)).clamp(-7, 7)
        got[name] = (code * step).view(rows, H, D).to(torch.int8)
    return got


def _fork_exact(table, lens, refs, parent, add, window, sinks):
    """Row by row: (table, lens, refs, [(from, to)] page copies)."""
    slots = table.shape[1]
    count = refs.astype(np.int64).copy()
    out = np.full((len(parent), slots), -1, dtype=np.int32)
    size = np.zeros(len(parent), dtype=np.int32)
    for p in table[table >= 0]:
        count[p] -= 1
    for i, par in enumerate(parent):
        if par < 0:
            continue
        size[i] = lens[par]
        for j in range(-(-int(lens[par]) // PAGE)):
            gone = window and j * PAGE >= sinks and j * PAGE + PAGE - 1 <= lens[par] - window
            if not gone and table[par, j] >= 0:
                out[i, j] = table[par, j]
                count[out[i, j]] += 1
    free = iter(np.nonzero(count == 0)[0])
    copies = []
    for i, par in enumerate(parent):
        n = int(size[i])
        if par < 0 or add[i] == 0:
            continue
        if n % PAGE and count[out[i, n // PAGE]] > 1:
            old, new = out[i, n // PAGE], next(free)
            count[old] -= 1
            count[new] = 1
            out[i, n // PAGE] = new
            copies.append((int(old), int(new)))
        for j in range(-(-n // PAGE), -(-(n + add[i]) // PAGE)):
            out[i, j] = next(free)
            count[out[i, j]] = 1
        size[i] = n + add[i]
    return out, size, count.astype(np.int32), copies


def _exact_fork(s):
    host = lambda t: t.cpu().numpy()                                                                # noqa: E731
    table, lens, refs, copies = _fork_exact(host(s.table), host(s.lens), host(s.refs), host(s.parent).tolist(),
                                            host(s.add).tolist(), s.window, s.sinks)
    pool = s.pool.clone()
    for a, b in copies:
        pool[:, b] = s.pool[:, a]
    return {"table": _i32(table), "lens": _i32(lens), "refs": _i32(refs), "pool": pool}


def _exact_compact(s):
    refs, table = s.refs.cpu().numpy(), s.table.cpu().numpy()
    used = [p for p in range(len(refs)) if refs[p]]
    holes = [p for p in range(len(used)) if not refs[p]]
    moved = np.full(len(refs), -1, dtype=np.int32)
    new_refs = np.zeros_like(refs)
    pool = s.pool.clone()
    for p in used:
        to = p if p < len(used) else holes.pop(0)
        moved[p] = to
        new_refs[to] = refs[p]
        if to != p:
            pool[:, to] = s.pool[:, p]
    new_table = np.array([[moved[p] if p >= 0 else -1 for p in row] for row in table], dtype=np.int32)
    return {"table": _i32(new_table), "lens": s.lens.clone(), "refs": _i32(new_refs), "moved": _i32(moved), "pool": pool}


def _exact_beams(s):
    rows, V = s.logits.shape
    lut, logs = s.lut.tolist(), s.logs.tolist()

    def log(v):
        k = 0
        while v >> k >= len(logs):
            k += 1
        return logs[v >> k] + k * s.step

    best, host = [], {"scores": s.scores.tolist(), "ended": s.ended.tolist()}
    allowed = torch.ones(V, dtype=torch.bool, device=s.logits.device) if s.allowed is None else s.allowed != 0
    legal = allowed.nonzero()[:, 0]
    for g in range(s.groups):
        found = []
        for r in range(g * s.beams, (g + 1) * s.beams):
            if host["scores"][r] == NO_SCORE:
                continue
            if host["ended"][r]:
                found.append((-host["scores"][r], r, s.eos))
                continue
            seen = torch.bincount(s.logits[r].long() + 128, minlength=256).tolist()
            top = max(v for v in range(256) if seen[v])
            total = sum(c * lut[v - top + 255] for v, c in enumerate(seen) if c)
            norm = log(total) - log(lut[255])
            x = s.logits[r][legal]
            pick = torch.sort(x.long(), descending=True, stable=True).indices[:s.keep]
            for v, t in zip(x[pick].tolist(), legal[pick].tolist()):
                found.append((-(host["scores"][r] + (v + 128 - top) * s.mult - norm), r, t))
        found = sorted(found)[:s.keep]
        best.append(found + [None] * (s.keep - len(found)))
    dev = s.logits.device

    def get(f, none, dtype):
        return torch.tensor([[none if b is None else f(b) for b in row] for row in best], dtype=dtype, device=dev)

    return {"scores": get(lambda b: -b[0], NO_SCORE, torch.int64), "parent": get(lambda b: b[1], -1, torch.int32),
            "token": get(lambda b: b[2], -1, torch.int32),
            "ended": get(lambda b: int(host["ended"][b[1]] or b[2] == s.eos), 0, torch.uint8)}


EXACT = {"attention": _exact_attention, "append": _exact_append, "fork": _exact_fork, "compact": _exact_compact,
         "beams": _exact_beams}


def exact(case, seed):
    return EXACT[case["family"]](PREPARE[case["family"]](case, seed))
