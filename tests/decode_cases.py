"""Caches of random sequences for the tests of the decoding operators: K and V rows, page tables over shuffled pages, and
the same on a device."""
import numpy as np

from anvil_mi355x import runtime as rt
from oracle import decode as od

PAGE = od.PAGE


def exp_lut(scale=0.05, bits=16):
    return np.rint(np.exp(np.arange(-255, 1) * scale) * (1 << bits)).astype(np.int64)


def fixed(ratio, bound):
    s = 31
    while bound * max(1, round(ratio * (1 << s))) + (1 << s >> 1) > (1 << 31) - 1:
        s -= 1
    return max(1, round(ratio * (1 << s))), s


class Sequences:
    """A batch of sequences of `lens` tokens, each token's K and V (heads, dim) int8, in `layers` layers."""

    def __init__(self, lens, heads, dim, seed=0, spare=3, layers=1, extra_slots=0, loud=None):
        rng = np.random.default_rng([seed, dim, heads, len(lens)])
        self.lens, self.heads, self.dim, self.layers = list(lens), heads, dim, layers
        need = [-(-n // PAGE) for n in lens]
        self.slots = max([1, *need]) + extra_slots
        self.pages = max(1, sum(need) + spare)
        order = rng.permutation(self.pages)
        self.table = np.full((len(lens), self.slots), -1, np.int32)
        self.refs = np.zeros(self.pages, np.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            self.refs[order[at:at + n]] = 1
            at += n
        amp = rng.uniform(2, 60, (heads, dim)) if loud is None else np.full((heads, dim), loud)
        draw = lambda n: np.clip(np.rint(rng.normal(0, 1, (n, heads, dim)) * amp), -128, 127).astype(np.int64)  # noqa: E731
        self.k = [[draw(n) for n in lens] for _ in range(layers)]
        self.v = [[draw(n) for n in lens] for _ in range(layers)]

    @property
    def page_bytes(self):
        return self.heads * 68 * od.stored_dim(self.dim)

    def pool(self, fill=None):
        """The pool that holds every sequence whole (bytes of no token as `fill` draws them)."""
        shape = (self.layers, self.pages, self.heads, 68 * od.stored_dim(self.dim))
        pool = np.zeros(shape, np.uint8) if fill is None else fill.integers(0, 256, shape).astype(np.uint8)
        for layer in range(self.layers):
            for i, n in enumerate(self.lens):
                for j in range(-(-n // PAGE)):
                    if self.table[i, j] < 0:
                        continue
                    for h in range(self.heads):
                        part = slice(j * PAGE, min(n, (j + 1) * PAGE))
                        k, v = (np.zeros((PAGE, self.dim), np.int64) for _ in range(2))
                        k[:part.stop - part.start] = self.k[layer][i][part, h]
                        v[:part.stop - part.start] = self.v[layer][i][part, h]
                        self.merge(pool[layer, self.table[i, j], h], od.pack_page(k, v), 0, part.stop - part.start)
        return pool

    def merge(self, into, page, t0, t1):
        """The bytes of tokens t0 .. t1 - 1 of one head's page into another's."""
        D = od.stored_dim(self.dim)
        NG = D // 32
        for t in range(t0, t1):
            into[t * (D // 2):(t + 1) * (D // 2)] = page[t * (D // 2):(t + 1) * (D // 2)]
            at = 32 * D + t // 4 * NG * 4 + np.arange(NG) * 4 + t % 4
            into[at] = page[at]
        v = into[34 * D:66 * D].reshape(D // 2, PAGE)
        v[:, t0:t1] = page[34 * D:66 * D].reshape(D // 2, PAGE)[:, t0:t1]
        v = into[66 * D:].reshape(NG, PAGE)
        v[:, t0:t1] = page[66 * D:].reshape(NG, PAGE)[:, t0:t1]


class OnDevice:
    """A Sequences' tables and a pool on a device, as an rt.Cache."""

    def __init__(self, dev, seqs, pool, table=None, lens=None, refs=None):
        self.dev, self.seqs = dev, seqs
        up = lambda a: dev.upload(np.ascontiguousarray(a, dtype=np.int32))                          # noqa: E731
        self.table = up(seqs.table if table is None else table)
        self.lens = up(seqs.lens if lens is None else lens)
        self.refs = up(seqs.refs if refs is None else refs)
        self.pool = pool if isinstance(pool, rt.DeviceBuffer) else dev.upload(pool)
        n = len(seqs.lens if lens is None else lens)
        self.cache = rt.Cache(self.pool, self.table, self.lens, self.refs, seqs=n, slots=seqs.slots, pages=seqs.pages,
                              heads=seqs.heads, dim=seqs.dim, layers=seqs.layers)
        self.n = n

    def successor(self, n=None):
        """An empty set of tables over the same pool, filled with a pattern that no step leaves."""
        n = self.n if n is None else n
        s = self.seqs
        return OnDevice(self.dev, s, self.pool, np.full((n, s.slots), 0x5A5A5A5A), np.full(n, 0x5A5A5A5A),
                        np.full(s.pages, 0x5A5A5A5A))

    def tables(self):
        s = self.seqs
        return (self.table.download((self.n, s.slots), np.int32), self.lens.download((self.n,), np.int32),
                self.refs.download((s.pages,), np.int32))

    def read_pool(self):
        s = self.seqs
        return self.pool.download((s.layers, s.pages, s.heads, 68 * od.stored_dim(s.dim)), np.uint8)


def starts_of(news):
    return np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
