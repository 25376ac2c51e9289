"""A CPU stand-in for the part of anvil_mi355x.runtime.Device that decode.KVCache calls: buffers on the host, argument checks by the
library's own entry points, tables by the numpy restatement. Test infrastructure only."""
import ctypes as C

import numpy as np

from anvil_mi355x import runtime as rt
from oracle import decode as od


class HostBuffer(rt.DeviceBuffer):
    def __init__(self, dev, nbytes):
        self.dev, self.nbytes = dev, int(nbytes)
        self.mem = np.zeros(self.nbytes + 64, np.uint8)
        self.ptr = -(-self.mem.ctypes.data // 64) * 64
        self.bytes = self.mem[self.ptr - self.mem.ctypes.data:][:self.nbytes]

    def upload(self, arr, offset=0):
        raw = np.ascontiguousarray(arr).view(np.uint8).reshape(-1)
        self.bytes[offset:offset + raw.size] = raw

    def download(self, shape, dtype, offset=0, into=None):
        n = int(np.prod(shape)) * np.dtype(dtype).itemsize
        return self.bytes[offset:offset + n].copy().view(dtype).reshape(shape)

    def free(self):
        pass


def _ints(ptr, n):
    return np.ctypeslib.as_array((C.c_int32 * max(1, n)).from_address(ptr))[:n]


class HostDevice:
    def __init__(self):
        self.pending = None

    def alloc(self, nbytes):
        return HostBuffer(self, nbytes)

    def upload(self, arr):
        b = HostBuffer(self, np.asarray(arr).nbytes)
        b.upload(arr)
        return b

    cache_bytes = rt.Device.cache_bytes

    @property
    def lib(self):
        return rt.library()

    def sync(self):
        e, self.pending = self.pending, None
        if e:
            raise e

    def _checked(self, name, *args):
        """What the entry point says of its arguments: without a context an accepted call ends there."""
        try:
            rt.library().call(name, None, *args)
        except ValueError as e:
            if "null context" not in str(e):
                raise

    @staticmethod
    def _tables(cache):
        n = cache.seqs
        return (_ints(cache.table, n * cache.slots).reshape(n, cache.slots), _ints(cache.lens, n), _ints(cache.refs, cache.pages))

    def cache_fork(self, cache, out, parent=None, add=None, window=0, sinks=0):
        self._checked("anvil_cache_fork", C.byref(cache), C.byref(out), rt._opt(parent), rt._opt(add), window, sinks)
        of = lambda b: None if b is None else b.download((out.seqs,), np.int32)                      # noqa: E731
        table, lens, refs = self._tables(cache)
        try:
            new = od.fork(table, lens, refs, of(parent), of(add), window, sinks)[:3]
        except od.OutOfPages:
            self.pending = MemoryError("a cache has too few free pages or slots for its new tokens")
            new = np.full((out.seqs, out.slots), -1), np.zeros(out.seqs), refs
        for to, x in zip(self._tables(out), new):
            to[...] = x

    def cache_compact(self, cache, out, moved):
        self._checked("anvil_cache_compact", C.byref(cache), C.byref(out), rt._opt(moved))
        table, lens, refs = self._tables(cache)
        new_table, new_refs, mapped, _ = od.compact(table, refs)
        for to, x in zip(self._tables(out), (new_table, lens, new_refs)):
            to[...] = x
        moved.upload(mapped.astype(np.int32))
