"""Operands of the experts' operators on a device: arrays in wider buffers whose every other byte is checked."""
import numpy as np

from anvil_mi355x import runtime as rt

NP = {"i8": np.int8, "i16": np.int16, "i32": np.int32}


class Rows:
    """A 2-D array as rows of a device buffer: `pad` elements between the rows, `off` elements before the first."""

    def __init__(self, dev, a, dtype, pad=0, off=0, seed=0):
        a = np.asarray(a)
        self.rows, self.cols = a.shape
        self.dtype, self.ld, self.off = dtype, self.cols + pad, off
        self.host = np.random.default_rng(seed).integers(-100, 100, off + self.rows * self.ld + 16).astype(NP[dtype])
        self.view(self.host)[...] = a
        self.buf = dev.upload(self.host)
        self.ptr = self.buf.ptr + off * self.host.itemsize

    def view(self, flat):
        return flat[self.off:self.off + self.rows * self.ld].reshape(self.rows, self.ld)[:, :self.cols]

    def expect(self, want, what=""):
        """The buffer holds `want` in the rows and what it held before around them."""
        full = self.host.copy()
        self.view(full)[...] = want
        got = self.buf.download(full.shape, full.dtype)
        np.testing.assert_array_equal(self.view(got), self.view(full), err_msg=what)
        np.testing.assert_array_equal(got, full, err_msg=f"{what}: outside of its rows")

    def get(self):
        return self.view(self.buf.download(self.host.shape, self.host.dtype)).astype(np.int64)


def flat(dev, a, dtype, off=0):
    a = np.asarray(a).reshape(1, -1)
    return Rows(dev, a, dtype, off=off)


def roots(n=1024, scale=1 << 20):
    return np.rint(scale / np.sqrt(np.maximum(0.5, np.arange(n)))).astype(np.int64)


def exp_lut(scale=0.08, bits=20):
    return np.rint(np.exp(np.arange(-255, 1) * scale) * (1 << bits)).astype(np.int64)


def act_lut():
    x = np.arange(-128, 128) / 16
    return np.clip(np.rint(x / (1 + np.exp(-x)) * 16), -128, 127).astype(np.int64)


def device():
    return rt.device(0)
