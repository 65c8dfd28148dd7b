"""The 8-bit operators in float64, and helpers to call the library on arrays."""
import numpy as np

from shim import q8_shim as Q

TYPES = {"f32": Q.F32, "f16": Q.F16, "bf16": Q.BF16}
# half a unit in the last place, relative
UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
# spacing of the smallest values, halved
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}
LEAST_SCALE = 2.0 ** -126


def stored(a, dtype):
    """`a` rounded to the type, as float64."""
    a = np.asarray(a, dtype=np.float32)
    if dtype == "f16":
        a = a.astype(np.float16)
    elif dtype == "bf16":
        a = Q.from_bf16(Q.to_bf16(a))
    return a.astype(np.float64)


def random_q(rng, rows, cols, lo=-127):
    return np.clip(np.rint(rng.normal(0, 35, (rows, cols))), lo, 127).astype(np.int8)


class Window:
    """A matrix inside a larger device buffer, `shift` values from its start, surrounded by a pattern."""

    def __init__(self, rows, cols, kind, pad=0, shift=0, values=None):
        self.rows, self.cols, self.kind, self.shift = rows, cols, kind, shift
        self.ld = cols + pad
        self.count = shift + max(rows, 1) * self.ld + 64
        host = np.full((1, self.count), 85, dtype=np.float32 if kind != "int8" else np.int8)
        if values is not None and values.size:
            at = shift + np.arange(rows)[:, None] * self.ld + np.arange(cols)[None, :]
            host[0, at.ravel()] = np.asarray(values, dtype=host.dtype).ravel()
        self.array = Q.Array.of(host, kind)
        self.start = self.array.numpy()[0].copy()
        self.ptr = self.array.ptr + shift * self.array.size

    def _places(self):
        return self.shift + np.arange(self.rows)[:, None] * self.ld + np.arange(self.cols)[None, :]

    def values(self):
        """The matrix; what lies around it must be as it was."""
        now = self.array.numpy()[0]
        outside = np.ones(self.count, dtype=bool)
        if self.rows and self.cols:
            outside[self._places().ravel()] = False
        assert np.array_equal(now[outside], self.start[outside], equal_nan=True), "written outside the matrix"
        if not self.rows or not self.cols:
            return np.zeros((self.rows, self.cols))
        return now[self._places()].astype(np.float64)


def norm(hidden, gain, eps):
    """n and rstd of rows of `hidden`, in float64."""
    rstd = 1.0 / np.sqrt((hidden ** 2).mean(axis=1) + eps)
    return hidden * rstd[:, None] * gain, rstd


def scales(n):
    return np.maximum(np.abs(n).max(axis=1) / 127.0, LEAST_SCALE)


def norm_backward(dn, hidden, gain, rstd, dres):
    u, xhat = dn * gain, hidden * rstd[:, None]
    dx = rstd[:, None] * (u - xhat * (u * xhat).mean(axis=1, keepdims=True))
    return dx + (0 if dres is None else dres), (dn * xhat).sum(axis=0)
