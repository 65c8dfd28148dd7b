"""ctypes binding of the 8-bit operators in libsgemm_shim.so (include/q8_shim.h).

``Ops`` is one handle: a stream and a workspace.  Its methods take device
memory as objects with a ``ptr`` (``Array`` here, ``DeviceBuffer`` of
sgemm_shim, or anything else that has one), ``None`` where an argument may be
left out, and enqueue their work.  A refused call raises ``SgemmError`` with the
library's message.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import numpy as np

from . import sgemm_shim as S

F32, F16, BF16 = 0, 1, 2
CALL_RMSNORM_BACKWARD, CALL_GEMM, CALL_GRAD_INPUT, CALL_GRAD_WEIGHT = 0, 1, 2, 3
MAX_K = 131071
MAX_SUM, MAX_SUM_F32 = 2097152, 699048    # longest sums of the gradients, with 16-bit types and with F32

_int, _u32, _f32, _vp, _size = ctypes.c_int, ctypes.c_uint32, ctypes.c_float, ctypes.c_void_p, ctypes.c_size_t

# every symbol the header declares, with (restype, argtypes)
SIGNATURES = {
    "q8_open": (_int, [ctypes.POINTER(_vp)]),
    "q8_close": (None, [_vp]),
    "q8_set_stream": (_int, [_vp, _vp]),
    "q8_synchronize": (_int, [_vp]),
    "q8_reserve": (_int, [_vp, _size]),
    "q8_workspace_size": (_int, [_int, _int, _u32, _u32, _u32, ctypes.POINTER(_size)]),
    "q8_quantize": (_int, [_vp, _int, _vp, _u32, _vp, _u32, _vp, _u32, _u32]),
    "q8_dequantize": (_int, [_vp, _int, _vp, _u32, _vp, _vp, _u32, _u32, _u32]),
    "q8_rmsnorm": (_int, [_vp, _int, _vp, _u32, _vp, _u32, _vp, _vp, _u32, _vp, _u32, _vp, _vp, _u32, _u32, _f32]),
    "q8_rmsnorm_backward": (_int, [_vp, _int, _vp, _u32, _vp, _u32, _vp, _vp, _vp, _u32, _vp, _u32, _vp, _u32, _u32]),
    "q8_gemm": (_int, [_vp, _int, _vp, _u32, _vp, _vp, _u32, _vp, _vp, _vp, _u32, _u32, _u32, _u32]),
    "q8_grad_input": (_int, [_vp, _int, _vp, _u32, _vp, _u32, _vp, _vp, _u32, _u32, _u32, _u32]),
    "q8_grad_weight": (_int, [_vp, _int, _vp, _u32, _vp, _u32, _vp, _int, _vp, _u32, _u32, _u32, _u32, _int]),
}

_lib: Optional[ctypes.CDLL] = None


def load_library() -> ctypes.CDLL:
    """The shim with the 8-bit operators' signatures set."""
    global _lib
    if _lib is None:
        lib = S.load_library()
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


def to_bf16(a: np.ndarray) -> np.ndarray:
    """float32 values rounded to bfloat16 (nearest, ties to even), as their 16 bits."""
    u = np.ascontiguousarray(a, dtype=np.float32).view(np.uint32)
    r = ((u + (0x7FFF + ((u >> 16) & 1))) >> 16).astype(np.uint16)
    return np.where((u & 0x7FFFFFFF) > 0x7F800000, ((u >> 16) | 0x40).astype(np.uint16), r)


def from_bf16(a: np.ndarray) -> np.ndarray:
    return (a.astype(np.uint32) << 16).view(np.float32)


class Array(S.DeviceBuffer):
    """A row-major device array.  `kind` is F32, F16, BF16 or "int8"; rows lie `ld` values apart."""

    def __init__(self, rows: int, cols: int, kind, ld: Optional[int] = None):
        self.rows, self.cols, self.kind = int(rows), int(cols), kind
        self.ld = self.cols if ld is None else int(ld)
        if self.ld < self.cols:
            raise ValueError(f"rows of {self.cols} values do not fit a leading dimension of {self.ld}")
        self.size = {F32: 4, F16: 2, BF16: 2, "int8": 1}[kind]
        super().__init__(max(1, self.rows * self.ld * self.size))

    @classmethod
    def of(cls, a: np.ndarray, kind=None, ld: Optional[int] = None) -> "Array":
        """`a` (1-D: one row) on the device, converted to `kind` (int8 arrays stay what they are)."""
        a = np.atleast_2d(a)
        kind = ("int8" if a.dtype == np.int8 else F32) if kind is None else kind
        out = cls(a.shape[0], a.shape[1], kind, ld)
        host = np.zeros((out.rows, out.ld), {F32: np.float32, F16: np.float16, BF16: np.uint16, "int8": np.int8}[kind])
        host[:, : out.cols] = to_bf16(a) if kind == BF16 else a
        if host.size:
            S._check("sgemm_memcpy_h2d", S.load_library().sgemm_memcpy_h2d(out.ptr, host.ctypes.data, host.nbytes))
        return out

    def numpy(self) -> np.ndarray:
        """The values on the host (bfloat16 as float32); waits for the device, but for a stream that was
        made not to wait for it: `synchronize` first."""
        host = np.empty((self.rows, self.ld), {F32: np.float32, F16: np.float16, BF16: np.uint16, "int8": np.int8}[self.kind])
        if host.size:
            S._check("sgemm_memcpy_d2h", S.load_library().sgemm_memcpy_d2h(host.ctypes.data, self.ptr, host.nbytes))
        host = host[:, : self.cols]
        return from_bf16(host) if self.kind == BF16 else host


def _p(a):
    return None if a is None else a.ptr


def _check_sizes(func: str, sizes: int):
    """`sizes`: all sizes or'ed.  One below 0 or past 32 bits would be cut to another one on its way."""
    if sizes >> 32:
        raise ValueError(f"{func}: a size or leading dimension is not in 0 .. 2^32 - 1")


def row_bytes(cols: int) -> int:
    """The least leading dimension of 8-bit rows that the products read without a copy."""
    return -(-int(cols) // 16) * 16


def workspace_size(call: int, dtype: int, m: int, n: int, k: int) -> int:
    out = _size()
    _check_sizes("q8_workspace_size", m | n | k)
    S._check("q8_workspace_size", load_library().q8_workspace_size(call, dtype, m, n, k, ctypes.byref(out)))
    return int(out.value)


class Ops:
    """One handle of the 8-bit operators.  Leading dimensions default to the tight ones."""

    def __init__(self):
        lib = load_library()
        h = _vp()
        S._check("q8_open", lib.q8_open(ctypes.byref(h)))
        self.handle = h.value
        self._lib = lib

    def quantize(self, dtype, x, q, scale, rows, cols, ldx=None, ldq=None):
        ldx, ldq = ldx or cols, ldq or cols
        _check_sizes("q8_quantize", rows | cols | ldx | ldq)
        rc = self._lib.q8_quantize(self.handle, dtype, _p(x), ldx, _p(q), ldq, _p(scale), rows, cols)
        if rc:
            S._check("q8_quantize", rc)

    def dequantize(self, dtype, q, scale, y, rows, cols, ldq=None, ldy=None):
        ldq, ldy = ldq or cols, ldy or cols
        _check_sizes("q8_dequantize", rows | cols | ldq | ldy)
        rc = self._lib.q8_dequantize(self.handle, dtype, _p(q), ldq, _p(scale), _p(y), ldy, rows, cols)
        if rc:
            S._check("q8_dequantize", rc)

    def rmsnorm(self, dtype, x, residual, gain, hidden, q, scale, rstd, rows, cols, eps=1e-5, ldx=None, ldr=None,
                ldh=None, ldq=None):
        """hidden = x + residual; its norm in 8 bits (residual, hidden and rstd may be None)."""
        ldx, ldr, ldh, ldq = ldx or cols, ldr or cols, ldh or cols, ldq or cols
        _check_sizes("q8_rmsnorm", rows | cols | ldx | ldr | ldh | ldq)
        rc = self._lib.q8_rmsnorm(self.handle, dtype, _p(x), ldx, _p(residual), ldr, _p(gain),
                                  _p(hidden), ldh, _p(q), ldq, _p(scale), _p(rstd), rows, cols, eps)
        if rc:
            S._check("q8_rmsnorm", rc)

    def rmsnorm_backward(self, dtype, dn, hidden, gain, rstd, dres, dx, dgain, rows, cols, lddn=None, ldh=None,
                         lddr=None, lddx=None):
        """dx and dgain (float32) from dn and, where not None, dres."""
        lddn, ldh, lddr, lddx = lddn or cols, ldh or cols, lddr or cols, lddx or cols
        _check_sizes("q8_rmsnorm_backward", rows | cols | lddn | ldh | lddr | lddx)
        rc = self._lib.q8_rmsnorm_backward(self.handle, dtype, _p(dn), lddn, _p(hidden), ldh, _p(gain),
                                           _p(rstd), _p(dres), lddr, _p(dx), lddx, _p(dgain), rows, cols)
        if rc:
            S._check("q8_rmsnorm_backward", rc)

    def gemm(self, dtype, qx, sx, qw, sw, bias, y, m, n, k, ldx=None, ldw=None, ldy=None):
        """y (m x n) = (qx sx) (qw sw)^T + bias."""
        ldx, ldw, ldy = ldx or k, ldw or k, ldy or n
        _check_sizes("q8_gemm", m | n | k | ldx | ldw | ldy)
        rc = self._lib.q8_gemm(self.handle, dtype, _p(qx), ldx, _p(sx), _p(qw), ldw, _p(sw), _p(bias), _p(y), ldy,
                               m, n, k)
        if rc:
            S._check("q8_gemm", rc)

    def grad_input(self, dtype, dy, qw, sw, dx, m, n, k, lddy=None, ldw=None, lddx=None):
        """dx (m x k) = dy (qw sw)."""
        lddy, ldw, lddx = lddy or n, ldw or k, lddx or k
        _check_sizes("q8_grad_input", m | n | k | lddy | ldw | lddx)
        rc = self._lib.q8_grad_input(self.handle, dtype, _p(dy), lddy, _p(qw), ldw, _p(sw), _p(dx), lddx,
                                     m, n, k)
        if rc:
            S._check("q8_grad_input", rc)

    def grad_weight(self, dtype, dy, qx, sx, out_dtype, dw, m, n, k, lddy=None, ldx=None, lddw=None, accumulate=False):
        """dw (n x k) = dy^T (qx sx), added to what dw holds with `accumulate`."""
        lddy, ldx, lddw = lddy or n, ldx or k, lddw or k
        _check_sizes("q8_grad_weight", m | n | k | lddy | ldx | lddw)
        rc = self._lib.q8_grad_weight(self.handle, dtype, _p(dy), lddy, _p(qx), ldx, _p(sx), out_dtype, _p(dw),
                                      lddw, m, n, k, int(accumulate))
        if rc:
            S._check("q8_grad_weight", rc)

    def reserve(self, nbytes: int):
        """Grows the workspace (a call under graph capture cannot)."""
        S._check("q8_reserve", self._lib.q8_reserve(self.handle, int(nbytes)))

    def set_stream(self, stream: Optional[int]):
        """Launch on a caller-owned hipStream_t (an integer handle; None: the handle's own stream)."""
        S._check("q8_set_stream", self._lib.q8_set_stream(self.handle, stream or None))

    def synchronize(self):
        S._check("q8_synchronize", self._lib.q8_synchronize(self.handle))

    def close(self):
        if getattr(self, "handle", None):
            self._lib.q8_close(self.handle)
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
