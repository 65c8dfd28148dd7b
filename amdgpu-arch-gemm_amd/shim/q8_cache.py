"""ctypes binding of the rotary, cache and attention operators in libsgemm_shim.so
(include/q8_cache.h).

``Ops`` is ``q8_shim.Ops`` (one handle: a stream and a workspace) with these
operators besides, so one handle serves a whole block.  Device memory is passed as objects with a
``ptr``.  ``Rotation``, ``Cache`` and ``Batch`` describe a model's and a batch's
sizes and memory; a program makes them once and keeps them.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import numpy as np

from . import q8_shim as Q
from . import sgemm_shim as S
from .q8_shim import BF16, F16, F32, Array, row_bytes  # noqa: F401

MAX_DIM, MAX_AXES = 256, 8

_int, _u32, _f32, _vp, _size = ctypes.c_int, ctypes.c_uint32, ctypes.c_float, ctypes.c_void_p, ctypes.c_size_t


class _Rotation(ctypes.Structure):
    _fields_ = [("dim", _u32), ("pairs", _u32), ("axes", _u32), ("neighbours", _u32), ("axis", ctypes.c_uint8 * 128)]


class _Cache(ctypes.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("k_scale", _vp), ("v_scale", _vp), ("pages", _u32), ("page_tokens", _u32),
                ("heads", _u32), ("dim", _u32)]


class _Batch(ctypes.Structure):
    _fields_ = [("starts", _vp), ("lengths", _vp), ("table", _vp), ("seqs", _u32), ("tokens", _u32), ("width", _u32),
                ("table_ld", _u32), ("longest", _u32)]


# every symbol the header declares, with (restype, argtypes)
SIGNATURES = {
    "q8_rotary": (_int, [_vp, _int, _vp, _vp, _u32, _vp, _u32, _vp, _vp, _u32, _u32, _u32, _int]),
    "q8_cache_write": (_int, [_vp, _int, _vp, _vp, _vp, _u32, _vp, _u32]),
    "q8_cache_read": (_int, [_vp, _int, _vp, _vp, _vp, _u32, _vp, _u32]),
    "q8_attention": (_int, [_vp, _int, _vp, _vp, _u32, _vp, _u32, _f32, _u32, _vp, _u32, _vp]),
    "q8_attention_workspace": (_int, [_int, _vp, _vp, _u32, ctypes.POINTER(_size)]),
}

_lib: Optional[ctypes.CDLL] = None


def load_library() -> ctypes.CDLL:
    """The shim with these operators' signatures set, and those of q8_shim."""
    global _lib
    if _lib is None:
        lib = Q.load_library()
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


_p, _check_sizes = Q._p, Q._check_sizes


def ints(a) -> S.DeviceBuffer:
    """`a` on the device as int32 (positions, starts, lengths, tables)."""
    a = np.asarray(a)
    host = np.ascontiguousarray(a, dtype=np.int32)
    if not np.array_equal(host, a):
        raise ValueError("ints: a value that int32 does not hold")
    out = S.DeviceBuffer(max(4, host.nbytes))
    if host.size:
        S._check("sgemm_memcpy_h2d", S.load_library().sgemm_memcpy_h2d(out.ptr, host.ctypes.data, host.nbytes))
    return out


class Rotation:
    """How positions turn heads of `dim` values: `axis` names each pair's axis (its length is the number of pairs)."""

    def __init__(self, dim: int, axis: Sequence[int], axes: int = 1, neighbours: bool = False):
        axis = [int(a) for a in axis]
        if len(axis) > MAX_DIM // 2 or any(a not in range(256) for a in axis):
            raise ValueError(f"Rotation: at most {MAX_DIM // 2} pairs, on axes below {MAX_AXES}")
        _check_sizes("Rotation", dim | axes)
        self.dim, self.pairs = dim, len(axis)
        self.form = _Rotation(dim, len(axis), axes, int(neighbours), (ctypes.c_uint8 * 128)(*axis))
        self.at = ctypes.addressof(self.form)


class Cache:
    """Pages of 8-bit keys and values of one layer; the memory is kept alive."""

    def __init__(self, k, v, k_scale, v_scale, pages: int, page_tokens: int, heads: int, dim: int):
        _check_sizes("Cache", pages | page_tokens | heads | dim)
        self.memory = (k, v, k_scale, v_scale)
        self.pages, self.page_tokens, self.heads, self.dim = pages, page_tokens, heads, dim
        self.form = _Cache(_p(k), _p(v), _p(k_scale), _p(v_scale), pages, page_tokens, heads, dim)
        self.at = ctypes.addressof(self.form)

    @classmethod
    def empty(cls, pages: int, page_tokens: int, heads: int, dim: int) -> "Cache":
        """A new one; what its pages hold is not defined until it is written."""
        rows = pages * heads * page_tokens
        return cls(Array(rows, row_bytes(dim), "int8"), Array(rows, row_bytes(dim), "int8"), Array(1, rows, F32), Array(1, rows, F32),
                   pages, page_tokens, heads, dim)


class Batch:
    """Sequences and their new tokens, described in device memory (int32), which is kept alive; `width` pages a row
    of the table, rows `table_ld` apart (default: width)."""

    def __init__(self, starts, lengths, table, seqs: int, tokens: int, width: int, table_ld: Optional[int] = None, longest: int = 0):
        table_ld = width if table_ld is None else table_ld
        _check_sizes("Batch", seqs | tokens | width | table_ld | longest)
        self.memory = (starts, lengths, table)
        self.seqs, self.tokens, self.width = seqs, tokens, width
        self.form = _Batch(_p(starts), _p(lengths), _p(table), seqs, tokens, width, table_ld, longest)
        self.at = ctypes.addressof(self.form)


def attention_workspace(dtype: int, cache: Cache, batch: Batch, heads: int) -> int:
    out = _size()
    _check_sizes("q8_attention_workspace", heads)
    S._check("q8_attention_workspace", load_library().q8_attention_workspace(dtype, cache.at, batch.at, heads, ctypes.byref(out)))
    return int(out.value)


class Ops(Q.Ops):
    """One handle of the 8-bit operators, these among them.  Leading dimensions default to the tight ones."""

    def __init__(self):
        load_library()
        super().__init__()

    def rotary(self, dtype, form: Rotation, x, positions, freq, y, tokens, heads, ldx=None, ldp=None, ldy=None, inverse=False):
        """y = x (tokens x heads of form.dim values) turned by its positions (int32, one row of `ldp` for each axis)."""
        cols = heads * form.dim
        ldx, ldp, ldy = ldx or cols, ldp or tokens, ldy or cols
        _check_sizes("q8_rotary", tokens | heads | ldx | ldp | ldy)
        rc = self._lib.q8_rotary(self.handle, dtype, form.at, _p(x), ldx, _p(positions), ldp, _p(freq), _p(y), ldy, tokens, heads,
                                 int(inverse))
        if rc:
            S._check("q8_rotary", rc)

    def cache_write(self, dtype, cache: Cache, batch: Batch, k, v, ldk=None, ldv=None):
        """The new tokens' keys and values (rows of cache.heads heads) to 8 bits, into their pages."""
        cols = cache.heads * cache.dim
        ldk, ldv = ldk or cols, ldv or cols
        _check_sizes("q8_cache_write", ldk | ldv)
        rc = self._lib.q8_cache_write(self.handle, dtype, cache.at, batch.at, _p(k), ldk, _p(v), ldv)
        if rc:
            S._check("q8_cache_write", rc)

    def cache_read(self, dtype, cache: Cache, batch: Batch, k, v, ldk=None, ldv=None):
        """The new tokens' keys and values back from their pages."""
        cols = cache.heads * cache.dim
        ldk, ldv = ldk or cols, ldv or cols
        _check_sizes("q8_cache_read", ldk | ldv)
        rc = self._lib.q8_cache_read(self.handle, dtype, cache.at, batch.at, _p(k), ldk, _p(v), ldv)
        if rc:
            S._check("q8_cache_read", rc)

    def attention(self, dtype, cache: Cache, batch: Batch, heads, q, out, lse=None, scale=None, window=0, ldq=None, ldo=None):
        """out = the new tokens' attention over the cache; lse (float32, tokens x heads) where it is wanted.  `scale`
        defaults to dim^-1/2; `window` > 0: only the last so many positions."""
        cols = heads * cache.dim
        ldq, ldo = ldq or cols, ldo or cols
        _check_sizes("q8_attention", heads | window | ldq | ldo)
        rc = self._lib.q8_attention(self.handle, dtype, cache.at, batch.at, heads, _p(q), ldq,
                                    cache.dim ** -0.5 if scale is None else scale, window, _p(out), ldo, _p(lse))
        if rc:
            S._check("q8_attention", rc)
