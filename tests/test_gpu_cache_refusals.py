"""What the rotary, cache and attention operators refuse, and that a refused call leaves its outputs alone."""
import numpy as np
import pytest

from shim import q8_cache as C
from shim import sgemm_shim as S

pytestmark = pytest.mark.gpu

INVALID, SHAPE = -1, -4
TOKENS, HEADS, KV, DIM, PAGES, PAGE = 4, 4, 2, 32, 3, 16
COLS, KCOLS, ROWS = HEADS * DIM, KV * DIM, PAGES * KV * PAGE


class At:
    def __init__(self, ptr):
        self.ptr = ptr


class Env:
    def __init__(self):
        f32 = lambda n: C.Array(1, n, C.F32)
        self.arrays = {"x": f32(TOKENS * COLS), "y": f32(TOKENS * COLS), "k": f32(TOKENS * KCOLS), "v": f32(TOKENS * KCOLS), "lse": f32(TOKENS * HEADS),
                       "ck": C.Array(ROWS, DIM, "int8"), "cv": C.Array(ROWS, DIM, "int8"), "sk": f32(ROWS), "sv": f32(ROWS), "positions": f32(2 * TOKENS),
                       "freq": f32(DIM // 2), "starts": f32(3), "lengths": f32(2), "table": f32(4)}
        self.__dict__.update(self.arrays)
        for b in self.arrays.values():
            S._check("sgemm_memset", S.load_library().sgemm_memset(b.ptr, 0x3c, b.nbytes))

    def form(self, dim=DIM, axis=(0,) * 16, axes=2):
        return C.Rotation(dim, axis, axes)

    def cache(self, pages=PAGES, page=PAGE, heads=KV, dim=DIM, **memory):
        m = {"k": self.ck, "v": self.cv, "k_scale": self.sk, "v_scale": self.sv, **memory}
        return C.Cache(m["k"], m["v"], m["k_scale"], m["v_scale"], pages, page, heads, dim)

    def batch(self, seqs=2, tokens=TOKENS, width=2, ld=None, **memory):
        m = {"starts": self.starts, "lengths": self.lengths, "table": self.table, **memory}
        return C.Batch(m["starts"], m["lengths"], m["table"], seqs, tokens, width, ld)

    def rotary(self, o, dtype=C.F32, form=None, x=0, positions=0, freq=0, y=0, tokens=TOKENS, heads=HEADS, **ld):
        x, positions, freq, y = (d if a == 0 else a for a, d in ((x, self.x), (positions, self.positions), (freq, self.freq), (y, self.y)))
        o.rotary(dtype, form or self.form(), x, positions, freq, y, tokens, heads, **ld)

    def write(self, o, dtype=C.F32, k=0, v=0, cache={}, batch={}, **ld):
        o.cache_write(dtype, self.cache(**cache), self.batch(**batch), self.k if k == 0 else k, self.v if v == 0 else v, **ld)

    def read(self, o, dtype=C.F32, k=0, v=0, cache={}, batch={}, **ld):
        o.cache_read(dtype, self.cache(**cache), self.batch(**batch), self.k if k == 0 else k, self.v if v == 0 else v, **ld)

    def attention(self, o, dtype=C.F32, heads=HEADS, q=0, out=0, lse=0, cache={}, batch={}, **more):
        o.attention(dtype, self.cache(**cache), self.batch(**batch), heads, self.x if q == 0 else q, self.y if out == 0 else out,
                    self.lse if lse == 0 else lse, **more)


@pytest.fixture(scope="module")
def env():
    with C.Ops() as ops:
        yield ops, Env()


CALLS = {
    "rotary: type": (INVALID, "type", lambda o, e: e.rotary(o, dtype=9)),
    "rotary: null x": (INVALID, "x is null", lambda o, e: e.rotary(o, x=None)),
    "rotary: null y": (INVALID, "y is null", lambda o, e: e.rotary(o, y=None)),
    "rotary: null positions": (INVALID, "positions is null", lambda o, e: e.rotary(o, positions=None)),
    "rotary: null freq": (INVALID, "freq is null", lambda o, e: e.rotary(o, freq=None)),
    "rotary: alignment": (INVALID, "aligned", lambda o, e: e.rotary(o, x=At(e.x.ptr + 2), tokens=1)),
    "rotary: part of x": (INVALID, "y overlaps x", lambda o, e: e.rotary(o, y=At(e.x.ptr + 4 * COLS), tokens=TOKENS - 1)),
    "rotary: x with another ld": (INVALID, "y overlaps x", lambda o, e: e.rotary(o, y=e.x, tokens=2, ldy=2 * COLS)),
    "rotary: y is positions": (INVALID, "overlaps positions", lambda o, e: e.rotary(o, y=e.positions, tokens=1, heads=1)),
    "rotary: ld of x": (SHAPE, "x: leading", lambda o, e: e.rotary(o, ldx=COLS - 1)),
    "rotary: ld of positions": (SHAPE, "positions: leading", lambda o, e: e.rotary(o, ldp=TOKENS - 1)),
    "rotary: pairs": (SHAPE, "pairs", lambda o, e: e.rotary(o, form=e.form(30, (0,) * 16))),
    "rotary: no axes": (SHAPE, "axes", lambda o, e: e.rotary(o, form=e.form(axes=0))),
    "rotary: many axes": (SHAPE, "axes", lambda o, e: e.rotary(o, form=e.form(axes=9))),
    "rotary: an axis that is not there": (INVALID, "on axis 2", lambda o, e: e.rotary(o, form=e.form(axis=(0, 2)))),
    "rotary: wide heads": (SHAPE, "257", lambda o, e: e.rotary(o, form=e.form(257))),
    "rotary: no values": (SHAPE, "heads of 0", lambda o, e: e.rotary(o, form=e.form(0, ()))),
    "rotary: many heads": (SHAPE, "2^24", lambda o, e: e.rotary(o, tokens=1, heads=2 ** 20)),
    "rotary: many tokens": (SHAPE, "31 bits", lambda o, e: e.rotary(o, tokens=2 ** 31)),
    "write: type": (INVALID, "type", lambda o, e: e.write(o, dtype=-1)),
    "write: null k": (INVALID, "k is null", lambda o, e: e.write(o, k=None)),
    "write: null cache": (INVALID, "cache v is null", lambda o, e: e.write(o, cache={"v": None})),
    "write: null scale": (INVALID, "k_scale is null", lambda o, e: e.write(o, cache={"k_scale": None})),
    "write: null table": (INVALID, "table is null", lambda o, e: e.write(o, batch={"table": None})),
    "write: null starts": (INVALID, "starts is null", lambda o, e: e.write(o, batch={"starts": None})),
    "write: null lengths": (INVALID, "lengths is null", lambda o, e: e.write(o, batch={"lengths": None})),
    "write: alignment": (INVALID, "16 bytes", lambda o, e: e.write(o, cache={"k": At(e.ck.ptr + 8), "pages": 1})),
    "write: ld of v": (SHAPE, "v: leading", lambda o, e: e.write(o, ldv=KCOLS - 1)),
    "write: ld of the table": (SHAPE, "table: leading", lambda o, e: e.write(o, batch={"ld": 1})),
    "write: k is the cache": (INVALID, "overlaps k", lambda o, e: e.write(o, k=e.ck, batch={"tokens": 1})),
    "write: one cache twice": (INVALID, "cache v overlaps cache k", lambda o, e: e.write(o, cache={"v": e.ck})),
    "write: table in the cache": (INVALID, "overlaps table", lambda o, e: e.write(o, batch={"table": e.ck})),
    "read: type": (INVALID, "type", lambda o, e: e.read(o, dtype=3)),
    "read: null v": (INVALID, "v is null", lambda o, e: e.read(o, v=None)),
    "read: into the cache": (INVALID, "overlaps cache", lambda o, e: e.read(o, k=e.ck, batch={"tokens": 1})),
    "read: k is v": (INVALID, "v overlaps k", lambda o, e: e.read(o, v=e.k)),
    "read: into the lengths": (INVALID, "overlaps lengths", lambda o, e: e.read(o, k=e.lengths, cache={"dim": 1, "heads": 1}, batch={"tokens": 1})),
    "attention: type": (INVALID, "type", lambda o, e: e.attention(o, dtype=5)),
    "attention: null q": (INVALID, "q is null", lambda o, e: e.attention(o, q=None)),
    "attention: null out": (INVALID, "out is null", lambda o, e: e.attention(o, out=None)),
    "attention: heads": (SHAPE, "multiple", lambda o, e: e.attention(o, heads=3)),
    "attention: no heads": (SHAPE, "multiple", lambda o, e: e.attention(o, heads=0)),
    "attention: scale": (INVALID, "scale", lambda o, e: e.attention(o, scale=float("nan"))),
    "attention: scale without end": (INVALID, "scale", lambda o, e: e.attention(o, scale=float("inf"))),
    "attention: scale past 2^100": (INVALID, "2^100", lambda o, e: e.attention(o, scale=-1.3e30)),
    "attention: ld of q": (SHAPE, "q: leading", lambda o, e: e.attention(o, ldq=COLS - 1)),
    "attention: ld of out": (SHAPE, "out: leading", lambda o, e: e.attention(o, ldo=COLS - 1)),
    "attention: out is q": (INVALID, "out overlaps q", lambda o, e: e.attention(o, out=e.x)),
    "attention: lse is out": (INVALID, "lse overlaps out", lambda o, e: e.attention(o, lse=e.y)),
    "attention: lse in the cache": (INVALID, "lse overlaps cache", lambda o, e: e.attention(o, lse=e.sk)),
    "attention: out is the table": (INVALID, "out overlaps table", lambda o, e: e.attention(o, out=e.table, q=e.x, heads=1, cache={"heads": 1, "dim": 1}, batch={"tokens": 1})),
    "attention: alignment of lse": (INVALID, "aligned", lambda o, e: e.attention(o, lse=At(e.lse.ptr + 2), batch={"tokens": 1})),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_refusals(env, name):
    code, what, call = CALLS[name]
    ops, e = env
    with pytest.raises(S.SgemmError) as error:
        call(ops, e)
    assert error.value.code == code and what in error.value.message, error.value.message
    ops.synchronize()
    for key, b in e.arrays.items():
        raw = S.DeviceView(b, 0, b.nbytes // 4 * 4).download().view(np.uint32)
        assert np.all(raw == 0x3c3c3c3c), key


def test_nothing_to_do_is_no_error(env):
    ops, e = env
    e.rotary(ops, tokens=0, x=None, positions=None, freq=None, y=None)
    e.rotary(ops, heads=0)
    for call in (e.write, e.read):
        call(ops, k=None, v=None, batch={"tokens": 0})
        call(ops, batch={"seqs": 0, "starts": None, "lengths": None, "table": None})
    e.attention(ops, q=None, out=None, lse=None, batch={"tokens": 0})
    ops.synchronize()
    for key, b in e.arrays.items():
        assert np.all(S.DeviceView(b, 0, b.nbytes // 4 * 4).download().view(np.uint32) == 0x3c3c3c3c), key
