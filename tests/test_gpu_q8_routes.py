"""The 8-bit products and gradients against float64 on every kernel that they run on (test_q8_routes.py checks that these
sizes reach them all).

One row of every 16 of a result is compared, over all its columns; the others must have been written, and nothing
beside them.  Tolerances are those of test_gpu_q8_products.py.
"""
import numpy as np
import pytest

from q8_reference import TINY, TYPES, UNIT, random_q, stored
from q8_routes import DIRECTS, GEMMS, GRADIENTS
from shim import q8_shim as Q
from shim import sgemm_shim as S

pytestmark = pytest.mark.gpu

KINDS = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16, "int8": np.int8}


@pytest.fixture(scope="module")
def ops():
    with Q.Ops() as o:
        yield o


class Matrix:
    """A device matrix in rows of `pad` more values, `shift` values after a multiple of 256 bytes; what the host does not
    set is all ones, which no result is."""

    def __init__(self, rows, cols, kind, pad=0, shift=0, values=None):
        self.rows, self.cols, self.kind, self.ld, self.shift = rows, cols, kind, cols + pad, shift
        self.host = np.empty(shift + rows * self.ld + 32, KINDS[kind])
        self.host.view(np.uint8)[:] = 0xFF
        if values is not None:
            self._matrix(self.host)[:, :cols] = Q.to_bf16(values) if kind == "bf16" else values
        self.buffer = S.DeviceBuffer(self.host.nbytes)
        S._check("sgemm_memcpy_h2d", S.load_library().sgemm_memcpy_h2d(self.buffer.ptr, self.host.ctypes.data, self.host.nbytes))
        self.ptr = self.buffer.ptr + shift * self.host.itemsize

    def _matrix(self, host):
        return host[self.shift: self.shift + self.rows * self.ld].reshape(self.rows, self.ld)

    def result(self, rows):
        """The given rows as float64."""
        now = np.empty_like(self.host)
        S._check("sgemm_memcpy_d2h", S.load_library().sgemm_memcpy_d2h(now.ctypes.data, self.buffer.ptr, now.nbytes))
        bits = {1: np.uint8, 2: np.uint16, 4: np.uint32}[now.itemsize]
        inside = self._matrix(now)[:, : self.cols]
        assert not np.any(inside.view(bits) == bits(-1 % (1 << 8 * now.itemsize))), "values that were not written"
        got = inside[rows].copy()
        self._matrix(now)[:, : self.cols] = self._matrix(self.host)[:, : self.cols]
        assert np.array_equal(now.view(bits), self.host.view(bits)), "written outside the matrix"
        return (Q.from_bf16(got) if self.kind == "bf16" else got).astype(np.float64)


def sample(rng, rows):
    """One row of every 16, the first and the last."""
    some = np.arange(0, rows, 16) + rng.integers(0, 16, -(-rows // 16))
    return np.unique(np.concatenate([[0], np.minimum(some, rows - 1), [rows - 1]]))


def _product(ops, m, n, k, pad, shift, dtype):
    print(f"gemm {m}x{n}x{k} +{pad} from {shift} {dtype}", flush=True)
    rng = np.random.default_rng(41)
    qx, qw = (rng.integers(-128, 128, (r, k), dtype=np.int8) for r in (m, n))
    sx, sw = (stored(np.exp(rng.normal(-4, 1, c)), "f32") for c in (m, n))
    b = stored(rng.normal(0, 1, n), dtype)
    wx, ww, y = Matrix(m, k, "int8", pad, shift, qx), Matrix(n, k, "int8", pad, shift, qw), Matrix(m, n, dtype, pad, shift)
    ops.gemm(TYPES[dtype], wx, Q.Array.of(sx), ww, Q.Array.of(sw), Q.Array.of(b, TYPES[dtype]), y, m, n, k, ldx=wx.ld, ldw=ww.ld,
             ldy=y.ld)
    ops.synchronize()
    rows = sample(rng, m)
    p = (qx[rows].astype(np.float64) @ qw.astype(np.float64).T) * sx[rows, None] * sw
    want = p + b
    bound = UNIT[dtype] * np.abs(want) + 4 * 2.0 ** -24 * (np.abs(p) + np.abs(b)) + TINY[dtype]
    _compare(y.result(rows), want, bound, dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m,n,k,pad,shift", GEMMS)
def test_product(ops, m, n, k, pad, shift, dtype):
    _product(ops, m, n, k, pad, shift, dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("pad,shift", [(0, 0), (1, 1), (2, 0), (0, 3)])
@pytest.mark.parametrize("m,n,k", DIRECTS)
def test_few_tokens(ops, m, n, k, pad, shift, dtype):
    _product(ops, m, n, k, pad, shift, dtype)


def _compare(got, want, bound, out):
    """Within the bound; half precision ends at 65504, and what rounds past it is infinite."""
    most = 65504 if out == "f16" else np.inf
    past = np.abs(want) >= most + 16 + bound
    assert np.array_equal(got[past], np.sign(want[past]) * np.inf)
    fits = np.abs(want) <= most - bound
    bad = fits & ~(np.abs(np.where(fits, got, want) - want) <= bound)
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


def _check(got, a, b, scales, add, dtype, out):
    """got = a b + add, the 8-bit operand b with its scales."""
    want, size, count = a @ b + add, np.abs(a) @ np.abs(b), a.shape[1]
    operand = 2.0 ** -23 if dtype == "f32" else UNIT[dtype]
    sums = count * (3 if dtype == "f32" else 1) * 2.0 ** -23
    low = np.abs(a).sum(axis=1)[:, None] * scales.max() * 2.0 ** -32 if dtype == "f16" else 0
    bound = UNIT[out] * np.abs(want) + (operand * 1.01 + sums) * size + 2.0 ** -23 * np.abs(add) + low + TINY[out]
    _compare(got, want, bound, out)
    rel = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert rel <= 1.2 * (UNIT[out] + operand) + 2.0 ** -23 * (2 + np.sqrt(3.0 * count)), rel


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m,n,k,pad,shift", GRADIENTS)
def test_gradients(ops, m, n, k, pad, shift, dtype):
    print(f"gradients {m}x{n}x{k} +{pad} from {shift} {dtype}", flush=True)
    rng = np.random.default_rng(43)
    t = TYPES[dtype]
    qx, qw = (random_q(rng, r, k) for r in (m, n))
    sx, sw = (stored(np.exp(rng.normal(-4, 1, c)), "f32") for c in (m, n))
    dy = stored(0.01 * rng.standard_normal((m, n), np.float32), dtype)
    wdy, wx, ww = Matrix(m, n, dtype, pad, shift, dy), Matrix(m, k, "int8", pad, shift, qx), Matrix(n, k, "int8", pad, shift, qw)
    dx, dw = Matrix(m, k, dtype, pad, shift), Matrix(n, k, dtype, pad, shift)
    old = rng.standard_normal((n, k), np.float32)
    dw32 = Matrix(n, k, "f32", pad, shift, old)
    dsx, dsw = Q.Array.of(sx), Q.Array.of(sw)
    ops.grad_input(t, wdy, ww, dsw, dx, m, n, k, lddy=wdy.ld, ldw=ww.ld, lddx=dx.ld)
    ops.grad_weight(t, wdy, wx, dsx, t, dw, m, n, k, lddy=wdy.ld, ldx=wx.ld, lddw=dw.ld)
    ops.grad_weight(t, wdy, wx, dsx, Q.F32, dw32, m, n, k, lddy=wdy.ld, ldx=wx.ld, lddw=dw32.ld, accumulate=True)
    ops.synchronize()
    rows = sample(rng, m)
    _check(dx.result(rows), dy[rows], qw * sw[:, None], sw, np.zeros(1), dtype, dtype)
    rows = sample(rng, n)
    a, b = np.ascontiguousarray(dy[:, rows].T), qx * sx[:, None]
    _check(dw.result(rows), a, b, sx, np.zeros(1), dtype, dtype)
    _check(dw32.result(rows), a, b, sx, old[rows].astype(np.float64), dtype, "f32")


def test_copied_rows_past_32_bit_offsets(ops):
    """Rows of tokens far apart, on a tile kernel: they are copied first."""
    m, n, k, ld = 1000, 999, 1008, 1 << 23
    rng = np.random.default_rng(45)
    qx, qw = random_q(rng, m, k), random_q(rng, n, k)
    far = S.DeviceBuffer((m - 1) * ld + k)
    for i in range(m):
        row = np.ascontiguousarray(qx[i])
        S._check("sgemm_memcpy_h2d", S.load_library().sgemm_memcpy_h2d(far.ptr + i * ld, row.ctypes.data, k))
    y = Matrix(m, n, "f32")
    ops.gemm(Q.F32, far, Q.Array.of(np.ones(m)), Q.Array.of(qw), Q.Array.of(np.ones(n)), None, y, m, n, k, ldx=ld)
    ops.synchronize()
    rows = np.arange(m)
    assert np.array_equal(y.result(rows), qx.astype(np.float64) @ qw.astype(np.float64).T)     # below 2^24
    far.close()


def test_scales_that_are_not_numbers_on_tiles(ops):
    """They reach their row or column, on a kernel that finishes itself and on one that adds K ranges."""
    rng = np.random.default_rng(46)
    for m, n, k in ((1000, 999, 1008), (1100, 128, 4096)):
        sx, sw = np.ones(m), np.ones(n)
        sx[m - 3], sw[n - 5] = np.nan, np.inf
        y = Q.Array(m, n, Q.BF16)
        ops.gemm(Q.BF16, Q.Array.of(random_q(rng, m, k)), Q.Array.of(sx), Q.Array.of(random_q(rng, n, k)), Q.Array.of(sw), None, y,
                 m, n, k)
        ops.synchronize()
        bad = ~np.isfinite(y.numpy())
        assert bad[m - 3].all() and bad[:, n - 5].all()
        bad[m - 3] = bad[:, n - 5] = False
        assert not bad.any()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_longest_sums(ops, dtype):
    """Exact: whole numbers of random signs, whose partial sums stay far below 2^24 (a deviation of 2^16 over all of them)."""
    few, summed, k = 9, Q.MAX_SUM_F32 if dtype == "f32" else Q.MAX_SUM, 14
    t = TYPES[dtype]
    rng = np.random.default_rng(47)
    q, d = rng.integers(-100, 101, (summed, k), dtype=np.int8), rng.integers(-1, 2, (few, summed), dtype=np.int8)
    want = d.astype(np.float64) @ q.astype(np.float64)
    assert np.abs(want).max() < 2.0 ** 20
    one, dq = Q.Array.of(np.ones(summed)), Q.Array.of(q)
    out = Q.Array(few, k, Q.F32)
    ops.grad_weight(t, Q.Array.of(np.ascontiguousarray(d.T).astype(np.float32), t), dq, one, Q.F32, out, summed, few, k)
    ops.synchronize()
    assert np.array_equal(out.numpy(), want)
    out = Q.Array(few, k, t)
    ops.grad_input(t, Q.Array.of(d.astype(np.float32), t), dq, one, out, few, summed, k)
    ops.synchronize()
    with np.errstate(over="ignore"):
        assert np.array_equal(out.numpy().astype(np.float64), stored(want, dtype))
