"""The 8-bit operators at the ends of their range."""
import numpy as np
import pytest

from q8_reference import random_q
from shim import q8_shim as Q
from shim import sgemm_shim as S

pytestmark = pytest.mark.gpu

WIDEST = 2 ** 32 - 1


@pytest.fixture(scope="module")
def ops():
    with Q.Ops() as o:
        yield o


class Wide:
    """A long device array, all bytes alike at first."""

    def __init__(self, count, kind, byte):
        self.kind = kind
        self.buffer = S.DeviceBuffer(count * np.dtype(kind).itemsize)
        self.ptr = self.buffer.ptr
        S._check("sgemm_memset", S.load_library().sgemm_memset(self.ptr, byte, self.buffer.nbytes))

    def _at(self, i):
        return self.ptr + i * np.dtype(self.kind).itemsize

    def put(self, i, values):
        v = np.ascontiguousarray(values, dtype=self.kind)
        S._check("sgemm_memcpy_h2d", S.load_library().sgemm_memcpy_h2d(self._at(i), v.ctypes.data, v.nbytes))

    def get(self, i, count):
        v = np.empty(count, self.kind)
        S._check("sgemm_memcpy_d2h", S.load_library().sgemm_memcpy_d2h(v.ctypes.data, self._at(i), v.nbytes))
        return v

    def close(self):
        self.buffer.close()


@pytest.fixture
def wide():
    made = []

    def make(*args):
        made.append(Wide(*args))
        return made[-1]

    yield make
    for w in made:
        w.close()


# columns past 2^31 and the last ones, where a counter of 32 bits passes 2^32
PLACES = [0, 2 ** 31 - 4, 2 ** 32 - 8200, 2 ** 32 - 2056]


def test_widest_row_quantized(ops, wide):
    x, q, s = wide(WIDEST, np.uint16, 0x3C), wide(WIDEST, np.int8, 0x55), Q.Array(1, 1, Q.F32)
    small = float(Q.from_bf16(np.array([0x3C3C], np.uint16))[0])
    x.put(WIDEST - 3, Q.to_bf16(np.array([4 * small, -4 * small, small], np.float32)))
    ops.quantize(Q.BF16, x, q, s, 1, WIDEST)
    ops.synchronize()
    assert abs(s.numpy()[0, 0] * 127 / (4 * small) - 1) <= 2.0 ** -22
    for at in PLACES:
        assert np.all(q.get(at, 8) == 32)       # 127 / 4 = 31.75
    assert np.array_equal(q.get(WIDEST - 5, 5), [32, 32, 127, -127, 32])


def test_widest_row_restored(ops, wide):
    q, y, s = wide(WIDEST, np.int8, 1), wide(WIDEST, np.float16, 0x55), Q.Array.of(np.array([0.5]))
    q.put(WIDEST - 2, [-3, 5])
    ops.dequantize(Q.F16, q, s, y, 1, WIDEST)
    ops.synchronize()
    for at in PLACES:
        assert np.all(y.get(at, 8) == 0.5)
    assert np.array_equal(y.get(WIDEST - 4, 4), [0.5, 0.5, -1.5, 2.5])


def test_widest_row_of_the_norm_backward(ops, wide):
    # dn, hidden and gain may be one and the same: u = v^2, xhat = v, and the mean of u xhat moves dx by 1e-4 of it
    v, dx, rstd = wide(WIDEST, np.uint16, 0x3C), wide(WIDEST, np.uint16, 0x55), Q.Array.of(np.array([1.0]))
    x = float(Q.from_bf16(np.array([0x3C3C], np.uint16))[0])
    ops.rmsnorm_backward(Q.BF16, v, v, v, rstd, None, dx, None, 1, WIDEST)
    ops.synchronize()
    for at in PLACES + [WIDEST - 8]:
        got = Q.from_bf16(dx.get(at, 8))
        assert np.all(np.abs(got - (x ** 2 - x ** 4)) <= 2.0 ** -7 * x ** 2)


@pytest.mark.parametrize("cols", [2 ** 20 * 32 + 40, 2 ** 27 + 5])
def test_gains_gradient_of_wide_rows(ops, wide, cols):
    """More columns than the work-groups of a launch sum at once, and than a launch has work-items for; dx in place of dn."""
    rows = 2
    dn, hidden, gain = (wide(n * cols, np.float16, b) for n, b in ((rows, 0x3C), (rows, 0x3A), (1, 0x3B)))
    dgain, rstd = wide(cols, np.float32, 0x55), Q.Array.of(np.array([1.0, 0.5]))
    d, h, g = (float(np.array([b * 257], np.uint16).view(np.float16)[0]) for b in (0x3C, 0x3A, 0x3B))
    dn.put(cols - 1, [2 * d])        # the first row's last column
    ops.rmsnorm_backward(Q.F16, dn, hidden, gain, rstd, None, dn, dgain, rows, cols)
    ops.synchronize()
    for at in (0, 31, 2 ** 25 - 8, cols - 50, cols - 9):
        assert np.allclose(dgain.get(at, 8), d * h * 1.5, rtol=2.0 ** -20, atol=0)
    assert np.allclose(dgain.get(cols - 1, 1), d * h * 2.5, rtol=2.0 ** -20, atol=0)
    # u - xhat mean(u xhat): a thread adds up to 131072 like terms in a row, within 131072 x 2^-24 = 0.8% of their sum,
    # of which xhat takes less than one; and a rounding to 2^-11
    for row, r in ((0, 1.0), (1, 0.5)):
        want = r * d * g * (1 - (h * r) ** 2)
        got = dn.get(row * cols + cols // 2, 8).astype(np.float64)
        assert np.all(np.abs(got - want) <= 2e-2 * abs(r * d * g)), (got, want)


# the direct kernel, tiles that finish themselves (128 x 128, 256 x 256), and K ranges
@pytest.mark.parametrize("m,n,k", [(3, 70, 200), (100, 90, 700), (1000, 999, 1008), (4001, 3905, 336), (1100, 128, 4096)])
def test_scales_whose_product_is_in_range(ops, m, n, k):
    """Sum times one scale passes FP32's range, the other scale brings it back; beside them ordinary tokens.  All exact."""
    rng = np.random.default_rng(48)
    qx, qw = random_q(rng, m, k), random_q(rng, n, k)
    sums = qx.astype(np.float64) @ qw.astype(np.float64).T
    assert 2.0 ** 9 < np.abs(sums).max() < 2.0 ** 24
    for big, small in ((120, -120), (-120, 120), (97, -100)):
        sx, sw = np.full(m, 2.0 ** big), np.full(n, 2.0 ** small)
        sx[::5] = 1.0 if big > 0 else 2.0 ** -118
        y = Q.Array(m, n, Q.F32)
        ops.gemm(Q.F32, Q.Array.of(qx), Q.Array.of(sx), Q.Array.of(qw), Q.Array.of(sw), None, y, m, n, k)
        ops.synchronize()
        assert np.array_equal(y.numpy(), sums * sx[:, None] * sw)


def test_workspaces_that_cannot_be():
    """Refused, and the handle works on."""
    rng = np.random.default_rng(49)
    m, n, k = 1100, 128, 4096       # K ranges: needs a workspace
    qx, qw = random_q(rng, m, k), random_q(rng, n, k)
    y = Q.Array(m, n, Q.F32)
    with Q.Ops() as o:
        assert Q.workspace_size(Q.CALL_GEMM, Q.F32, m, n, k) > 0
        for nbytes in (2 ** 64 - 1, 2 ** 64 - 2 ** 21 + 1, 2 ** 60):
            with pytest.raises(S.SgemmError) as e:
                o.reserve(nbytes)
            assert e.value.code > 0
            o.gemm(Q.F32, Q.Array.of(qx), Q.Array.of(np.ones(m)), Q.Array.of(qw), Q.Array.of(np.ones(n)), None, y, m, n, k)
            o.synchronize()
            assert np.array_equal(y.numpy(), qx.astype(np.float64) @ qw.astype(np.float64).T)


# from the operands as they are, and laid out
@pytest.mark.parametrize("m,n,k", [(64, 64, 64), (130, 4100, 133)])
@pytest.mark.parametrize("exponent", [-110, -60, 0, 118])
def test_fp32_gradients_keep_every_bit(ops, m, n, k, exponent):
    """One product for each result, so all that is rounded is the sum of its three terms: three roundings of 2^-23 at most."""
    rng = np.random.default_rng(50)
    dy = rng.uniform(1, 2, (m, n)).astype(np.float32).astype(np.float64) * 2.0 ** exponent
    qw = np.zeros((n, k), np.int8)
    qw[rng.integers(0, n, k), np.arange(k)] = rng.integers(1, 128, k)
    dx = Q.Array(m, k, Q.F32)
    ops.grad_input(Q.F32, Q.Array.of(dy), Q.Array.of(qw), Q.Array.of(np.ones(n)), dx, m, n, k)
    ops.synchronize()
    want = dy @ qw
    assert np.all(np.abs(dx.numpy() - want) <= 3 * 2.0 ** -23 * want)
    qx = np.zeros((m, k), np.int8)
    qx[rng.integers(0, m, k), np.arange(k)] = rng.integers(1, 128, k)
    dw = Q.Array(n, k, Q.F32)
    ops.grad_weight(Q.F32, Q.Array.of(dy), Q.Array.of(qx), Q.Array.of(np.ones(m)), Q.F32, dw, m, n, k)
    ops.synchronize()
    want = dy.T @ qx
    assert np.all(np.abs(dw.numpy() - want) <= 3 * 2.0 ** -23 * want)


def test_norm_without_eps(ops):
    """A row of zeros has no norm then; others have theirs."""
    x = np.ones((3, 64))
    x[1] = 0
    q, s, rstd = Q.Array(3, 64, "int8"), Q.Array(1, 3, Q.F32), Q.Array(1, 3, Q.F32)
    ops.rmsnorm(Q.F32, Q.Array.of(x), None, Q.Array.of(np.ones(64)), None, q, s, rstd, 3, 64, eps=0.0)
    ops.synchronize()
    assert np.array_equal(q.numpy(), np.where(x > 0, 127, 0)) and np.array_equal(rstd.numpy()[0], [1, np.inf, 1])
    assert np.isnan(s.numpy()[0, 1]) and np.all(np.abs(s.numpy()[0, ::2] * 127 - 1) <= 2.0 ** -23)
