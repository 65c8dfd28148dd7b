"""The 8-bit product and its gradients against float64.

Tolerances.  q8_gemm's sums are exact; a conversion, two products and a sum round
to 2^-24 each, and the result to its type.  The gradients' 16-bit operand is
rounded once (UNIT of the type), n products are summed in FP32 in some order (n *
2^-23 of the sum of magnitudes), and the result is rounded.
"""
import numpy as np
import pytest

from q8_reference import TINY, TYPES, UNIT, Window, random_q, stored
from test_gpu_noalloc_streams import _Hip, _ok
from shim import q8_shim as Q
from shim import sgemm_shim as S

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    with Q.Ops() as o:
        yield o


def _product(ops, m, n, k, dtype, pad=0, shift=0, bias=False, seed=21, lo=-128):
    rng = np.random.default_rng(seed)
    t = TYPES[dtype]
    qx, qw = random_q(rng, m, k, lo), random_q(rng, n, k, lo)
    sx, sw = (stored(np.exp(rng.normal(-4, 1, c)), "f32") for c in (m, n))
    b = stored(rng.normal(0, 1, n), dtype) if bias else None
    wx, ww = Window(m, k, "int8", pad, shift, qx), Window(n, k, "int8", pad, shift, qw)
    y = Window(m, n, t, pad, shift)
    ops.gemm(t, wx, Q.Array.of(sx), ww, Q.Array.of(sw), None if b is None else Q.Array.of(b, t), y, m, n, k,
             ldx=wx.ld, ldw=ww.ld, ldy=y.ld)
    ops.synchronize()
    p = (qx.astype(np.float64) @ qw.astype(np.float64).T) * sx[:, None] * sw
    want = p + (0 if b is None else b)
    bound = UNIT[dtype] * np.abs(want) + 4 * 2.0 ** -24 * (np.abs(p) + (0 if b is None else np.abs(b))) + TINY[dtype]
    got = y.values()
    assert np.all(np.abs(got - want) <= bound), (m, n, k, np.abs(got - want).max())
    return got


# a token to a few, past the few; one column to ragged tiles; sums of one to odd ends of a K tile
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 64, 64), (1, 1000, 4096), (2, 129, 517), (16, 333, 1000), (17, 31, 127),
                                   (33, 257, 129), (64, 512, 2048), (65, 1, 1), (65, 130, 16), (127, 129, 130),
                                   (129, 127, 4097), (333, 129, 517), (513, 300, 64), (1000, 999, 65), (300, 4000, 129)])
def test_gemm(ops, m, n, k, dtype):
    print(f"gemm {m}x{n}x{k} {dtype}", flush=True)
    _product(ops, m, n, k, dtype, bias=(m + n) % 2 == 1)


@pytest.mark.parametrize("pad,shift", [(1, 0), (3, 5), (16, 16), (15, 1), (0, 3)])
@pytest.mark.parametrize("m,n,k", [(5, 70, 200), (40, 33, 65), (200, 140, 512), (130, 260, 1001)])
def test_gemm_rows_that_start_anywhere(ops, m, n, k, pad, shift):
    _product(ops, m, n, k, "bf16", pad, shift, bias=True)


# each tile of the few-token kernel, from whole dwords and from between them
@pytest.mark.parametrize("pad,shift", [(0, 0), (1, 1), (2, 0), (0, 3)])
@pytest.mark.parametrize("m,n,k", [(3, 200, 1300), (2, 70, 8300), (3, 12300, 140), (20, 5000, 140), (20, 12300, 140), (50, 5000, 200),
                                   (50, 12300, 140), (100, 90, 700), (300, 900, 72)])
def test_gemm_few_tokens_from_any_byte(ops, m, n, k, pad, shift):
    print(f"gemm {m}x{n}x{k} +{pad} from {shift}", flush=True)
    _product(ops, m, n, k, "f16", pad, shift, bias=True)


# whole rows of 16 bytes that hold values past the sum, which must not count
@pytest.mark.parametrize("k", [1, 15, 17, 100, 127, 130, 250, 255])
def test_gemm_sums_that_end_inside_a_piece(ops, k):
    for m in (20, 150):
        _product(ops, m, 140, k, "f32", pad=-k % 16 + 16)


@pytest.mark.parametrize("m,n,k", [(128, 128, 8192), (512, 512, 16384), (300, 200, 40000), (1100, 128, 4096), (257, 257, 131071)])
def test_gemm_in_k_ranges(ops, m, n, k):
    first = _product(ops, m, n, k, "f32")
    assert np.array_equal(_product(ops, m, n, k, "f32"), first)


def test_gemm_largest_sums(ops):
    """Every product is 2^14 and their sum 131071 * 2^14, just inside 32 bits."""
    k = Q.MAX_K
    for m in (3, 70):
        qx, qw = np.full((m, k), -128, np.int8), np.full((5, k), -128, np.int8)
        y = Window(m, 5, Q.F32)
        one = Q.Array.of(np.ones(m))
        ops.gemm(Q.F32, Q.Array.of(qx), one, Q.Array.of(qw), Q.Array.of(np.ones(5)), None, y, m, 5, k)
        ops.synchronize()
        assert np.all(y.values() == np.float32(k * 2.0 ** 14))


def test_gemm_scales_that_are_not_numbers_stay_in_their_row(ops):
    rng = np.random.default_rng(3)
    for m in (9, 100):
        n, k = 40, 64
        sx, sw = np.ones(m), np.ones(n)
        sx[4], sw[7] = np.nan, np.inf
        y = Window(m, n, Q.BF16)
        ops.gemm(Q.BF16, Q.Array.of(random_q(rng, m, k)), Q.Array.of(sx), Q.Array.of(random_q(rng, n, k)), Q.Array.of(sw),
                 None, y, m, n, k)
        ops.synchronize()
        bad = ~np.isfinite(y.values())
        assert bad[4].all() and bad[:, 7].all()
        bad[4] = bad[:, 7] = False
        assert not bad.any()


def test_empty_sums_and_outputs(ops):
    for m in (3, 100):
        one, b = Q.Array.of(np.ones(m)), Q.Array.of(np.arange(40.0))
        y = Window(m, 40, Q.F32)
        ops.gemm(Q.F32, None, one, None, Q.Array.of(np.ones(40)), b, y, m, 40, 0)
        ops.synchronize()
        assert np.array_equal(y.values(), np.tile(np.arange(40.0), (m, 1)))
        ops.gemm(Q.F32, None, None, None, None, None, None, 0, 40, 8)
        ops.gemm(Q.F32, None, None, None, None, None, None, m, 0, 8)
        dx, dw = Window(m, 24, Q.BF16), Window(40, 24, Q.F32)
        ops.grad_input(Q.BF16, None, None, None, dx, m, 0, 24)
        ops.grad_weight(Q.BF16, None, None, None, Q.F32, dw, 0, 40, 24, accumulate=True)    # nothing is added
        ops.synchronize()
        assert np.all(dx.values() == 0) and np.all(dw.values() == 85)
        ops.grad_weight(Q.F16, None, None, None, Q.F32, dw, 0, 40, 24)
        ops.synchronize()
        assert np.all(dw.values() == 0)


def _gradients(ops, m, n, k, dtype, pad=0, shift=0, out=None, accumulate=False, seed=31, spread=1.0):
    rng = np.random.default_rng(seed)
    t = TYPES[dtype]
    out = out or dtype
    qx, qw = random_q(rng, m, k), random_q(rng, n, k)
    sx, sw = (stored(np.exp(rng.normal(-4, spread, c)), "f32") for c in (m, n))
    dy = stored(0.01 * rng.normal(0, 1, (m, n)), dtype)
    if m > 4:
        dy[3] = 0
    old = stored(rng.normal(0, 1, (n, k)), out)
    wdy, wx, ww = Window(m, n, t, pad, shift, dy), Window(m, k, "int8", pad, shift, qx), Window(n, k, "int8", pad, shift, qw)
    dx, dw = Window(m, k, t, pad, shift), Window(n, k, TYPES[out], pad, shift, old)
    ops.grad_input(t, wdy, ww, Q.Array.of(sw), dx, m, n, k, lddy=wdy.ld, ldw=ww.ld, lddx=dx.ld)
    ops.grad_weight(t, wdy, wx, Q.Array.of(sx), TYPES[out], dw, m, n, k, lddy=wdy.ld, ldx=wx.ld, lddw=dw.ld,
                    accumulate=accumulate)
    ops.synchronize()
    for got, a, b, s, kind, add in ((dx.values(), dy, qw * sw[:, None], sw, dtype, 0),
                                    (dw.values(), dy.T, qx * sx[:, None], sx, out, old if accumulate else 0)):
        want, size, count = a @ b + add, np.abs(a) @ np.abs(b), a.shape[1]
        operand = 2.0 ** -23 if dtype == "f32" else UNIT[dtype]
        sums = count * (3 if dtype == "f32" else 1) * 2.0 ** -23
        # half precision: values below 2^-14 of 2^-7 of the largest scale keep steps of 2^-24 of that
        low = np.abs(a).sum(axis=1)[:, None] * s.max() * 2.0 ** -32 if dtype == "f16" else 0
        bound = (UNIT[kind] * np.abs(want) + (operand * 1.01 + sums) * size + 2.0 ** -23 * np.abs(add) + low + TINY[kind])
        # half precision ends at 65504, and what rounds past it is infinite
        most = 65504 if kind == "f16" else np.inf
        past = np.abs(want) >= most + 16 + bound
        assert np.array_equal(got[past], np.sign(want[past]) * np.inf)
        fits = np.abs(want) <= most - bound
        got, want, bound = got[fits], want[fits], bound[fits]
        assert np.all(np.abs(got - want) <= bound), (m, n, k, dtype, np.abs(got - want).max())
        # and on the whole: independent roundings of the operand, of sums and of the result
        rel = np.linalg.norm(got - want) / np.linalg.norm(want)
        assert rel <= 1.2 * (UNIT[kind] + operand) + 2.0 ** -23 * (2 + np.sqrt(3.0 * count)), rel
    return dx.values(), dw.values()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 64, 40), (7, 129, 33), (64, 64, 64), (130, 128, 257), (333, 129, 517),
                                   (500, 1000, 72), (1000, 999, 409)])
def test_gradients(ops, m, n, k, dtype):
    print(f"gradients {m}x{n}x{k} {dtype}", flush=True)
    _gradients(ops, m, n, k, dtype)


@pytest.mark.parametrize("dtype,pad,shift", [("bf16", 8, 8), ("bf16", 3, 1), ("f16", 16, 16), ("f16", 1, 0), ("f32", 4, 3)])
def test_gradients_rows_that_start_anywhere(ops, dtype, pad, shift):
    _gradients(ops, 150, 136, 200, dtype, pad, shift)


@pytest.mark.parametrize("dtype,out", [("bf16", "f32"), ("f16", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f32")])
def test_weight_gradients_accumulate(ops, dtype, out):
    _gradients(ops, 140, 150, 130, dtype, out=out, accumulate=True)


def test_gradients_with_scales_far_apart(ops):
    for dtype in TYPES:
        _gradients(ops, 200, 150, 130, dtype, spread=4.0)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_gradients_in_k_ranges(ops, dtype):
    first = _gradients(ops, 6000, 100, 60, dtype)
    again = _gradients(ops, 6000, 100, 60, dtype)
    assert all(np.array_equal(a, b) for a, b in zip(first, again))


# The sizes above are taken from the operands as they are, most of these are laid out: the input's
# gradient, the weights', or both.
LAID_OUT = [(1301, 1203, 1501, 0, 0), (130, 4100, 133, 0, 0), (4100, 130, 133, 0, 0), (2050, 130, 1000, 3, 1),
            (333, 5000, 129, 8, 8), (9, 30, 6, 0, 0), (30, 7, 70, 1, 1), (2701, 2203, 1301, 0, 0)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m,n,k,pad,shift", LAID_OUT)
def test_gradients_laid_out(ops, m, n, k, pad, shift, dtype):
    print(f"gradients {m}x{n}x{k} +{pad} {dtype}", flush=True)
    _gradients(ops, m, n, k, dtype, pad, shift)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("call", [Q.CALL_GRAD_INPUT, Q.CALL_GRAD_WEIGHT])
def test_sizes_reach_both_routes(call, dtype):
    needs = [Q.workspace_size(call, TYPES[dtype], m, n, k) for m, n, k, _, _ in LAID_OUT]
    assert sum(need > 0 for need in needs) >= 3
    assert Q.workspace_size(call, TYPES[dtype], 64, 64, 64) == 0


@pytest.mark.parametrize("dtype,out", [("bf16", "f32"), ("f16", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f32")])
def test_weight_gradients_laid_out_accumulate(ops, dtype, out):
    _gradients(ops, 4100, 130, 133, dtype, out=out, accumulate=True)


# ends of tiles (64 and 128 rows, 64 columns), of the last values of a row that are taken with those
# before them, of a wave's steps (32) and of four or eight waves' turns
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m,n,k", [(32, 32, 4), (33, 39, 5), (63, 65, 7), (65, 64, 68), (127, 129, 67), (129, 136, 63), (40, 8, 64),
                                   (160, 161, 30), (511, 160, 61), (513, 513, 60), (545, 1100, 131)])
def test_gradients_ends(ops, m, n, k, dtype):
    print(f"gradients {m}x{n}x{k} {dtype}", flush=True)
    _gradients(ops, m, n, k, dtype)
    _gradients(ops, m, n, k, dtype, 5, 3, accumulate=True)


def test_gradients_against_differences(ops):
    """The product is linear in its 8-bit operands: a step of one in an operand changes a
    loss by exactly its gradient times the scale."""
    m, n, k = 70, 33, 40
    rng = np.random.default_rng(5)
    qx, qw = random_q(rng, m, k, -100), random_q(rng, n, k, -100)
    sx, sw = (2.0 ** rng.integers(-3, 3, c) for c in (m, n))     # exact products throughout
    c = rng.integers(-4, 5, (m, n)).astype(np.float64)

    def loss(qx, qw):
        y = Q.Array(m, n, Q.F32)
        ops.gemm(Q.F32, Q.Array.of(qx), Q.Array.of(sx), Q.Array.of(qw), Q.Array.of(sw), None, y, m, n, k)
        ops.synchronize()
        return (y.numpy().astype(np.float64) * c).sum()

    dx, dw = Q.Array(m, k, Q.F32), Q.Array(n, k, Q.F32)
    ops.grad_input(Q.F32, Q.Array.of(c), Q.Array.of(qw), Q.Array.of(sw), dx, m, n, k)
    ops.grad_weight(Q.F32, Q.Array.of(c), Q.Array.of(qx), Q.Array.of(sx), Q.F32, dw, m, n, k)
    ops.synchronize()
    base = loss(qx, qw)
    for i, j in ((0, 0), (69, 39), (17, 5), (64, 20)):
        step = qx.copy()
        step[i, j] += 1
        assert loss(step, qw) - base == dx.numpy()[i, j] * sx[i]
    for i, j in ((0, 0), (32, 39), (16, 5)):
        step = qw.copy()
        step[i, j] += 1
        assert loss(qx, step) - base == dw.numpy()[i, j] * sw[i]


def test_gradients_of_values_that_are_not_numbers(ops):
    """They reach the rows and columns that depend on them, and no others."""
    m, n, k = 100, 72, 66
    rng = np.random.default_rng(6)
    qx, qw = random_q(rng, m, k), random_q(rng, n, k)
    qx[qx == 0], qw[qw == 0] = 1, 1
    one_m, one_n = Q.Array.of(np.ones(m)), Q.Array.of(np.ones(n))
    for dtype, t in TYPES.items():
        dy = stored(rng.normal(0, 1, (m, n)), dtype)
        dy[10, 20], dy[50, 60] = np.inf, np.nan
        dx, dw = Q.Array(m, k, t), Q.Array(n, k, t)
        ops.grad_input(t, Q.Array.of(dy, t), Q.Array.of(qw), one_n, dx, m, n, k)
        ops.grad_weight(t, Q.Array.of(dy, t), Q.Array.of(qx), one_m, t, dw, m, n, k)
        ops.synchronize()
        for got, inf, nan, q in ((dx.numpy(), 10, 50, qw[20]), (dw.numpy(), 20, 60, qx[10])):
            assert np.array_equal(got[inf], np.sign(q.astype(np.float64)) * np.inf), dtype
            assert np.all(np.isnan(got[nan]))
            rest = np.delete(got, [inf, nan], axis=0)
            assert np.all(np.isfinite(rest))


@pytest.mark.parametrize("m,n,k", [(100, 72, 66), (97, 105, 35), (4100, 130, 133), (130, 4100, 133)])
def test_infinities_anywhere_in_a_sum(ops, m, n, k):
    """Also in the values before a sum's last ones, which are loaded with them."""
    rng = np.random.default_rng(16)
    qx, qw = random_q(rng, m, k), random_q(rng, n, k)
    qx[qx == 0], qw[qw == 0] = 1, 1
    one_m, one_n = Q.Array.of(np.ones(m)), Q.Array.of(np.ones(n))
    for dtype, t in TYPES.items():
        for back in (1, 9, 20, 31, 33):
            dy = stored(rng.normal(0, 1, (m, n)), dtype)
            i, j = m - back, n - back
            dy[i, j] = np.inf
            dx, dw = Q.Array(m, k, t), Q.Array(n, k, t)
            ops.grad_input(t, Q.Array.of(dy, t), Q.Array.of(qw), one_n, dx, m, n, k)
            ops.grad_weight(t, Q.Array.of(dy, t), Q.Array.of(qx), one_m, t, dw, m, n, k)
            ops.synchronize()
            for got, row, q in ((dx.numpy(), i, qw[j]), (dw.numpy(), j, qx[i])):
                assert np.array_equal(got[row], np.sign(q.astype(np.float64)) * np.inf), (dtype, back)
                assert np.all(np.isfinite(np.delete(got, row, axis=0)))


@pytest.mark.parametrize("m,n,k", [(100, 72, 66), (4100, 130, 133), (130, 4100, 133)])
def test_scales_that_are_not_numbers_reach_every_sum(ops, m, n, k):
    rng = np.random.default_rng(17)
    qx, qw = random_q(rng, m, k), random_q(rng, n, k)
    qx[m - 2], qw[n - 2] = 0, 0
    sx, sw = np.ones(m), np.ones(n)
    sx[m - 2], sw[n - 2] = np.nan, np.nan
    for dtype, t in TYPES.items():
        dy = Q.Array.of(stored(rng.normal(0, 1, (m, n)), dtype), t)
        dx, dw = Q.Array(m, k, t), Q.Array(n, k, t)
        ops.grad_input(t, dy, Q.Array.of(qw), Q.Array.of(sw), dx, m, n, k)
        ops.grad_weight(t, dy, Q.Array.of(qx), Q.Array.of(sx), t, dw, m, n, k)
        ops.synchronize()
        assert np.all(np.isnan(dx.numpy())) and np.all(np.isnan(dw.numpy()))


def test_operands_past_32_bit_offsets(ops):
    """Rows far apart: the last token's start past 2^32 bytes."""
    m, n, k, ld = 130, 20, 64, 1 << 25
    rng = np.random.default_rng(8)
    for rows in (40, m):      # few tokens, and copied rows
        q = random_q(rng, rows, k)
        far = S.DeviceBuffer((rows - 1) * ld + k)
        for i in range(rows):
            row = np.ascontiguousarray(q[i])
            S._check("sgemm_memcpy_h2d", S.load_library().sgemm_memcpy_h2d(far.ptr + i * ld, row.ctypes.data, k))
        qw, y = random_q(rng, n, k), Q.Array(rows, n, Q.F32)
        ops.gemm(Q.F32, far, Q.Array.of(np.ones(rows)), Q.Array.of(qw), Q.Array.of(np.ones(n)), None, y, rows, n, k, ldx=ld)
        ops.synchronize()
        assert np.array_equal(y.numpy(), (q.astype(np.float64) @ qw.astype(np.float64).T))
        far.close()


# taken as they are, and laid out: the weights' with fewer than eight channels, the input's with fewer than four features
@pytest.mark.parametrize("n,k", [(20, 64), (7, 64), (20, 3)])
def test_gradient_operands_past_32_bit_offsets(ops, n, k):
    """Rows far apart: the last ones start past 2^32 bytes."""
    m, ld = 130, 1 << 25
    rng = np.random.default_rng(18)

    def far(values, size):
        buffer = S.DeviceBuffer((len(values) - 1) * ld * size + values.shape[1] * size)
        for i, row in enumerate(values):
            row = np.ascontiguousarray(row)
            S._check("sgemm_memcpy_h2d", S.load_library().sgemm_memcpy_h2d(buffer.ptr + i * ld * size, row.ctypes.data, row.nbytes))
        return buffer

    q, ones = random_q(rng, m, k), Q.Array.of(np.ones(m))
    dy = rng.integers(-8, 9, (m, n)).astype(np.float64)        # exact products and sums throughout
    wq = far(q, 1)
    dw = Q.Array(n, k, Q.F32)
    ops.grad_weight(Q.F16, Q.Array.of(dy, Q.F16), wq, ones, Q.F32, dw, m, n, k, ldx=ld)
    ops.synchronize()
    assert np.array_equal(dw.numpy(), dy.T @ q)
    # as many channels as there were tokens: the weights' rows are far apart
    dx = Q.Array(n, k, Q.F32)
    ops.grad_input(Q.F32, Q.Array.of(dy.T), wq, ones, dx, n, m, k, ldw=ld)
    ops.synchronize()
    assert np.array_equal(dx.numpy(), dy.T @ q)
    wq.close()
    wdy = far(dy.astype(np.float16), 2)
    ops.grad_weight(Q.F16, wdy, Q.Array.of(q), ones, Q.F32, dw, m, n, k, lddy=ld)
    qw, dx = random_q(rng, n, k), Q.Array(m, k, Q.F16)
    ops.grad_input(Q.F16, wdy, Q.Array.of(qw), Q.Array.of(np.ones(n)), dx, m, n, k, lddy=ld)
    ops.synchronize()
    assert np.array_equal(dw.numpy(), dy.T @ q)
    assert np.array_equal(dx.numpy().astype(np.float64), stored(dy @ qw, "f16"))
    wdy.close()


# both gradients from operands as they are, and the weights' or the input's laid out
@pytest.mark.parametrize("m,n,k", [(300, 200, 4100), (4100, 200, 300), (300, 4100, 200)])
def test_captured_calls_replay(ops, m, n, k):
    """A graph of a training step's calls replays with the bits of the eager calls, also
    after the handle's workspace has been replaced by a larger one."""
    rng = np.random.default_rng(9)
    hip = _Hip()
    stream = hip.stream()
    x, g = Q.Array.of(rng.normal(0, 1, (m, k)), Q.BF16), Q.Array.of(np.ones(k), Q.BF16)
    ldq = Q.row_bytes(k)
    qx, sx, rstd = Q.Array(m, k, "int8", ldq), Q.Array(1, m, Q.F32), Q.Array(1, m, Q.F32)
    qw, sw = Q.Array.of(random_q(rng, n, k), "int8", ldq), Q.Array.of(np.full(n, 0.01))
    dy = Q.Array.of(rng.normal(0, 1, (m, n)), Q.BF16)
    y, dn, dw, dx, dg = (Q.Array(m, n, Q.BF16), Q.Array(m, k, Q.BF16), Q.Array(n, k, Q.BF16), Q.Array(m, k, Q.BF16),
                         Q.Array(1, k, Q.F32))

    def step(o):
        o.rmsnorm(Q.BF16, x, None, g, None, qx, sx, rstd, m, k, ldq=ldq)
        o.gemm(Q.BF16, qx, sx, qw, sw, None, y, m, n, k, ldx=ldq, ldw=ldq)
        o.grad_weight(Q.BF16, dy, qx, sx, Q.BF16, dw, m, n, k, ldx=ldq)
        o.grad_input(Q.BF16, dy, qw, sw, dn, m, n, k, ldw=ldq)
        o.rmsnorm_backward(Q.BF16, dn, x, g, rstd, None, dx, dg, m, k)

    outs = (qx, sx, y, dw, dn, dx, dg)
    with Q.Ops() as o:
        step(o)
        o.synchronize()
        want = [a.numpy().copy() for a in outs]
        need = max(Q.workspace_size(c, Q.BF16, m, n, k) for c in range(4))
    o = Q.Ops()
    try:
        o.set_stream(stream.value)
        hip.begin(stream, 0)
        try:
            with pytest.raises(S.SgemmError) as e:      # nothing is reserved yet
                o.rmsnorm_backward(Q.BF16, dn, x, g, rstd, None, dx, dg, m, k)
            assert e.value.code == -4 and "q8_reserve" in e.value.message
        finally:
            _ok(hip.lib.hipGraphExecDestroy(hip.end(stream)))
        o.reserve(need)
        hip.begin(stream, 0)
        try:
            step(o)
        finally:
            exe = hip.end(stream)
        for _ in range(3):
            for a in outs:
                S._check("sgemm_memset", S.load_library().sgemm_memset(a.ptr, 0x11, a.nbytes))
            _ok(hip.lib.hipGraphLaunch(exe, stream))
            o.synchronize()
            assert all(np.array_equal(a.numpy(), b) for a, b in zip(outs, want))
            step(o)     # eager, between the replays
            o.synchronize()
            assert all(np.array_equal(a.numpy(), b) for a, b in zip(outs, want))
            need *= 2
            o.reserve(need)
        _ok(hip.lib.hipGraphExecDestroy(exe))
    finally:
        o.set_stream(None)
        o.close()
        hip.lib.hipStreamDestroy(stream)
