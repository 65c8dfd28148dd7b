"""Quantisation, the norm with its 8-bit result, its gradients and the restoring, against float64.

Tolerances.  A row's sums take at most 8 R + 10 additions one after the other (R
pieces of eight values a thread, up to five here), so they are within 50 * 2^-24
of the sum of magnitudes; results add a rounding to their type.
"""
import numpy as np
import pytest

from q8_reference import TINY, TYPES, UNIT, Window, norm, norm_backward, scales, stored
from shim import q8_shim as Q

pytestmark = pytest.mark.gpu

SUM = 50 * 2.0 ** -24
# one value, odd, the sizes at which another kernel takes over, and past them
COLS = [1, 7, 8, 129, 512, 513, 1000, 1024, 1025, 2049, 4096, 4097, 8200, 16384, 16391]
LONG = [32768, 32776, 40001]


@pytest.fixture(scope="module")
def ops():
    with Q.Ops() as o:
        yield o


def _data(rows, cols, dtype, seed):
    rng = np.random.default_rng(seed)
    x = rng.normal(0, 1, (rows, cols)) * np.exp(rng.normal(0, 0.5, (rows, 1)))
    if rows > 2:
        x[1] = 0
    return stored(x, dtype), rng


def _check_q(q, s, n):
    """q s is n to within half a step and what the scale's rounding moves."""
    assert np.abs(q).max(initial=0) <= 127
    assert np.all(np.abs(s - scales(n)) <= 2 * SUM * scales(n))
    assert np.all(np.abs(q * s[:, None] - n) <= s[:, None] * (0.5 + 127 * 3 * SUM))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cols,pad,shift", [(c, 0, 0) for c in COLS] + [(c, 3, 1) for c in (1, 129, 1000, 4096)] +
                         [(c, 0, 0) for c in LONG])
def test_quantize_and_restore(ops, dtype, cols, pad, shift):
    rows = 5
    x, _ = _data(rows, cols, dtype, 11)
    dx = Window(rows, cols, TYPES[dtype], pad, shift, x)
    q, s, y = Window(rows, cols, "int8", pad, shift), Window(1, rows, Q.F32), Window(rows, cols, TYPES[dtype], pad, shift)
    ops.quantize(TYPES[dtype], dx, q, s, rows, cols, ldx=dx.ld, ldq=q.ld)
    ops.dequantize(TYPES[dtype], q, s, y, rows, cols, ldq=q.ld, ldy=y.ld)
    ops.synchronize()
    qv, sv = q.values(), s.values()[0]
    _check_q(qv, sv, x)
    want = stored((qv * sv[:, None]).astype(np.float32), dtype)
    assert np.array_equal(y.values(), want)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cols,pad,shift,residual,keep", [(c, 0, 0, True, True) for c in COLS] +
                         [(c, 5, 1, c % 2 == 0, True) for c in (7, 1000, 4096, 8200)] +
                         [(c, 0, 0, False, False) for c in (8, 1025)] +
                         [(c, 1, 0, True, k) for c in LONG for k in (True, False)])
def test_norm(ops, dtype, cols, pad, shift, residual, keep):
    rows, t, eps = 6, TYPES[dtype], 1e-5
    x, rng = _data(rows, cols, dtype, 12)
    r = stored(rng.normal(0, 1, (rows, cols)), dtype) if residual else None
    if r is not None:
        r[1] = 0
    g = stored(1 + 0.2 * rng.normal(0, 1, cols), dtype)
    wx, wg = Window(rows, cols, t, pad, shift, x), Window(1, cols, t, 0, shift, g[None])
    wr = Window(rows, cols, t, pad, 0, r) if residual else None
    wh = Window(rows, cols, t, 0, shift) if keep else None
    q, s = Window(rows, cols, "int8", pad, shift), Window(1, rows, Q.F32)
    rstd = Window(1, rows, Q.F32) if keep else None
    ops.rmsnorm(t, wx, wr, wg, wh, q, s, rstd, rows, cols, eps, ldx=wx.ld, ldr=wx.ld, ldh=cols, ldq=q.ld)
    ops.synchronize()
    h = stored(x + (r if residual else 0), dtype)    # the sums here are exact in float32 or rounded alike
    n, want_rstd = norm(h, g, eps)
    if keep:
        got = wh.values()
        assert np.all(np.abs(got - (x + (r if residual else 0))) <= 1.0001 * UNIT[dtype] * np.abs(h) + TINY[dtype])
        n, want_rstd = norm(got, g, eps)
        assert np.all(np.abs(rstd.values()[0] - want_rstd) <= SUM * want_rstd)
    _check_q(q.values(), s.values()[0], n)


def test_norm_in_place(ops):
    rows, cols = 3, 1000
    x, rng = _data(rows, cols, "bf16", 13)
    r = stored(rng.normal(0, 1, (rows, cols)), "bf16")
    g = Q.Array.of(np.ones(cols), Q.BF16)
    outs = []
    for which in ("apart", "x", "residual"):
        wx, wr = Window(rows, cols, Q.BF16, values=x), Window(rows, cols, Q.BF16, values=r)
        wh = {"apart": Window(rows, cols, Q.BF16), "x": wx, "residual": wr}[which]
        q, s = Window(rows, cols, "int8"), Window(1, rows, Q.F32)
        ops.rmsnorm(Q.BF16, wx, wr, g, wh, q, s, None, rows, cols)
        ops.synchronize()
        outs.append((wh.values(), q.values(), s.values()))
    for o in outs[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(o, outs[0]))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_values_that_are_not_numbers_stay_in_their_row(ops, dtype):
    rows, cols, t = 6, 700, TYPES[dtype]
    x, _ = _data(rows, cols, dtype, 14)
    x[0, 3], x[2, 699], x[4, 0] = np.inf, np.nan, -np.inf
    wx = Window(rows, cols, t, values=x)
    q, s, y = Window(rows, cols, "int8"), Window(1, rows, Q.F32), Window(rows, cols, t)
    g = Q.Array.of(np.ones(cols), t)
    for norm_too in (False, True):
        if norm_too:
            ops.rmsnorm(t, wx, None, g, None, q, s, None, rows, cols)
        else:
            ops.quantize(t, wx, q, s, rows, cols)
        ops.dequantize(t, q, s, y, rows, cols)
        ops.synchronize()
        bad = np.array([True, False, True, False, True, False])
        assert np.array_equal(np.isnan(s.values()[0]), bad)
        assert np.all(q.values()[bad] == 0) and np.all(np.isnan(y.values()[bad]))
        assert np.all(np.isfinite(y.values()[~bad]))


@pytest.mark.parametrize("top", [0.0, 1e-45, 1e-40, 2.0 ** -126, 1e-36, 1e-30, 1e30, 3.3e38])
def test_scales_of_extreme_rows(ops, top):
    x = np.full((2, 64), top, dtype=np.float32)
    x[:, ::2] *= -1
    x[:, 5] = 0
    wx, q, s = Window(2, 64, Q.F32, values=x), Window(2, 64, "int8"), Window(1, 2, Q.F32)
    ops.quantize(Q.F32, wx, q, s, 2, 64)
    ops.synchronize()
    _check_q(q.values(), s.values()[0], x.astype(np.float64))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols,pad,shift,res", [(1, 1, 0, 0, True), (1, 4096, 0, 0, False), (3, 7, 0, 0, True),
                                                     (300, 512, 0, 0, True), (1000, 999, 5, 0, True),
                                                     (2500, 130, 3, 1, False), (33, 1025, 0, 0, True),
                                                     (70, 4097, 0, 1, True), (40, 8200, 1, 0, False),
                                                     (9, 16384, 0, 0, True), (1030, 16400, 0, 0, True)])
def test_norm_backward(ops, dtype, rows, cols, pad, shift, res):
    t = TYPES[dtype]
    h, rng = _data(rows, cols, dtype, 15)
    dn = stored(0.1 * rng.normal(0, 1, (rows, cols)), dtype)
    if rows > 4:
        dn[3] = 0
    g = stored(1 + 0.2 * rng.normal(0, 1, cols), dtype)
    rstd = stored(1 / np.sqrt((h ** 2).mean(axis=1) + 1e-5), "f32")
    d = stored(0.1 * rng.normal(0, 1, (rows, cols)), dtype) if res else None
    wdn, wh, wg = (Window(rows, cols, t, pad, shift, dn), Window(rows, cols, t, 0, shift, h),
                   Window(1, cols, t, 0, 0, g[None]))
    wd = Window(rows, cols, t, pad, 0, d) if res else None
    wr, wx, wgain = Window(1, rows, Q.F32, values=rstd[None]), Window(rows, cols, t, pad, shift), Window(1, cols, Q.F32)
    runs = []
    for _ in range(2):
        ops.rmsnorm_backward(t, wdn, wh, wg, wr, wd, wx, wgain, rows, cols, lddn=wdn.ld, ldh=cols, lddr=wdn.ld, lddx=wx.ld)
        ops.synchronize()
        runs.append((wx.values(), wgain.values()[0]))
    assert np.array_equal(runs[0][0], runs[1][0]) and np.array_equal(runs[0][1], runs[1][1])
    dx, dgain = norm_backward(dn, h, g, rstd, d)
    xhat = h * rstd[:, None]
    size = rstd[:, None] * (np.abs(dn * g) + np.abs(xhat) * np.abs(dn * g * xhat).mean(axis=1, keepdims=True))
    bound = UNIT[dtype] * np.abs(dx) + SUM * (size + (0 if d is None else np.abs(d))) + TINY[dtype]
    assert np.all(np.abs(runs[0][0] - dx) <= bound)
    # at most a row range's rows, its share of the ranges, and 20 more additions
    adds = rows / min(rows, 512) + min(rows, 1024) / 16 + 20
    assert np.all(np.abs(runs[0][1] - dgain) <= adds * 2.0 ** -24 * np.abs(dn * xhat).sum(axis=0))


def test_norm_backward_against_differences(ops):
    rows, cols, eps = 4, 24, 1e-5
    rng = np.random.default_rng(16)
    x, g, c = rng.normal(0, 1, (rows, cols)), 1 + 0.2 * rng.normal(0, 1, cols), rng.normal(0, 1, (rows, cols))
    x, g, c = (stored(a, "f32") for a in (x, g, c))
    _, rstd = norm(x, g, eps)
    dx, dgain = Q.Array(rows, cols, Q.F32), Q.Array(1, cols, Q.F32)
    ops.rmsnorm_backward(Q.F32, Q.Array.of(c), Q.Array.of(x), Q.Array.of(g), Q.Array.of(rstd), None, dx, dgain, rows, cols)
    ops.synchronize()

    def loss(x, g):
        return (norm(x, g, eps)[0] * c).sum()

    step = 1e-4    # central differences in float64: 1e-8 of curvature, 1e-11 of rounding
    for i in range(rows):
        for j in range(cols):
            e = np.zeros((rows, cols))
            e[i, j] = step
            assert abs((loss(x + e, g) - loss(x - e, g)) / (2 * step) - dx.numpy()[i, j]) < 1e-5
    for j in range(cols):
        e = np.zeros(cols)
        e[j] = step
        assert abs((loss(x, g + e) - loss(x, g - e)) / (2 * step) - dgain.numpy()[0, j]) < 1e-5


@pytest.mark.parametrize("which", ["dn", "dres"])
@pytest.mark.parametrize("cols", [1000, 16400])
def test_norm_backward_in_place(ops, which, cols):
    rows = 5
    h, rng = _data(rows, cols, "bf16", 17)
    dn, d = (stored(rng.normal(0, 1, (rows, cols)), "bf16") for _ in range(2))
    g, r = Q.Array.of(np.ones(cols), Q.BF16), Q.Array.of(np.ones(rows))
    wh, outs = Window(rows, cols, Q.BF16, values=h), []
    for place in (None, which):
        wdn, wd = Window(rows, cols, Q.BF16, values=dn), Window(rows, cols, Q.BF16, values=d)
        wx = {None: Window(rows, cols, Q.BF16), "dn": wdn, "dres": wd}[place]
        wgain = Window(1, cols, Q.F32)
        ops.rmsnorm_backward(Q.BF16, wdn, wh, g, r, wd, wx, wgain, rows, cols)
        ops.synchronize()
        outs.append((wx.values(), wgain.values()))
    assert all(np.array_equal(a, b) for a, b in zip(*outs))


def test_no_rows(ops):
    x, s, gain = Q.Array(1, 64, Q.F32), Q.Array(1, 64, Q.F32), Q.Array.of(np.full(64, 7.0))
    q = Q.Array(1, 64, "int8")
    ops.quantize(Q.F32, x, q, s, 0, 64)
    ops.rmsnorm(Q.F32, x, None, gain, None, q, s, None, 0, 64)
    ops.dequantize(Q.F32, q, s, x, 0, 64)
    ops.rmsnorm_backward(Q.F32, None, None, s, None, None, None, gain, 0, 64)    # a sum over no rows
    ops.synchronize()
    assert np.all(gain.numpy() == 0)


def test_many_short_rows(ops):
    rows = (1 << 20) * 4 + 77    # more than the work-groups of a launch have at once
    x = np.arange(rows * 2, dtype=np.float32).reshape(rows, 2) % 1009 - 500
    wx, q, s, y = Q.Array.of(x), Q.Array(rows, 2, "int8"), Q.Array(1, rows, Q.F32), Q.Array(rows, 2, Q.F32)
    ops.quantize(Q.F32, wx, q, s, rows, 2)
    ops.dequantize(Q.F32, q, s, y, rows, 2)
    ops.synchronize()
    sv = s.numpy()[0].astype(np.float64)
    _check_q(q.numpy().astype(np.float64), sv, x.astype(np.float64))
    assert np.all(np.abs(y.numpy() - x) <= 0.501 * sv[:, None])
