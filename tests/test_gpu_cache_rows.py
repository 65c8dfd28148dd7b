"""Rotary positions, and keys and values into the paged cache and back, against float64."""
import numpy as np
import pytest

from cache_reference import Case, angles, rotary
from q8_reference import LEAST_SCALE, TINY, UNIT, TYPES, Window, stored
from shim import q8_cache as C

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    with C.Ops() as o:
        yield o


def turn(ops, rng, dtype, tokens, heads, dim, pairs, axes=1, neighbours=False, inverse=False, pad=0, shift=0, far=5000, in_place=False):
    kind = TYPES[dtype]
    x = stored(rng.normal(0, 1, (tokens, heads * dim)), dtype)
    positions = rng.integers(-far // 10, far, (axes, tokens + 2)).astype(np.int32)
    axis = [int(a) for a in rng.integers(0, axes, pairs)]
    freq = (1e4 ** -(np.arange(pairs) / max(1, pairs))).astype(np.float32)
    form = C.Rotation(dim, axis, axes, neighbours)
    wx = Window(tokens, heads * dim, kind, pad, shift, x)
    wy = wx if in_place else Window(tokens, heads * dim, kind, pad, shift)
    f = C.Array.of(freq) if pairs else None
    ops.rotary(kind, form, wx, C.ints(positions), f, wy, tokens, heads, ldx=wx.ld, ldp=tokens + 2, ldy=wy.ld, inverse=inverse)
    ops.synchronize()
    got = wy.values().reshape(tokens, heads, dim)
    x = x.reshape(tokens, heads, dim)
    want = rotary(x, angles(positions[:, :tokens], axis, freq), neighbours, inverse)
    # sine and cosine: the rounded rest of the angle (2^-24 of at most pi / 4) and the functions' last place, 2^-22 in all;
    # two products and a sum, each rounded once
    size = np.zeros_like(x)
    one, two = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if neighbours else (slice(0, pairs), slice(pairs, 2 * pairs))
    size[:, :, one] = size[:, :, two] = np.abs(x[:, :, one]) + np.abs(x[:, :, two])
    off = size * (2.0 ** -22 + 2.0 ** -23)
    assert np.all(np.abs(got - want) <= off + (np.abs(want) + off) * UNIT[dtype] + TINY[dtype])
    if 2 * pairs < dim:
        assert np.array_equal(got[:, :, 2 * pairs:], x[:, :, 2 * pairs:])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,pairs", [(1, 1, 2, 1), (1, 40, 128, 64), (37, 5, 80, 40), (3, 7, 33, 16), (5, 3, 96, 13),
                                                    (1100, 3, 72, 36), (2, 2, 256, 128), (9, 4, 256, 100), (1, 600, 64, 32)])
def test_rotary(ops, dtype, neighbours, tokens, heads, dim, pairs):
    rng = np.random.default_rng(tokens * 1000 + dim)
    turn(ops, rng, dtype, tokens, heads, dim, pairs, axes=3, neighbours=neighbours)
    turn(ops, rng, dtype, tokens, heads, dim, pairs, neighbours=neighbours, inverse=True, pad=5, shift=3, in_place=True)


@pytest.mark.parametrize("pairs,dim", [(0, 8), (0, 1), (1, 3), (4, 8), (7, 14), (8, 17)])
def test_rotary_of_few_pairs(ops, pairs, dim):
    rng = np.random.default_rng(pairs)
    for neighbours in (False, True):
        turn(ops, rng, "f32", 19, 3, dim, pairs, axes=8, neighbours=neighbours, pad=1, shift=1)
        turn(ops, rng, "bf16", 19, 3, dim, pairs, neighbours=neighbours, in_place=True)


def test_far_positions(ops):
    """Angles of 2^31 and of the frequencies 1 and 1/10000 there: the whole turns are taken off exactly."""
    rng = np.random.default_rng(3)
    positions = np.array([[0, 1, -1, 1_000_003, 2 ** 31 - 1, -2 ** 31, 123456789]], np.int32)
    freq = np.array([1.0, 0.7071067, 1e-4, 3.1415927], np.float32)
    x = rng.normal(0, 1, (7, 8)).astype(np.float32).astype(np.float64)
    dx, y = C.Array.of(x, C.F32), C.Array(7, 8, C.F32)
    form = C.Rotation(8, [0] * 4)
    ops.rotary(C.F32, form, dx, C.ints(positions), C.Array.of(freq), y, 7, 1)
    ops.synchronize()
    # the exact product's residue, with integers: position * freq has 55 bits, 2 pi is taken to 80
    two_pi = 2 * 3141592653589793238462643383279502884197 * 10 ** 40
    unit = 10 ** 79
    angle = np.zeros((7, 4))
    for i, p in enumerate(positions[0]):
        for j, f in enumerate(freq):
            num, den = float(f).as_integer_ratio()
            exact = int(p) * num * unit // den
            angle[i, j] = (exact % two_pi) / unit
    want = rotary(x.reshape(7, 1, 8), angle, False, False).reshape(7, 8)
    size = np.abs(x[:, :4]) + np.abs(x[:, 4:])
    assert np.all(np.abs(y.numpy() - want) <= np.tile(size, 2) * (2.0 ** -22 + 2.0 ** -23) + np.abs(want) * 2.0 ** -24)


def test_gradient_is_the_inverse_turn(ops):
    """Against differences: d(sum w y) / dx, w any, by moving each value of one token."""
    rng = np.random.default_rng(4)
    dim, form = 12, C.Rotation(12, [0, 1, 0, 1], 2, True)
    positions, freq = C.ints(np.array([[17], [5]])), C.Array.of(np.array([1.0, 0.3, 0.1, 0.03], np.float32))
    x, w = rng.normal(0, 1, (1, dim)), rng.normal(0, 1, (1, dim))
    y, g = C.Array(1, dim, C.F32), C.Array(1, dim, C.F32)
    ops.rotary(C.F32, form, C.Array.of(w, C.F32), positions, freq, g, 1, 1, inverse=True)

    def loss(x):
        ops.rotary(C.F32, form, C.Array.of(x, C.F32), positions, freq, y, 1, 1)
        ops.synchronize()
        return float((w * y.numpy().astype(np.float64)).sum())

    got = g.numpy()[0]
    for d in range(dim):
        step = np.zeros((1, dim))
        step[0, d] = 1.0
        # the turn is linear: a difference of any step is the derivative, here of 2 with 2^-21 of its values' size
        assert abs((loss(x + step) - loss(x - step)) / 2 - got[d]) <= 2.0 ** -19 * np.abs(w).sum()


SEQUENCES = {
    "decoding": [(1, 5), (1, 33), (1, 1), (1, 64)],
    "chunks": [(7, 20), (16, 16), (33, 70), (1, 2)],
    "empty ones": [(0, 5), (3, 3), (0, 0), (0, 9), (5, 21), (0, 1)],
    "longer than their sequence": [(9, 4), (2, 7), (3, 0)],
    "one": [(1, 1)],
}


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim,page,kv_heads", [(128, 16, 8), (64, 5, 3), (33, 24, 1), (256, 1, 2), (80, 64, 5), (1, 3, 2)])
@pytest.mark.parametrize("name", list(SEQUENCES))
def test_cache(ops, dtype, dim, page, kv_heads, name):
    rng = np.random.default_rng(dim + page)
    kind = TYPES[dtype]
    case = Case(rng, SEQUENCES[name], kv_heads, kv_heads, dim, page, extra_rows=3, front_rows=2, width_more=1, ld_more=2)
    case.table[0, 0] = case.pages        # one page that is not there
    cols = kv_heads * dim
    k, v = (stored(rng.normal(0, 3, (case.tokens, cols)) * np.exp(rng.normal(0, 2, (case.tokens, 1))), dtype) for _ in range(2))
    if case.tokens > 8:
        k[4] = 0
        v[5, 0] = np.nan
        k[6, cols - 1] = np.inf
    cache, batch = case.upload()
    wk, wv = Window(case.tokens, cols, kind, 3, 1, k), Window(case.tokens, cols, kind, 5, 2, v)
    ops.cache_write(kind, cache, batch, wk, wv, ldk=wk.ld, ldv=wv.ld)
    ops.synchronize()
    got = case.download()
    left = [np.ones(a.shape, bool) for a in got]
    back = {"k": np.full((case.tokens, cols), 85.0), "v": np.full((case.tokens, cols), 85.0)}
    for b, token, p in case.rows():
        at = case.place(b, p)
        for name_, x, q, s, i in (("k", k, got[0], got[2], 0), ("v", v, got[1], got[3], 1)):
            if at is None:
                back[name_][token] = 0
                continue
            page_, slot = at
            left[i][page_, :, slot] = left[i + 2][page_, :, slot] = False
            for h in range(kv_heads):
                row, steps, scale = x[token, h * dim:(h + 1) * dim], q[page_, h, slot], s[page_, h, slot]
                assert not steps[dim:].any()
                steps = steps[:dim].astype(np.float64)
                if not np.all(np.isfinite(row)):
                    assert np.isnan(scale) and not steps.any()
                else:
                    want = max(np.abs(row).max() / 127, LEAST_SCALE)
                    assert abs(scale - want) <= want * 2.0 ** -23
                    exact = row / want
                    # rounded to nearest; the quotient is off by three roundings, 128 * 3 * 2^-24
                    assert np.all(np.abs(steps - exact) <= 0.5 + 128 * 3 * 2.0 ** -24)
                back[name_][token, h * dim:(h + 1) * dim] = steps * np.float64(scale)
    for now, before, kept in zip(got, (case.k, case.v, case.sk, case.sv), left):
        assert np.array_equal(now[kept], before[kept])
    for read in {dtype, "bf16"}:
        rk, rv = Window(case.tokens, cols, TYPES[read], 1, 3), Window(case.tokens, cols, TYPES[read], 0, 0)
        ops.cache_read(TYPES[read], cache, batch, rk, rv, ldk=rk.ld, ldv=rv.ld)
        ops.synchronize()
        for window, want in ((rk, back["k"]), (rv, back["v"])):
            values = window.values()
            assert np.array_equal(np.isnan(values), np.isnan(want))
            with np.errstate(over="ignore"):    # what passes the type's range is infinite in both
                assert np.array_equal(np.nan_to_num(values, nan=0.0), np.nan_to_num(stored(want, read), nan=0.0))


def test_many_sequences_and_tokens(ops):
    """More sequences than a work-group has threads, and more tokens than one takes."""
    rng = np.random.default_rng(9)
    sequences = [(int(c), int(c + t)) for c, t in zip(rng.integers(0, 12, 1500), rng.integers(0, 9, 1500))]
    case = Case(rng, sequences, 2, 2, 32, 4)
    k, v = (stored(rng.normal(0, 1, (case.tokens, 64)), "bf16") for _ in range(2))
    cache, batch = case.upload()
    rk, rv = C.Array(case.tokens, 64, C.F32), C.Array(case.tokens, 64, C.F32)
    ops.cache_write(C.BF16, cache, batch, C.Array.of(k, C.BF16), C.Array.of(v, C.BF16))
    ops.cache_read(C.F32, cache, batch, rk, rv)
    ops.synchronize()
    for x, r in ((k, rk.numpy()), (v, rv.numpy())):
        x, r = x.reshape(-1, 32), r.reshape(-1, 32)
        assert np.all(np.abs(r - x) <= np.abs(x).max(1, keepdims=True) / 127 * 0.5001)


def test_starts_outside_the_rows_are_cut(ops):
    rng = np.random.default_rng(10)
    case = Case(rng, [(4, 9), (5, 12)], 1, 1, 16, 4)
    before = case.starts.copy()
    case.starts = np.array([-2, 4, 30])
    k = stored(rng.normal(0, 1, (case.tokens, 16)), "f32")
    cache, batch = case.upload()
    rk, rv = C.Array(case.tokens, 16, C.F32), C.Array(case.tokens, 16, C.F32)
    d = C.Array.of(k, C.F32)
    ops.cache_write(C.F32, cache, batch, d, d)
    ops.cache_read(C.F32, cache, batch, rk, rv)
    ops.synchronize()
    assert case.tokens == before[-1] == 9
    q = case.download()[0]
    for b, token, p in case.rows():
        page, slot = case.place(b, p)
        assert np.abs(q[page, 0, slot, :16] - k[token] * 127 / np.abs(k[token]).max()).max() <= 0.5001
    assert np.all(np.abs(rk.numpy() - k) <= np.abs(k).max(1, keepdims=True) / 127 * 0.5001)
