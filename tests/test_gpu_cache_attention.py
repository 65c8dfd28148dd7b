"""Attention of new tokens over the paged cache, against float64."""
import numpy as np
import pytest

from cache_reference import Case
from q8_reference import TYPES, Window, stored
from shim import q8_cache as C

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    with C.Ops() as o:
        yield o


def check(ops, rng, case, dtype, window=0, scale=None, pad=0, shift=0, spread=1.0, q=None, lse=True):
    kind, cols = TYPES[dtype], case.heads * case.dim
    if q is None:
        q = stored(rng.normal(0, spread, (case.tokens, cols)), dtype)
    cache, batch = case.upload()
    wq, wo = Window(case.tokens, cols, kind, pad, shift, q), Window(case.tokens, cols, kind, pad, shift)
    wl = Window(1, case.tokens * case.heads, C.F32) if lse else None
    ops.attention(kind, cache, batch, case.heads, wq, wo, wl, scale=scale, window=window, ldq=wq.ld, ldo=wo.ld)
    ops.synchronize()
    out, want_lse, sums = case.attention(q, case.dim ** -0.5 if scale is None else scale, window)
    off, off_lse = case.bounds(out, want_lse, sums, dtype)
    got = wo.values().reshape(case.tokens, case.heads, case.dim)
    mine = np.zeros(case.tokens, bool)
    for _, token, _ in case.rows():
        mine[token] = True
    assert np.all(got[~mine] == 85), "rows of no chunk changed"
    wrong = np.abs(got - out) > off
    wrong[~mine] = False
    assert np.all(np.isfinite(got[mine])) and not wrong.any(), (
        f"{int(wrong.sum())} of {wrong.size} wrong, the first at {np.argwhere(wrong)[0]}: {got[tuple(np.argwhere(wrong)[0])]} "
        f"for {out[tuple(np.argwhere(wrong)[0])]}, {np.nanmax(np.abs(got - out)[mine] / off[mine])} times the bound")
    if lse:
        got = wl.values().reshape(case.tokens, case.heads)
        assert np.all(got[~mine] == 85)
        empty = np.isinf(want_lse)
        assert np.all(np.isneginf(got[mine & True][empty[mine]]))
        fine = mine[:, None] & ~empty
        assert np.all(np.abs(got[fine] - want_lse[fine]) <= off_lse[fine])


DECODING = [(1, 300), (1, 1), (1, 64), (1, 65), (1, 517), (1, 31), (1, 2)]
CHUNKS = [(70, 190), (33, 33), (1, 129), (130, 131), (2, 64), (5, 260)]
PROMPTS = [(257, 257), (64, 64), (1, 1), (40, 40)]
ODD = [(0, 10), (9, 4), (3, 0), (0, 0), (4, 200), (0, 7)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 2, 128, 16), (4, 4, 64, 16), (5, 1, 80, 24), (16, 1, 256, 7), (3, 3, 33, 1),
                                                     (6, 2, 1, 64), (40, 2, 96, 16), (2, 1, 192, 32)])
@pytest.mark.parametrize("sequences", [DECODING, CHUNKS, PROMPTS, ODD], ids=["decoding", "chunks", "prompts", "odd"])
def test_attention(ops, dtype, heads, kv_heads, dim, page, sequences):
    rng = np.random.default_rng(dim * 7 + heads)
    case = Case(rng, sequences, heads, kv_heads, dim, page, extra_rows=3, front_rows=2, width_more=1, ld_more=1)
    check(ops, rng, case, dtype, pad=3, shift=1)


@pytest.mark.parametrize("window", [1, 2, 31, 64, 100, 129, 5000, 2 ** 32 - 1])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_windows(ops, dtype, window):
    rng = np.random.default_rng(window % 1000)
    case = Case(rng, [(1, 300), (150, 420), (9, 4), (64, 64)], 4, 2, 64, 16)
    check(ops, rng, case, dtype, window=window)


@pytest.mark.parametrize("longest", [0, 1, 16, 400, 2 ** 32 - 1])
@pytest.mark.parametrize("sequences", [[(1, 700), (1, 40)], [(200, 400), (1, 700)], [(17, 90)]])
def test_any_longest_gives_the_same(ops, longest, sequences):
    rng = np.random.default_rng(5)
    case = Case(rng, sequences, 8, 2, 128, 16, longest=longest)
    check(ops, rng, case, "bf16")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("sequences", [[(1, 2500)], [(1, 5000), (1, 3), (1, 1200)], [(3, 4000), (2, 2)], [(90, 3000)]])
def test_long_caches(ops, dtype, sequences):
    rng = np.random.default_rng(6)
    check(ops, rng, Case(rng, sequences, 8, 2, 128, 16), dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("sequences", [[(1, 300), (1, 90), (1, 20)], [(130, 300), (40, 90)]])
def test_pages_that_are_not_there(ops, dtype, sequences):
    """Their keys are left out; a sequence with none of its pages has rows of zeros."""
    rng = np.random.default_rng(7)
    case = Case(rng, sequences, 4, 1, 64, 8)
    case.table[0, :30:3] = -1
    case.table[0, 5] = case.pages
    case.table[0, 7] = -2 ** 31
    case.table[1, :] = 2 ** 31 - 1
    check(ops, rng, case, dtype)
    case.table[0, :] = -7
    check(ops, rng, case, dtype, window=9)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("sequences", [[(1, 37), (1, 100)], [(35, 37), (70, 100)]])
def test_what_is_not_seen_has_no_effect(ops, dtype, sequences):
    """NaN, infinite and huge scales behind the sequences, in other pages and before the window."""
    rng = np.random.default_rng(8)
    case = Case(rng, sequences, 4, 2, 64, 16)
    seen = np.zeros(case.sk.shape, bool)
    window = 20
    first = {b: min([p for x, _, p in case.rows() if x == b]) for b in range(2)}
    for b, (_, length) in enumerate(case.sequences):
        for p in range(max(0, first[b] - window + 1), length):
            page, slot = case.place(b, p)
            seen[page, :, slot] = True
    bad = np.array([np.nan, np.inf, -np.inf, 3e38], np.float32)
    for s in (case.sk, case.sv):
        s[~seen] = bad[np.arange((~seen).sum()) % 4]
    case.k[~seen] = case.v[~seen] = -128
    check(ops, rng, case, dtype, window=window)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("sequences", [[(1, 40), (1, 90)], [(30, 40), (60, 90)]])
@pytest.mark.parametrize("where", ["k", "v", "q"])
def test_nan_reaches_the_rows_that_see_it(ops, dtype, sequences, where):
    rng = np.random.default_rng(9)
    case = Case(rng, sequences, 4, 2, 64, 16)
    q = stored(rng.normal(0, 1, (case.tokens, 256)), dtype)
    page, slot = case.place(0, 25)
    if where == "q":
        q[0, 70] = np.nan
    else:
        (case.sk if where == "k" else case.sv)[page, 1, slot] = np.nan
    cache, batch = case.upload()
    out = C.Array(case.tokens, 256, TYPES[dtype])
    ops.attention(TYPES[dtype], cache, batch, 4, C.Array.of(q, TYPES[dtype]), out)
    ops.synchronize()
    got = np.isnan(out.numpy().reshape(case.tokens, 4, 64))
    for b, token, p in case.rows():
        for h in range(4):
            hit = (token, h) == (0, 1) if where == "q" else b == 0 and p >= 25 and h >= 2
            assert np.all(got[token, h] == hit), (token, h)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("sequences", [[(1, 300)], [(60, 300)]])
def test_large_and_small_scores_and_values(ops, dtype, sequences):
    """Scores that leave one key, scores of hundreds below zero that grow along the keys, a scale below zero; values of very
    different size."""
    rng = np.random.default_rng(10)
    case = Case(rng, sequences, 4, 2, 64, 16)
    check(ops, rng, case, dtype, spread=20.0)
    check(ops, rng, case, dtype, scale=-0.3)
    check(ops, rng, case, dtype, scale=0.0)
    for p in range(300):        # keys along one direction, larger and larger, and of the other sign in the first half
        page, slot = case.place(0, p)
        case.k[page, :, slot, :64] = 100
        case.sk[page, :, slot] = (1 + p) / 3000
    q = stored(rng.normal(0, 0.1, (case.tokens, 256)) + 1, dtype)
    check(ops, rng, case, dtype, q=q)
    check(ops, rng, case, dtype, q=-q)
    case.sv *= np.exp2(rng.integers(-60, 9, case.sv.shape)).astype(np.float32)
    check(ops, rng, case, dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** 60])
def test_scales_far_from_one(ops, dtype, scale):
    if dtype == "f16":
        pytest.skip("results of that size are no F16 values")
    rng = np.random.default_rng(11)
    case = Case(rng, [(1, 200), (40, 200)], 4, 2, 64, 16, scale=scale)
    check(ops, rng, case, dtype)


def test_without_lse_and_without_rows(ops):
    rng = np.random.default_rng(12)
    case = Case(rng, [(1, 20), (20, 40)], 4, 2, 64, 16)
    check(ops, rng, case, "bf16", lse=False)
    cache, batch = case.upload()
    empty = C.Batch(*batch.memory, 0, 0, case.width)
    ops.attention(C.BF16, cache, empty, 4, None, None)
    ops.cache_write(C.BF16, cache, empty, None, None)
    ops.cache_read(C.BF16, cache, empty, None, None)
    none = C.Batch(*batch.memory, 2, case.tokens, 0)      # no pages: every row is zeros
    q, out, lse = C.Array(case.tokens, 256, C.BF16), C.Array.of(np.ones((case.tokens, 256)), C.BF16), C.Array(1, case.tokens * 4, C.F32)
    ops.attention(C.BF16, cache, none, 4, q, out, lse)
    ops.synchronize()
    assert not out.numpy().any() and np.all(np.isneginf(lse.numpy()))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim,page,window", [(128, 16, 0), (128, 7, 100), (64, 64, 0), (33, 16, 300), (256, 16, 90)])
def test_many_rows(ops, dtype, dim, page, window):
    """Rows from which on the keys are laid out beforehand (dim up to 128); pages that are not there, a whole step of keys among
    them; nothing of a sequence's; a chunk longer than its sequence."""
    rng = np.random.default_rng(13)
    case = Case(rng, [(300, 700), (0, 9), (250, 250), (270, 200)], 16, 2, dim, page, extra_rows=1, front_rows=1, width_more=1)
    case.table[0, 3] = -1
    case.table[0, -(-128 // page): -(-330 // page)] = case.pages
    case.table[3, :] = -1
    bad = rng.random(case.sk.shape) < 0.5       # behind the sequences
    used = np.zeros(case.sk.shape, bool)
    for b, (_, length) in enumerate(case.sequences):
        for p in range(length):
            at = case.place(b, p)
            if at:
                used[at[0], :, at[1]] = True
    case.sk[bad & ~used] = np.nan
    case.sv[bad & ~used] = np.inf
    check(ops, rng, case, dtype, window=window)
