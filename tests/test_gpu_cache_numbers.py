"""Attention where its arithmetic could leave FP32 or half precision, against float64: value scales of zero and far from one
another, sums of very different weights, scores of any size."""
import numpy as np
import pytest

from cache_reference import Case
from q8_reference import TINY, TYPES, UNIT, stored
from shim import q8_cache as C
from test_gpu_cache_attention import check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    with C.Ops() as o:
        yield o


class Numbers(Case):
    """Case, with any value scale, 0 among them."""

    def attention(self, q, scale, window):
        assert not window
        group = self.heads // self.kv_heads
        q = q.reshape(-1, self.heads, self.dim)
        out, lse = np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
        spread, products, steps = np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(q.shape)
        self.values = np.zeros(q.shape)         # the sum of the |8-bit values| of the keys that are seen
        for b, token, p in self.rows():
            at = np.arange(p + 1)
            page, slot = self.table[b, at // self.page].astype(np.int64), at % self.page
            for h in range(self.heads):
                g = h // group
                k = self.k[page, g, slot, : self.dim].astype(np.float64) * self.sk[page, g, slot].astype(np.float64)[:, None]
                v, sv = self.v[page, g, slot, : self.dim].astype(np.float64), self.sv[page, g, slot].astype(np.float64)
                t = k @ q[token, h] * scale
                m = t.max()
                w = np.exp(t - m)
                total = w.sum()
                out[token, h] = (w * sv) @ v / total
                lse[token, h] = m + np.log(total)
                spread[token, h] = (w * sv) @ np.abs(v) / total
                self.values[token, h] = np.abs(v).sum(0)
                steps[token, h] = (w * sv).max() * self.values[token, h] / total
                products[token, h] = (np.abs(k) @ np.abs(q[token, h])).max() * abs(scale)
        return out, lse, (spread, products, steps)

    def bounds(self, out, lse, sums, dtype):
        """Case's, and where values are next to nothing beside the sum of the weights: a weight times its scale is then below
        2^6 and off by half of half precision's least step, 2^-25, while the sum is 2^106 at the least (the row's reference is
        2^106 below a weight whose value is that small)."""
        off, off_lse = super().bounds(out, lse, sums, dtype)
        return off + 2.0 ** -131 * self.values * (1.0 if dtype != "f32" else 0.0), off_lse


# Tiles of few rows, one piece and several; of many; images.
WAYS = {"few": [(1, 5), (1, 100), (1, 129)], "pieces": [(1, 2000)], "few and many": [(3, 5), (70, 100), (40, 129)], "many": [(90, 700)],
        "images": [(520, 620)]}


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("way", list(WAYS))
def test_value_scales_of_zero(ops, dtype, way):
    """No values at all; values of some keys only, whose scores are far below and far above the others'."""
    rng = np.random.default_rng(3)
    case = Numbers(rng, WAYS[way], 4, 2, 64, 16)
    held = case.sv.copy()
    case.sv[:] = 0
    check(ops, rng, case, dtype)
    for sign in (0, -1, 1):
        case.sv = held.copy()
        none = rng.random(case.sv.shape) < 0.5
        case.sv[none] = 0
        q = stored(rng.normal(0, 0.3, (case.tokens, 4 * 64)), dtype)
        if sign:        # scores of the keys without values are 140 nats below or above the others'
            case.sk[:] = 0.02
            case.k[..., 0] = np.where(none, sign * 127, 0)
            q[:, ::64] = 448
        check(ops, rng, case, dtype, q=q)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("way", list(WAYS))
@pytest.mark.parametrize("rise", [8.3, 14.0, 15.0, 40.0])
def test_rows_without_values_and_scores_that_grow(ops, dtype, way, rise):
    """Keys and values as q8_cache_write stores them: no values up to three quarters of a sequence, the scores there rising by
    `rise` nats, then values whose scores are the largest, and 14 nats below it."""
    rng = np.random.default_rng(int(rise))
    case = Numbers(rng, WAYS[way], 4, 2, 64, 16)
    cache, batch = case.upload()
    lengths = case.lengths
    whole = C.Batch(C.ints(np.concatenate([[0], np.cumsum(lengths)])), batch.memory[1], batch.memory[2], len(lengths), int(lengths.sum()), case.width)
    for below in (0.0, 14.0):
        k, v = rng.normal(0, 0.02, (int(lengths.sum()), 2, 64)), rng.normal(0.5, 1, (int(lengths.sum()), 2, 64))
        at = 0
        for n in lengths:
            part = np.arange(n) / max(1, 0.75 * n)
            k[at:at + n, :, 0] = np.where(part < 1, part * rise, rise - below)[:, None]
            v[at:at + n][part < 1] = 0
            at += n
        ops.cache_write(C.F32, cache, whole, C.Array.of(k.reshape(-1, 128)), C.Array.of(v.reshape(-1, 128)))
        ops.synchronize()
        case.k, case.v, case.sk, case.sv = case.download()
        assert (case.sv == np.float32(2.0 ** -126)).sum() >= 2 * sum(int(0.75 * n) for n in lengths)
        q = stored(rng.normal(0, 0.3, (case.tokens, 4 * 64)), dtype)
        q[:, ::64] = 8          # with the scale, dim^-1/2, one score a unit of the first value
        check(ops, rng, case, dtype, q=q)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("sequences", [[(1, 200), (1, 161)] * 130, [(40, 64), (33, 64)], *list(WAYS.values())[1:]],
                         ids=["one piece", "one piece of many", *list(WAYS)[1:]])
@pytest.mark.parametrize("where", ["later", "second half"])
def test_sums_of_lanes_and_pieces(ops, dtype, sequences, where):
    """No values, and a few scores 14.1 nats, 20.3 bits, above those that come first: exponentials of 2^106 and then 2^126.3, two
    of which FP32 holds and four not.  They are two of one lane and two of another, in a row's second 32 keys or far behind."""
    rng = np.random.default_rng(6)
    case = Numbers(rng, sequences, 4, 2, 64, 16)
    case.sv[:] = 2.0 ** -126
    case.v[:] = 0
    case.k[..., 0] = 0
    case.sk[:] = 0.001
    for b, (_, length) in enumerate(case.sequences):
        for p in range(length):
            if p % 16 in (0, 4) and (128 <= p < 160 if where == "later" else p % 64 >= 32):
                page, slot = case.place(b, p)
                case.k[page, :, slot, 0] = 47
    q = stored(rng.normal(0, 0.3, (case.tokens, 4 * 64)), dtype)
    q[:, ::64] = 2400       # 2400 * 47 * 0.001 / 8 = 14.1
    check(ops, rng, case, dtype, q=q)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("way", list(WAYS))
@pytest.mark.parametrize("scale", [2.0 ** -115, 2.0 ** -100, 2.0 ** 100])
def test_values_near_the_ends_of_fp32(ops, dtype, way, scale):
    rng = np.random.default_rng(5)
    check(ops, rng, Numbers(rng, WAYS[way], 4, 2, 64, 16, scale=scale), dtype)


class Scores(Numbers):
    """Scores that FP32 holds exactly: q and the keys' scales are powers of two, and a key's first value is all that q meets."""

    def bounds(self, out, lse, sums, dtype):
        """Keys that a row sees differ by whole steps of the scores, 2^16 nats and more, or not at all: those of the largest score
        have one weight, the others none, and the scores' roundings, which are the same for equal ones, touch lse only.  So `out` is
        off by the weights' rounding to 11 bits (FP32: 2^-22), the exponentials' 2^-22 and as many roundings as there are keys in
        numerator and sum.  Up to 2^24 the reference is off its place by a unit at most, so the row's largest weight is 2^5 or more when it
        is rounded, and half precision's least step 2^-30 of it.  lse: six factors and terms, each rounded to 2^-24."""
        keys = max([1] + [int(n) for n in self.lengths])
        spread, _, steps = sums
        rel = 1.01 * ((2.0 ** -11 if dtype != "f32" else 2.0 ** -22) + 2.0 ** -21 + 2 * (keys + 8) * 2.0 ** -24)
        off = spread * rel + (0 if dtype == "f32" else 1.01 * 2.0 ** -30 * steps + 2.0 ** -131 * self.values)
        return off + (np.abs(out) + off) * UNIT[dtype] + TINY[dtype], 8 * 2.0 ** -24 * np.abs(lse) + (keys + 16) * 2.0 ** -23


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("way", list(WAYS))
@pytest.mark.parametrize("step", [2.0 ** 16, 2.0 ** 20, 2.0 ** 25, 2.0 ** 30, 2.0 ** 60, 2.0 ** 90])
def test_scores_of_any_size(ops, dtype, way, step):
    """Up to 100 such steps above and below zero, in any order along the keys, rising, falling, and none above zero; value scales that
    differ by up to 2^69."""
    rng = np.random.default_rng(9)
    case = Scores(rng, WAYS[way], 4, 2, 64, 16)
    case.sk[:] = step
    case.sv *= np.exp2(rng.integers(-60, 9, case.sv.shape)).astype(np.float32)
    q = np.zeros((case.tokens, 4 * 64))
    q[:, ::64] = 8          # with the scale, dim^-1/2, one step of the scores a unit of a key's first value
    q[:, 64] = -8           # one head sees them the other way round
    for order in ("any", "rising", "falling", "below"):
        case.k[..., 0] = rng.integers(-100, 1 if order == "below" else 101, case.k.shape[:3])
        for b, (_, length) in enumerate(case.sequences):
            if order in ("rising", "falling"):
                for p in range(length):
                    page, slot = case.place(b, p)
                    case.k[page, :, slot, 0] = (1 if order == "rising" else -1) * (200 * p // length - 100)
        check(ops, rng, case, dtype, q=q)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("way", list(WAYS))
def test_one_score_a_little_above_large_ones(ops, dtype, way):
    """Scores of 2^24, all the same, and one key's 2^9 above them: a row is the mean of the values that it sees, or that key's."""
    rng = np.random.default_rng(10)
    case = Scores(rng, WAYS[way], 4, 2, 64, 16)
    case.sk[:] = 2.0 ** 18
    case.sv[:] = 1 / 64
    case.k[..., 0] = 64
    q = np.zeros((case.tokens, 4 * 64))
    q[:, ::64] = 8
    case.k[..., 1] = 0
    for b, (_, length) in enumerate(case.sequences):
        page, slot = case.place(b, length // 3)
        case.k[page, :, slot, 1] = 64
    q[:, 1::64] = 2.0 ** -12         # 2^18 2^-12 64 / 8 = 2^9
    check(ops, rng, case, dtype, q=q)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("way", list(WAYS))
@pytest.mark.parametrize("dim", [80, 128, 256])
def test_the_same_with_wider_heads(ops, dtype, way, dim):
    """Scores of up to 2^37 that rise along the keys, value scales of 0, and exponentials that FP32 holds two of, on the kernels for more than 64
    values a head."""
    rng = np.random.default_rng(dim)
    scores = Scores(rng, WAYS[way], 4, 2, dim, 16)
    q = np.zeros((scores.tokens, 4 * dim))
    q[:, ::dim] = 8
    scores.sk[:] = 2.0 ** 30
    for b, (_, length) in enumerate(scores.sequences):
        for p in range(length):
            page, slot = scores.place(b, p)
            scores.k[page, :, slot, 0] = 200 * p // length - 100
    check(ops, rng, scores, dtype, q=q, scale=0.125)
    case = Numbers(rng, WAYS[way], 4, 2, dim, 16)
    case.sv[rng.random(case.sv.shape) < 0.5] = 0
    check(ops, rng, case, dtype)
    case.sv[:], case.v[:], case.sk[:] = 2.0 ** -126, 0, 0.001
    case.k[..., 0] = 0
    for b, (_, length) in enumerate(case.sequences):
        for p in range(length):
            if p % 16 in (0, 4) and p % 64 >= 32:
                page, slot = case.place(b, p)
                case.k[page, :, slot, 0] = 47
    q = stored(rng.normal(0, 0.3, (case.tokens, 4 * dim)), dtype)
    q[:, ::dim] = 2400
    check(ops, rng, case, dtype, q=q, scale=0.125)
