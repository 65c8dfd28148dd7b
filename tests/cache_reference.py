"""The rotary, cache and attention operators in float64, and a batch of sequences on the device."""
import numpy as np

from q8_reference import LEAST_SCALE, TINY, TYPES, UNIT, Window, stored
from shim import q8_cache as C

KINDS = TYPES


def angles(positions, axis, freq):
    """tokens x pairs, exact but for float64's rounding of the product."""
    freq = np.asarray(freq, np.float32).astype(np.float64)
    return np.stack([positions[a].astype(np.float64) * f for a, f in zip(axis, freq)], 1) if len(axis) else np.zeros((positions.shape[1], 0))


def rotary(x, angle, neighbours, inverse):
    """x: tokens x heads x dim."""
    pairs = angle.shape[1]
    one, two = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if neighbours else (slice(0, pairs), slice(pairs, 2 * pairs))
    c, s = np.cos(angle)[:, None, :], np.sin(angle)[:, None, :] * (-1 if inverse else 1)
    y = x.copy()
    y[:, :, one] = x[:, :, one] * c - x[:, :, two] * s
    y[:, :, two] = x[:, :, two] * c + x[:, :, one] * s
    return y


class Case:
    """Sequences over a cache that holds random rows: chunks and lengths, pages in random places."""

    def __init__(self, rng, sequences, heads, kv_heads, dim, page, extra_rows=0, front_rows=0, spare_pages=2, width_more=0,
                 ld_more=0, longest=0, scale=None):
        self.sequences = list(sequences)
        self.heads, self.kv_heads, self.dim, self.page = heads, kv_heads, dim, page
        self.pitch = -(-dim // 16) * 16
        chunks, lengths = [s[0] for s in sequences], [s[1] for s in sequences]
        needed = [-(-max(t, 0) // page) for t in lengths]
        self.width = max(needed, default=0) + width_more
        self.pages = sum(needed) + spare_pages
        order = rng.permutation(self.pages)
        self.table = rng.integers(-5, 2 ** 31 - 1, (len(sequences), self.width + ld_more)).astype(np.int32)
        self.table[:, : self.width] = -1
        at = 0
        for b, n in enumerate(needed):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.starts = front_rows + np.concatenate([[0], np.cumsum(chunks)]).astype(np.int64)
        self.lengths = np.array(lengths, np.int64)
        self.tokens = int(self.starts[-1]) + extra_rows
        shape = (self.pages, kv_heads, page)
        self.k = np.zeros(shape + (self.pitch,), np.int8)
        self.v = np.zeros(shape + (self.pitch,), np.int8)
        self.k[..., :dim] = np.clip(np.rint(rng.normal(0, 45, shape + (dim,))), -127, 127)
        self.v[..., :dim] = np.clip(np.rint(rng.normal(10, 40, shape + (dim,))), -127, 127)
        self.sk = (np.exp(0.3 * rng.normal(0, 1, shape)) / 40).astype(np.float32)
        self.sv = (np.exp(0.5 * rng.normal(0, 1, shape)) / 40).astype(np.float32)
        if scale is not None:
            self.sv *= np.float32(scale)
        self.longest = longest

    def place(self, b, p):
        """Page and slot of position p, None if it is not there."""
        if p < 0 or p >= self.width * self.page:
            return None
        page = int(self.table[b, p // self.page])
        return (page, p % self.page) if 0 <= page < self.pages else None

    def upload(self):
        rows = self.pages * self.kv_heads * self.page
        self.memory = [C.Array.of(self.k.reshape(rows, self.pitch)), C.Array.of(self.v.reshape(rows, self.pitch)),
                       C.Array.of(self.sk.reshape(1, rows)), C.Array.of(self.sv.reshape(1, rows))]
        cache = C.Cache(*self.memory, self.pages, self.page, self.kv_heads, self.dim)
        batch = C.Batch(C.ints(self.starts), C.ints(self.lengths), C.ints(self.table), len(self.sequences), self.tokens, self.width,
                        table_ld=self.table.shape[1], longest=self.longest)
        return cache, batch

    def download(self):
        shape = self.k.shape[:3]
        k, v, sk, sv = (m.numpy() for m in self.memory)
        return k.reshape(self.k.shape), v.reshape(self.v.shape), sk.reshape(shape), sv.reshape(shape)

    def rows(self):
        """(sequence, token, position) of the chunks' tokens."""
        for b, (first, end) in enumerate(zip(self.starts[:-1], self.starts[1:])):
            for token in range(max(0, first), min(end, self.tokens)):
                yield b, token, int(self.lengths[b]) - min(int(end), self.tokens) + token

    def attention(self, q, scale, window):
        """out, lse, and per row: the sums of |weight v|, the largest sum of |products| of a score, and the sums of |v|'s steps
        times the largest weight of a step (its key's weight times the values' scale)."""
        group = self.heads // self.kv_heads
        q = q.reshape(-1, self.heads, self.dim)
        out, lse = np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
        spread, products, steps = np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(q.shape)
        held = {}
        for b, token, p in self.rows():
            if b not in held:
                n = max(0, min(int(self.lengths[b]), self.width * self.page))
                at = np.arange(n)
                page = self.table[b, at // self.page].astype(np.int64)
                there = (page >= 0) & (page < self.pages)
                page = np.where(there, page, 0)
                held[b] = (there, self.sv[page, :, at % self.page].astype(np.float64), *(c[page, :, at % self.page, : self.dim].astype(np.float64) * s[page, :, at % self.page].astype(np.float64)[..., None]
                                    for c, s in ((self.k, self.sk), (self.v, self.sv))))
            there, sv, k, v = held[b]
            at = np.arange(len(there))
            seen = there & (at <= p) & ((at > p - window) if window else True)
            if not seen.any():
                continue
            for h in range(self.heads):
                kk, vv = k[seen, h // group], v[seen, h // group]
                t = kk @ q[token, h] * scale
                m = t.max()
                w = np.exp(t - m)
                total = w.sum()
                out[token, h] = w @ vv / total
                lse[token, h] = m + np.log(total)
                spread[token, h] = w @ np.abs(vv) / total
                s = sv[seen, h // group]
                steps[token, h] = (w * s).max() * np.abs(vv / s[:, None]).sum(0) / total
                products[token, h] = (np.abs(kk) @ np.abs(q[token, h])).max() * abs(scale)
        return out, lse, (spread, products, steps)

    def bounds(self, out, lse, sums, dtype):
        """How far out and lse may be off: the scores' products and sums in FP32 (an error of dim + 8 roundings of the
        largest sum of products: the dim - 1 additions, four factors, the exponential's argument and its base), which the
        weights follow to first order, twice, for numerator and sum; exp2 to 2^-22; as many roundings again as keys for the
        sums; the weights' rounding to 11 bits for 16-bit types (another 2^-23 of a term cut off for F32); the result's rounding.
        Half precision's steps are 2^-24 at the least, a weight (times its scale) is off by half of one; the row's largest is 2^6 or
        more when it is rounded, as R is moved only to bring it there, so the error is 2^-31 of that one.  The second order of
        these (below 2^-10 of them) is in the factor 1.01."""
        spread, products, steps = sums
        keys = max([1] + [int(n) for n in self.lengths])
        score = (self.dim + 8) * 2.0 ** -24 * products + 2.0 ** -22 * np.where(np.isfinite(lse), np.abs(lse), 0)
        adds = (keys + 8) * 2.0 ** -24
        weight = 2.0 ** -11 if dtype != "f32" else 2.0 ** -22
        rel = 1.01 * (2 * score + 2.0 ** -21 + 2 * adds + weight)
        off = spread * rel[..., None] + (0 if dtype == "f32" else 1.01 * 2.0 ** -31 * steps)
        return off + (np.abs(out) + off) * UNIT[dtype] + TINY[dtype], 1.01 * (score + adds + 2.0 ** -21) + np.where(np.isfinite(lse), np.abs(lse), 0) * 2.0 ** -22
