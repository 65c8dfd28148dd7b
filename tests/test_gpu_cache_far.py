"""Attention with a window at positions far into tables that are far wider than what is resident, against float64."""
import numpy as np
import pytest

from cache_reference import Case
from q8_reference import TYPES, stored
from shim import q8_cache as C
from test_gpu_cache_attention import check

PAGE = 65536
WIDTH = (2 ** 31 - 2 ** 16) // PAGE - 1       # as wide as tables may be: 2147352576 positions


class Far(Case):
    """One sequence of `length` tokens of which only the pages that the chunk's windows reach are there."""

    def __init__(self, rng, chunk, length, window, heads, kv_heads, dim):
        self.window = window
        first = length - chunk - window + 1
        pages = range(max(0, first) // PAGE, (length - 1) // PAGE + 1)
        super().__init__(rng, [(chunk, len(pages) * PAGE)], heads, kv_heads, dim, PAGE, spare_pages=0)
        resident = self.table[0].copy()
        self.width = WIDTH
        self.table = np.full((1, WIDTH), -1, np.int32)
        self.table[0, list(pages)] = resident
        self.sequences, self.lengths = [(chunk, length)], np.array([length], np.int64)

    def attention(self, q, scale, window):
        assert window == self.window
        group, n = self.heads // self.kv_heads, self.tokens
        q = q.reshape(n, self.kv_heads, group, self.dim)
        p = (int(self.lengths[0]) - n + np.arange(n))[:, None] - np.arange(window)      # tokens x their windows' keys
        assert p.min() >= 0
        page, slot = self.table[0, p // PAGE].astype(np.int64), p % PAGE
        out, lse = np.zeros((n, self.heads, self.dim)), np.zeros((n, self.heads))
        spread, products, steps = np.zeros(out.shape), np.zeros(lse.shape), np.zeros(out.shape)
        for h in range(self.kv_heads):
            of = slice(h * group, (h + 1) * group)
            sv = self.sv[page, h, slot].astype(np.float64)
            k = self.k[page, h, slot, : self.dim] * self.sk[page, h, slot].astype(np.float64)[..., None]
            v = self.v[page, h, slot, : self.dim] * sv[..., None]
            t = np.matmul(q[:, h], k.transpose(0, 2, 1)) * scale
            m = t.max(2, keepdims=True)
            w = np.exp(t - m)
            total = w.sum(2)
            lse[:, of] = m[..., 0] + np.log(total)
            out[:, of] = np.matmul(w, v) / total[..., None]
            spread[:, of] = np.matmul(w, np.abs(v)) / total[..., None]
            steps[:, of] = (w * sv[:, None]).max(2)[..., None] * np.abs(self.v[page, h, slot, : self.dim].astype(np.float64)).sum(1)[:, None] / total[..., None]
            products[:, of] = np.matmul(np.abs(q[:, h]), np.abs(k).transpose(0, 2, 1)).max(2) * abs(scale)
        return out, lse, (spread, products, steps)

    def bounds(self, out, lse, sums, dtype):
        held, self.lengths = self.lengths, np.array([self.window])      # a row sums a window's keys
        try:
            return super().bounds(out, lse, sums, dtype)
        finally:
            self.lengths = held


@pytest.fixture(scope="module")
def ops():
    with C.Ops() as o:
        yield o


# One token; rows in tiles of 256 and of 128, several pieces and one piece (as long as the table); narrow and wide heads.
@pytest.mark.parametrize("dtype,chunk,heads,kv_heads,dim", [("bf16", 1, 4, 2, 64), ("f32", 1, 4, 1, 128), ("f16", 60, 4, 2, 64), ("f32", 60, 4, 2, 64),
                                                            ("bf16", 1100, 64, 1, 64), ("f16", 1100, 64, 1, 33), ("f32", 600, 64, 1, 64),
                                                            ("bf16", 600, 64, 1, 136)])
@pytest.mark.parametrize("length", [200000, PAGE * WIDTH - 1])
@pytest.mark.gpu
def test_a_window_far_into_a_wide_table(ops, dtype, chunk, heads, kv_heads, dim, length):
    rng = np.random.default_rng(chunk + dim)
    window = 40
    check(ops, rng, Far(rng, chunk, length, window, heads, kv_heads, dim), dtype, window=window)


def test_those_plans_have_pieces_as_long_as_the_table():
    """The chunks of 600 and 1100 tokens run in one piece: no sums of pieces, no images."""
    for dtype, chunk, dim in ((C.BF16, 1100, 64), (C.F16, 1100, 33), (C.F32, 600, 64), (C.BF16, 600, 136)):
        cache, batch = C.Cache(None, None, None, None, 2, PAGE, 1, dim), C.Batch(None, None, None, 1, chunk, WIDTH)
        assert C.attention_workspace(dtype, cache, batch, 64) == 0
