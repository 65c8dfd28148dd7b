"""The rotary, cache and attention operators as a decoder block runs them: together, captured, on other streams, in a large cache."""
import gc

import numpy as np
import pytest

from cache_reference import Case, angles, rotary
from q8_reference import TINY, TYPES, UNIT, stored
from shim import q8_cache as C
from shim import sgemm_shim as S
from test_gpu_noalloc_streams import _Hip, _ok

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, PAGE = 4, 2, 64, 16
COLS = (HEADS + 2 * KV) * DIM       # of a token's queries, keys and values, columns of one product


class At:
    def __init__(self, ptr):
        self.ptr = ptr


class Block:
    """What follows a block's first product: the queries and keys turned where they are, keys and values into the cache, attention."""

    def __init__(self, form, kind, cache, batch, rows):
        self.form, self.kind, self.cache, self.batch, self.rows = form, kind, cache, batch, rows
        self.x = C.Array(rows, COLS, kind)
        self.out, self.lse = C.Array(rows, HEADS * DIM, kind), C.Array(rows, HEADS, C.F32)
        self.freq = C.Array.of((1e4 ** -(np.arange(form.pairs) / form.pairs)).astype(np.float32))
        self.positions = C.ints(np.zeros((form.form.axes, rows)))

    def fill(self, x, positions):
        for to, host in ((self.x, C.Q.to_bf16(x) if self.kind == C.BF16 else np.asarray(x, np.float32 if self.kind == C.F32 else np.float16)),
                         (self.positions, np.asarray(positions, np.int32))):
            host = np.ascontiguousarray(host)
            S._check("sgemm_memcpy_h2d", S.load_library().sgemm_memcpy_h2d(to.ptr, host.ctypes.data, host.nbytes))

    def run(self, o):
        keys, values = At(self.x.ptr + HEADS * DIM * self.x.size), At(self.x.ptr + (HEADS + KV) * DIM * self.x.size)
        # queries and keys are neighbours: one call turns both
        o.rotary(self.kind, self.form, self.x, self.positions, self.freq, self.x, self.rows, HEADS + KV, ldx=COLS, ldy=COLS)
        o.cache_write(self.kind, self.cache, self.batch, keys, values, ldk=COLS, ldv=COLS)
        o.attention(self.kind, self.cache, self.batch, HEADS, self.x, self.out, self.lse, ldq=COLS)


def put(buffer, values):
    host = np.ascontiguousarray(values, np.int32)
    S._check("sgemm_memcpy_h2d", S.load_library().sgemm_memcpy_h2d(buffer.ptr, host.ctypes.data, host.nbytes))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("prompt", [90, 530])
def test_a_prompt_token_by_token(dtype, prompt):
    """A prompt in one call, in chunks, and token by token: the same cache, bit for bit, and results within the bounds."""
    rng = np.random.default_rng(prompt)
    kind = TYPES[dtype]
    form = C.Rotation(DIM, [0] * 12 + [1] * 10 + [2] * 10, 3)
    x = stored(rng.normal(0, 1, (prompt, COLS)), dtype)
    positions = np.stack([np.arange(prompt), np.arange(prompt) // 7, np.arange(prompt) % 7])
    case = Case(rng, [(prompt, prompt)], HEADS, KV, DIM, PAGE)
    got = []
    with C.Ops() as o:
        for chunk in (prompt, 37, 1):
            cache, _ = case.upload()
            starts, lengths = C.ints([0, 0]), C.ints([0])
            table = C.ints(case.table)
            out, q = np.zeros((prompt, HEADS * DIM)), np.zeros((prompt, HEADS * DIM))
            lse = np.zeros((prompt, HEADS))
            block = None
            for at in range(0, prompt, chunk):
                n = min(chunk, prompt - at)
                if block is None or block.rows != n:
                    block = Block(form, kind, cache, C.Batch(starts, lengths, table, 1, n, case.width, longest=n), n)
                put(starts, [0, n])
                put(lengths, [at + n])
                block.fill(x[at:at + n], positions[:, at:at + n])
                block.run(o)
                o.synchronize()
                out[at:at + n], lse[at:at + n], q[at:at + n] = block.out.numpy(), block.lse.numpy(), block.x.numpy()[:, : HEADS * DIM]
            got.append((case.download(), out, lse, q))
    for held, out, lse, q in got:
        assert all(np.array_equal(a, b) for a, b in zip(held, got[0][0])) and np.array_equal(q, got[0][3])
    case.k, case.v, case.sk, case.sv = got[0][0]
    turned = rotary(x[:, : HEADS * DIM].reshape(prompt, HEADS, DIM), angles(positions, form.form.axis[: form.pairs], (1e4 ** -(np.arange(32) / 32)).astype(np.float32)), False, False)
    off = 4 * np.abs(x).max() * 2.0 ** -22      # as in test_gpu_cache_rows.py, for the largest values
    assert np.all(np.abs(got[0][3].reshape(turned.shape) - turned) <= off + (np.abs(turned) + off) * UNIT[dtype] + TINY[dtype])
    want, want_lse, sums = case.attention(got[0][3], DIM ** -0.5, 0)
    off, off_lse = case.bounds(want, want_lse, sums, dtype)
    for _, out, lse, _ in got:
        assert np.all(np.abs(out.reshape(want.shape) - want) <= off) and np.all(np.abs(lse - want_lse) <= off_lse)


@pytest.mark.parametrize("sequences,longest", [([(1, 700), (1, 900), (1, 30)], 1), ([(90, 700), (1, 300), (50, 64)], 90), ([(600, 600)], 600),
                                               ([(90, 1500)], 90)])
def test_captured_calls_replay(sequences, longest):
    """One graph serves later lengths, pages and chunks: every replay has the bits of the eager calls, which run between the
    replays on the same handle, and after its workspace was replaced."""
    rng = np.random.default_rng(len(sequences))
    case = Case(rng, sequences, HEADS, KV, DIM, PAGE, width_more=2, spare_pages=9)
    form = C.Rotation(DIM, [0] * 32)
    x = stored(rng.normal(0, 1, (case.tokens, COLS)), "bf16")
    gc.collect()        # a buffer that an earlier test left in a cycle, freed during a capture, would end it
    gc.disable()
    hip = _Hip()
    stream = hip.stream()
    o = C.Ops()
    cache, batch = case.upload()
    block = Block(form, C.BF16, cache, batch, case.tokens)
    starts, lengths, table = batch.memory
    try:
        o.set_stream(stream.value)
        need = C.attention_workspace(C.BF16, cache, batch, HEADS)
        assert need > 0
        hip.begin(stream, 0)
        try:
            with pytest.raises(S.SgemmError) as e:
                o.attention(C.BF16, cache, batch, HEADS, block.x, block.out, ldq=COLS)
            assert e.value.code == -4 and "q8_reserve" in e.value.message
        finally:
            _ok(hip.lib.hipGraphExecDestroy(hip.end(stream)))
        o.reserve(need)
        hip.begin(stream, 0)
        try:
            block.run(o)
        finally:
            exe = hip.end(stream)
        before = case.k, case.v, case.sk, case.sv
        for turn in range(4):
            # lengths shrink, pages change places, one is not there; the chunks shrink too
            put(lengths, case.lengths - 7 * turn)
            pages = case.table.copy()
            if turn:
                pages[:, : case.width] = np.where(pages[:, : case.width] >= 0, (pages[:, : case.width] + turn) % case.pages, -1)
                pages[0, 1] = -1
            put(table, pages)
            put(starts, np.maximum(case.starts - (turn == 3), 0))
            positions = np.arange(case.tokens)[None] + turn
            block.fill(x, positions)
            block.run(o)
            o.synchronize()
            want = (block.out.numpy().copy(), block.lse.numpy().copy(), *case.download())
            assert np.all(np.isfinite(want[0])) and np.any(want[0] != 0)
            for m in (block.out, block.lse):
                S._check("sgemm_memset", S.load_library().sgemm_memset(m.ptr, 0, m.nbytes))
            for m, host in zip(case.memory, before):        # the cache as it was before the eager call
                host = np.ascontiguousarray(host)
                S._check("sgemm_memcpy_h2d", S.load_library().sgemm_memcpy_h2d(m.ptr, host.ctypes.data, host.nbytes))
            block.fill(x, positions)
            _ok(hip.lib.hipGraphLaunch(exe, stream))
            o.synchronize()
            rows = slice(0, int(case.starts[-1]) - (turn == 3))
            got = (block.out.numpy(), block.lse.numpy(), *case.download())
            for i, (a, b) in enumerate(zip(got, want)):
                a, b = (a[rows], b[rows]) if i < 2 else (a, b)
                assert np.array_equal(a, b), (turn, i)
            before = want[2:]
            need *= 2
            o.reserve(need)
        _ok(hip.lib.hipGraphExecDestroy(exe))
    finally:
        gc.enable()
        o.set_stream(None)
        o.close()
        hip.lib.hipStreamDestroy(stream)


def test_two_handles_at_once():
    """Two handles on their own streams over one cache that both read: neither changes the other's results."""
    rng = np.random.default_rng(4)
    case = Case(rng, [(1, 4000), (1, 2500), (1, 60)], HEADS, KV, DIM, PAGE, longest=1)
    cache, batch = case.upload()
    qs = [C.Array.of(rng.normal(0, 1, (3, HEADS * DIM)), C.BF16) for _ in range(2)]
    outs = [C.Array(3, HEADS * DIM, C.BF16) for _ in range(2)]
    a, b = C.Ops(), C.Ops()
    try:
        want = []
        for o, q, out in zip((a, b), qs, outs):
            o.attention(C.BF16, cache, batch, HEADS, q, out)
            o.synchronize()
            want.append(out.numpy().copy())
        assert not np.array_equal(*want)
        for _ in range(20):
            for o, q, out in zip((a, b), qs, outs):
                o.attention(C.BF16, cache, batch, HEADS, q, out)
        a.synchronize()
        b.synchronize()
        assert all(np.array_equal(out.numpy(), w) for out, w in zip(outs, want))
    finally:
        a.close()
        b.close()


def test_offsets_past_32_bits():
    """Rows, pages and tokens whose byte offsets pass 2^32 (the first by sign, too) give the bits of the same ones close together."""
    rng = np.random.default_rng(6)
    sequences, heads, kv, dim, page = [(600, 700), (1, 900), (1, 60)], 8, 4, 128, 16
    near = Case(rng, sequences, heads, kv, dim, page)
    pages = (9 << 30) // (kv * page * dim)              # 9 GiB of keys and as many of values
    far = C.Cache.empty(pages, page, kv, dim)
    close, batch = near.upload()
    # page i of the near cache is one of the last of the far one, some of them just past 2^31 and 2^32 bytes
    places = pages - 1 - 3 * np.arange(near.pages)
    places[:2] = (1 << 31) // (kv * page * dim), (1 << 32) // (kv * page * dim)
    table = np.where(near.table >= 0, places[np.clip(near.table, 0, near.pages - 1)], -1)
    far_batch = C.Batch(batch.memory[0], batch.memory[1], C.ints(table), len(sequences), near.tokens, near.width)
    cols, kcols, ld = heads * dim, kv * dim, 6 << 20    # 602 rows of 12 MiB
    size = 2 * ((near.tokens - 1) * ld + cols)
    assert size > 7 << 30 and near.tokens * heads // kv >= 1024
    wide = [S.DeviceBuffer(size) for _ in range(2)]
    with C.Ops() as o:
        # whole sequences into both caches
        whole = int(near.lengths.sum())
        starts = C.ints(np.concatenate([[0], np.cumsum(near.lengths)]))
        k, v = (C.Array.of(rng.normal(0, 1, (whole, kcols)), C.BF16) for _ in range(2))
        back = []
        for cache, pages_ in ((close, batch.memory[2]), (far, far_batch.memory[2])):
            all_ = C.Batch(starts, batch.memory[1], pages_, len(sequences), whole, near.width)
            o.cache_write(C.BF16, cache, all_, k, v)
            r = [C.Array(whole, kcols, C.F32) for _ in range(2)]
            o.cache_read(C.F32, cache, all_, *r)
            o.synchronize()
            back.append([a.numpy() for a in r])
        assert all(np.array_equal(a, b) for a, b in zip(*back)) and np.all(np.isfinite(back[0][0]))
        x = C.Array.of(rng.normal(0, 1, (near.tokens, cols)), C.BF16)
        y, tight = C.Array(near.tokens, cols, C.BF16), C.Array(near.tokens, cols, C.BF16)
        lse, far_lse = C.Array(near.tokens, heads, C.F32), C.Array(near.tokens, heads, C.F32)
        form, freq, positions = C.Rotation(dim, [0] * 64), C.Array.of(np.linspace(1, 0.01, 64)), C.ints(np.arange(near.tokens)[None])
        still = C.Rotation(dim, [])
        # rotary from and to rows far apart
        o.rotary(C.BF16, form, x, positions, freq, tight, near.tokens, heads)
        o.rotary(C.BF16, form, x, positions, freq, wide[0], near.tokens, heads, ldy=ld)
        o.rotary(C.BF16, still, wide[0], None, None, y, near.tokens, heads, ldx=ld)
        o.synchronize()
        assert np.array_equal(y.numpy(), tight.numpy())
        want = C.Array(near.tokens, cols, C.BF16)
        for longest in (600, 1):
            for b in (batch, far_batch):
                b.form.longest = longest
            o.attention(C.BF16, close, batch, heads, tight, want, lse)
            o.attention(C.BF16, far, far_batch, heads, wide[0], wide[1], far_lse, ldq=ld, ldo=ld)
            o.rotary(C.BF16, still, wide[1], None, None, y, near.tokens, heads, ldx=ld)
            o.synchronize()
            assert np.array_equal(y.numpy(), want.numpy()) and np.array_equal(lse.numpy(), far_lse.numpy())
            assert np.all(np.isfinite(y.numpy())) and np.any(y.numpy() != 0)
        # one sequence's prompt, from images
        one, far_one = (C.Batch(C.ints([0, near.tokens]), C.ints([700]), t, 1, near.tokens, near.width, table_ld=near.width)
                        for t in (batch.memory[2], far_batch.memory[2]))
        o.attention(C.BF16, close, one, heads, tight, want, lse)
        o.attention(C.BF16, far, far_one, heads, wide[0], wide[1], far_lse, ldq=ld, ldo=ld)
        o.rotary(C.BF16, still, wide[1], None, None, y, near.tokens, heads, ldx=ld)
        o.synchronize()
        assert np.array_equal(y.numpy(), want.numpy()) and np.array_equal(lse.numpy(), far_lse.numpy())
