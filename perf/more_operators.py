"""The work that the rotary, cache and attention operators for language models are measured on.

What a decoder's block does between the product that gives queries, keys and values
and the one that takes the attention's output: positions turn queries and keys, keys
and values go into a paged cache as 8-bit rows with a scale for each head of each
token, and the new tokens attend to the cache.  A sequence's new tokens are its
chunk; one token each is decoding, a chunk as long as its sequence is a prompt.
Tokens of all chunks follow one another as rows.

One pass is one of
  rotary   heads turned by positions on one or three axes, or turned back (the gradient)
  cache    a chunk's keys and values written in 8 bits, and read back
  attend   the chunks' attention over the cache
  step     all of them, as a serving step calls them: queries and keys turned, keys and
           values written, the chunks' attention
"""
import functools
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _case(name, op, dtype, seqs=1, chunk=(1, 1), context=(1, 1), heads=32, kv_heads=8, dim=128, page=16, window=0, pad=0,
          pairs=64, axes=1, neighbours=False, inverse=False, first=0):
    return {"name": name, "op": op, "dtype": dtype, "seqs": seqs, "chunk_lo": chunk[0], "chunk_hi": chunk[1],
            "context_lo": context[0], "context_hi": context[1], "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "window": window, "pad": pad, "pairs": pairs, "axes": axes, "neighbours": neighbours, "inverse": inverse,
            "first": first}


def listed():
    return [
        # the smallest call: one token's queries and keys, far into a text
        _case("rotary_1x40x128", "rotary", "bf16", kv_heads=8, first=1_000_000),
        # a batch of prompts with images: time, height and width
        _case("rotary_16384x40x128", "rotary", "bf16", chunk=(16384, 16384), axes=3),
        # the gradient of a part of odd heads, neighbouring values paired, rows padded
        _case("rotary_bwd_1001x25x80", "rotary", "f32", chunk=(1001, 1001), heads=20, kv_heads=5, dim=80, pairs=26, pad=3,
              neighbours=True, inverse=True),
        # a batch of prompts into the cache and back
        _case("cache_16384x8x128", "cache", "bf16", seqs=8, chunk=(2048, 2048), context=(2048, 4096)),
        # odd chunks that start and end inside pages of odd length, narrow heads
        _case("cache_1239x3x80", "cache", "f16", seqs=7, chunk=(1, 353), context=(353, 900), kv_heads=3, dim=80, page=24, pad=5),
        # one token of one sequence through everything
        _case("step_1x2048", "step", "bf16", context=(2048, 2048)),
        # decoding one sequence
        _case("attend_1x4096", "attend", "bf16", context=(4096, 4096)),
        # decoding one very long one
        _case("attend_1x131072", "attend", "bf16", context=(131072, 131072), page=64),
        # decoding a batch of different lengths
        _case("attend_64x8192", "attend", "f16", seqs=64, context=(1024, 8192)),
        # the next chunks of long prompts, beside what the cache holds already
        _case("attend_4x512x8192", "attend", "bf16", seqs=4, chunk=(512, 512), context=(4096, 8192)),
        # odd heads, chunks and pages in 32 bits, with a window
        _case("attend_5x77x1501", "attend", "f32", seqs=5, chunk=(3, 77), context=(97, 1501), heads=15, kv_heads=3, dim=80, page=24,
              window=401, pad=7),
        # the largest: a whole prompt
        _case("attend_8192x8192", "attend", "bf16", chunk=(8192, 8192), context=(8192, 8192)),
    ]


MOST_FLOPS = 4 * 128 * 32 * 8192 * 4096      # of an attention: the whole prompt's
MOST_VALUES = 16384 * 40 * 128               # of a rotation or a cache's chunk
MOST_CACHE = 64 * 8192 * 8 * 128             # values of all sequences' keys, each as long as the longest


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["rotary", "cache", "attend", "attend", "attend", "step"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"]) if op != "step" else rng.choice(["bf16", "f16"])
    group = rng.choice([1, 2, 4, 4, 5, 8, 8, 16])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8, 16])
    dim = rng.choice([64, 128, 128, 128, 256, 80, 96, 72, 33])
    page = rng.choice([16, 16, 64, 128, 24, 1, 5])
    pad = rng.choice([0, 0, 0, 3, 16])
    pairs = dim // 2 if rng.random() < 0.7 else rng.randint(1, dim // 2)
    form = dict(pairs=pairs, axes=rng.choice([1, 1, 3]), neighbours=rng.random() < 0.3, first=rng.choice([0, 0, log(1, 4_000_000)]))
    if op == "rotary":
        tokens = log(1, 16384)
        while tokens * kv_heads * (group + 1) * dim > MOST_VALUES:
            tokens = max(1, tokens // 2)
        case = _case("", op, dtype, chunk=(tokens, tokens), heads=kv_heads * group, kv_heads=kv_heads, dim=dim, pad=pad,
                     inverse=rng.random() < 0.5, **form)
    else:
        seqs = log(1, 128)
        hi = log(1, 8192) if op != "step" and rng.random() < 0.6 else rng.choice([1, 1, 2, 4])
        chunk = (rng.choice([1, hi]), hi)
        context = log(hi, max(hi, 32768))
        least = max(hi, context // rng.choice([1, 2, 8]))

        def too_much():
            return (seqs * context * kv_heads * dim > MOST_CACHE or 4 * dim * seqs * hi * context * kv_heads * group > MOST_FLOPS
                    or (op == "cache" and seqs * hi * kv_heads * dim > MOST_VALUES))

        while too_much() and seqs > 1:
            seqs = seqs // 2
        while too_much():
            context = max(1, context // 2)
            hi = min(hi, context)
            chunk, least = (min(chunk[0], hi), hi), max(hi, min(least, context))
        window = rng.choice([0, 0, 0, log(1, 4096)]) if op == "attend" else 0
        case = _case("", op, dtype, seqs, chunk, (least, context), kv_heads * group, kv_heads, dim, page, window, pad, **form)
    del case["name"]
    return case


class _Buffer:
    """A torch tensor's memory as the entry points take it."""

    def __init__(self, t):
        self.tensor = t
        self.ptr = t.data_ptr()


def _lengths(case):
    """Tokens of each chunk, and of each sequence with its chunk."""
    n = case["seqs"]
    step = next(s for s in (7, 11, 13, 1) if math.gcd(s, n) == 1)     # lengths in no order
    part = [(b * step % n) / max(1, n - 1) for b in range(n)]
    chunks = [case["chunk_lo"] + round((case["chunk_hi"] - case["chunk_lo"]) * (b / max(1, n - 1))) for b in range(n)]
    contexts = [case["context_lo"] + round((case["context_hi"] - case["context_lo"]) * p) for p in part]
    if n == 1:
        chunks, contexts = [case["chunk_hi"]], [case["context_hi"]]
    return chunks, [max(c, t) for c, t in zip(chunks, contexts)]


def _tokens(case):
    return sum(_lengths(case)[0])


def _pitch(dim):
    return -(-dim // 16) * 16


def _width(case):
    """Pages in a row of the table."""
    return -(-max(_lengths(case)[1]) // case["page"])


def _axis(case):
    """The axis of each pair: a quarter of them for time, the rest for height and width."""
    pairs = case["pairs"]
    if case["axes"] == 1:
        return [0] * pairs
    time = pairs // 4
    height = (pairs - time) // 2
    return [0] * time + [1] * height + [2] * (pairs - time - height)


def _inputs(case, seed):
    dtype, dim, pad = TYPES[case["dtype"]], case["dim"], case["pad"]
    heads, kv_heads, page, seqs = case["heads"], case["kv_heads"], case["page"], case["seqs"]
    op, tokens = case["op"], _tokens(case)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    def rows(t):
        """The heads of each token after one another, in rows of `pad` more values."""
        t = t.reshape(t.shape[0], -1)
        out = torch.zeros((t.shape[0], t.shape[1] + pad), device="cuda", dtype=dtype)
        out[:, : t.shape[1]] = t
        return out

    def vectors(n, h, offset):
        # channels have an offset, heads differ in size, a few channels stand out
        return (normal(n, h, dim) + offset * normal(1, h, dim)) * torch.exp(0.2 * normal(1, h, 1)) * (1 + 2 * (normal(1, h, dim) > 2.2))

    s = {}
    if op in ("rotary", "step"):
        at = torch.arange(tokens, device="cuda", dtype=torch.int32) + case["first"]
        if op == "step":
            chunks, contexts = _lengths(case)
            at = torch.cat([torch.arange(t - c, t, device="cuda", dtype=torch.int32) for c, t in zip(chunks, contexts)])
        positions = at.repeat(case["axes"], 1)
        if case["axes"] == 3:     # images of 24 by 32 between texts
            inside = at % 1024
            image = inside < 768
            corner = at - inside
            positions[0] = torch.where(image, corner, at)
            positions[1] = torch.where(image, corner + inside // 32, at)
            positions[2] = torch.where(image, corner + inside % 32, at)
        s["positions"] = positions.contiguous()
        s["freq"] = (1e6 ** (-torch.arange(case["pairs"], device="cuda", dtype=torch.float64) / case["pairs"])).float()
    if op == "rotary":
        s["x"] = rows(vectors(tokens, heads + kv_heads, 0.5))
    if op == "step":      # one product's rows: queries, keys, values
        s["x"] = rows(torch.cat([vectors(tokens, heads, 0.3), vectors(tokens, kv_heads, 0.3), vectors(tokens, kv_heads, 0.5)], 1))
    if op == "cache":
        s["k"], s["v"] = rows(vectors(tokens, kv_heads, 1.0)), rows(vectors(tokens, kv_heads, 0.5))
    if op == "attend":
        s["q"] = rows(vectors(tokens, heads, 0.3))
    if op != "rotary":
        chunks, contexts = _lengths(case)
        width = _width(case)
        needed = [-(-t // page) for t in contexts]
        pages = sum(needed) + 3
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)     # pages lie anywhere
        table = torch.full((seqs, width), -1, device="cuda", dtype=torch.int32)
        at = 0
        for b, n in enumerate(needed):
            table[b, :n] = order[at:at + n]
            at += n
        s["table"] = table
        s["starts"] = torch.tensor([sum(chunks[:b]) for b in range(seqs + 1)], dtype=torch.int32, device="cuda")
        s["lengths"] = torch.tensor(contexts, dtype=torch.int32, device="cuda")
        shape = (pages, kv_heads, page)
        for name, offset in (("k", 20.0), ("v", 15.0)):
            q = torch.zeros(shape + (_pitch(dim),), device="cuda", dtype=torch.int8)
            for h in range(kv_heads):       # a head at a time: the 32-bit values take four times the room
                channels = offset * normal(1, 1, dim)
                q[:, h, :, :dim] = torch.round(30 * normal(pages, page, dim) + channels).clamp_(-127, 127).to(torch.int8)
            s["cache_" + name] = q
            s["scale_" + name] = torch.exp(0.25 * normal(*shape)) / 40
    return s


def prepare(case, seed):
    dtype, dim, pad = TYPES[case["dtype"]], case["dim"], case["pad"]
    heads, kv_heads, op = case["heads"], case["kv_heads"], case["op"]
    state, tokens = _inputs(case, seed), _tokens(case)

    def empty(cols, dt=dtype):
        return torch.zeros((tokens, cols), device="cuda", dtype=dt)

    out = {}
    if op in ("rotary", "step"):
        out["y"] = empty((heads + kv_heads) * dim + pad)
    if op == "cache":
        back = torch.bfloat16 if case["dtype"] == "f32" else dtype
        out["k"], out["v"] = empty(kv_heads * dim, back), empty(kv_heads * dim, back)
    if op in ("attend", "step"):
        out["o"] = empty(heads * dim + pad)
    if op == "attend":
        out["lse"] = empty(heads, torch.float32)
    buffers = {name: _Buffer(t) for name, t in {**state, **{"out_" + n: t for n, t in out.items()}}.items()}
    # kept: the forms, the cache's and the batch's descriptions, as a program keeps them from call to call
    return {"case": case, "in": state, "out": out, "buffers": buffers, "kept": {}}


def _plain_rotary(case, s, heads):
    dim, pairs, tokens = case["dim"], case["pairs"], s["positions"].shape[1]
    x = s["x"][:, : heads * dim].float().reshape(tokens, heads, dim)
    at = s["positions"][torch.tensor(_axis(case), device=x.device)].double()      # pairs, tokens
    angle = (at * s["freq"].double()[:, None]).t()[:, None, :]
    c, n = angle.cos().float(), angle.sin().float()
    if case["inverse"]:
        n = -n
    one, two = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if case["neighbours"] else (slice(0, pairs), slice(pairs, 2 * pairs))
    y = x.clone()
    y[:, :, one] = x[:, :, one] * c - x[:, :, two] * n
    y[:, :, two] = x[:, :, two] * c + x[:, :, one] * n
    return y.reshape(tokens, -1).to(TYPES[case["dtype"]])


def _places(case, s):
    """Each new token's sequence, its place among the chunk's, its page and its slot."""
    token = torch.arange(_tokens(case), device="cuda")
    starts = s["starts"].long()
    seq = torch.searchsorted(starts, token, right=True) - 1
    local = token - starts[seq]
    at = s["lengths"].long()[seq] - (starts[seq + 1] - starts[seq]) + local
    return seq, local, s["table"].long()[seq, at // case["page"]], at % case["page"]


def _plain_write(case, s, name, x):
    dim = case["dim"]
    x = x.float().reshape(x.shape[0], case["kv_heads"], dim)
    scale = (x.abs().amax(2) / 127).clamp_min(2.0 ** -126)
    _, _, page, slot = _places(case, s)
    s["cache_" + name][page, :, slot, :dim] = torch.round(x / scale[..., None]).clamp(-127, 127).to(torch.int8)
    s["scale_" + name][page, :, slot] = scale


def _plain_read(case, s, name, dtype):
    _, _, page, slot = _places(case, s)
    y = s["cache_" + name][page, :, slot, : case["dim"]].float() * s["scale_" + name][page, :, slot][..., None]
    return y.reshape(y.shape[0], -1).to(dtype)


def _plain_attend(case, s, q):
    dim, kv_heads, page, most = case["dim"], case["kv_heads"], case["page"], max(_lengths(case)[1])
    group, longest, seqs = case["heads"] // kv_heads, max(_lengths(case)[0]), case["seqs"]
    key = torch.arange(most, device="cuda")
    where = s["table"].long()[:, key // page].clamp_min(0)

    def vectors(name):      # sequences, heads, keys, values
        v = s["cache_" + name][where, :, (key % page)[None, :], :dim].float() * s["scale_" + name][where, :, (key % page)[None, :]][..., None]
        return v.permute(0, 2, 1, 3).contiguous()

    lengths, starts = s["lengths"].long(), s["starts"].long()
    n = starts[1:] - starts[:-1]
    row = torch.arange(longest, device="cuda")
    padded = q.float()[(starts[:-1, None] + row).clamp_max(q.shape[0] - 1)]         # sequences, tokens, values
    padded = padded.reshape(seqs, longest, kv_heads, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, kv_heads, longest * group, dim)
    scores = torch.matmul(padded.contiguous(), vectors("k").transpose(2, 3).contiguous()).mul_(dim ** -0.5)
    scores = scores.reshape(seqs, kv_heads, longest, group, most)
    at = (lengths - n)[:, None] + row                                               # each new token's position
    seen = key[None, None, :] <= at[:, :, None]
    if case["window"]:
        seen &= key[None, None, :] > at[:, :, None] - case["window"]
    scores.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(seqs, kv_heads, longest * group, most), vectors("v")).reshape(seqs, kv_heads, longest, group, dim)
    o = o / total
    lse = (top + total.log())[..., 0]
    seq, local, _, _ = _places(case, s)
    o = o.permute(0, 2, 1, 3, 4)[seq, local].reshape(q.shape[0], -1)
    return o.to(TYPES[case["dtype"]]), lse.permute(0, 2, 1, 3)[seq, local].reshape(q.shape[0], -1)


def _plain(case, s):
    op, dim, heads, kv_heads = case["op"], case["dim"], case["heads"], case["kv_heads"]
    if op == "rotary":
        return {"y": _plain_rotary(case, s, heads + kv_heads)}
    if op == "cache":
        cols, back = kv_heads * dim, torch.bfloat16 if case["dtype"] == "f32" else TYPES[case["dtype"]]
        _plain_write(case, s, "k", s["k"][:, :cols])
        _plain_write(case, s, "v", s["v"][:, :cols])
        return {"k": _plain_read(case, s, "k", back), "v": _plain_read(case, s, "v", back)}
    if op == "attend":
        o, lse = _plain_attend(case, s, s["q"][:, : heads * dim])
        return {"o": o, "lse": lse}
    y = _plain_rotary(case, s, heads + kv_heads)
    end = (heads + kv_heads) * dim
    _plain_write(case, s, "k", y[:, heads * dim:])
    _plain_write(case, s, "v", s["x"][:, end:end + kv_heads * dim])
    return {"y": y, "o": _plain_attend(case, s, y[:, : heads * dim])[0]}


@functools.lru_cache(maxsize=1)
def _framework():
    """The binding, and the handle that a program keeps."""
    sys.path.insert(0, os.path.join(os.getcwd(), "amdgpu-arch-gemm_amd"))
    from shim import q8_cache as C

    return C, C.Ops()


def _kept(state):
    """What a program makes once of a model's and a batch's sizes."""
    kept = state["kept"]
    if not kept:
        C, _ = _framework()
        case, b = state["case"], state["buffers"]
        if case["op"] in ("rotary", "step"):
            kept["form"] = C.Rotation(case["dim"], _axis(case), case["axes"], case["neighbours"])
        if case["op"] != "rotary":
            kept["cache"] = C.Cache(b["cache_k"], b["cache_v"], b["scale_k"], b["scale_v"], state["in"]["cache_k"].shape[0],
                                    case["page"], case["kv_heads"], case["dim"])
            kept["batch"] = C.Batch(b["starts"], b["lengths"], b["table"], case["seqs"], _tokens(case), _width(case),
                                    longest=max(_lengths(case)[0]))
    return kept


class _At:
    """A place in a buffer."""

    def __init__(self, b, values):
        self.ptr = b.ptr + values * b.tensor.element_size()


def _kernels(state):
    C, ops = _framework()
    case, out, b, kept = state["case"], state["out"], state["buffers"], _kept(state)
    op, dim, heads, kv_heads, pad = case["op"], case["dim"], case["heads"], case["kv_heads"], case["pad"]
    types = {"f32": C.F32, "f16": C.F16, "bf16": C.BF16}
    dtype, all_heads = types[case["dtype"]], heads + kv_heads
    if op == "rotary":
        ld = all_heads * dim + pad
        ops.rotary(dtype, kept["form"], b["x"], b["positions"], b["freq"], b["out_y"], out["y"].shape[0], all_heads, ldx=ld, ldy=ld,
                   inverse=case["inverse"])
        return {"y": out["y"][:, : all_heads * dim]}
    if op == "cache":
        ld = kv_heads * dim + pad
        ops.cache_write(dtype, kept["cache"], kept["batch"], b["k"], b["v"], ldk=ld, ldv=ld)
        ops.cache_read(C.BF16 if case["dtype"] == "f32" else dtype, kept["cache"], kept["batch"], b["out_k"], b["out_v"])
        return {"k": out["k"], "v": out["v"]}
    ldo = heads * dim + pad
    if op == "attend":
        ops.attention(dtype, kept["cache"], kept["batch"], heads, b["q"], b["out_o"], b["out_lse"], scale=dim ** -0.5,
                      window=case["window"], ldq=ldo, ldo=ldo)
        return {"o": out["o"][:, : heads * dim], "lse": out["lse"]}
    ldx, ldy = (all_heads + kv_heads) * dim + pad, all_heads * dim + pad
    ops.rotary(dtype, kept["form"], b["x"], b["positions"], b["freq"], b["out_y"], out["y"].shape[0], all_heads, ldx=ldx, ldy=ldy)
    ops.cache_write(dtype, kept["cache"], kept["batch"], _At(b["out_y"], heads * dim), _At(b["x"], all_heads * dim), ldk=ldy, ldv=ldx)
    ops.attention(dtype, kept["cache"], kept["batch"], heads, b["out_y"], b["out_o"], None, scale=dim ** -0.5, ldq=ldy, ldo=ldo)
    return {"y": out["y"][:, : all_heads * dim], "o": out["o"][:, : heads * dim]}


def run(state):
    if own:
        return _kernels(state)
    return _plain(state["case"], state["in"])


def _pairs_seen(case):
    """(Keys read, pairs of a new token and a key it sees) of all sequences."""
    keys = pairs = 0
    window = case["window"] or 1 << 40
    for n, t in zip(*_lengths(case)):
        keys += min(t, n - 1 + window)
        full = max(0, min(n, t - window + 1)) if window <= t else 0      # new tokens that see a whole window
        rest = n - full
        pairs += full * window + rest * (t - n + 1) + rest * (rest - 1) // 2
    return keys, pairs


def work(case):
    op, dim, heads, kv_heads, tokens = case["op"], case["dim"], case["heads"], case["kv_heads"], _tokens(case)
    size = 4 if case["dtype"] == "f32" else 2
    turned = tokens * (heads + kv_heads) * dim
    rotary = {"bytes": 2 * turned * size + 4 * tokens * case["axes"] + 4 * case["pairs"], "flops": 3 * turned}
    chunk = 2 * tokens * kv_heads * dim
    rows = 2 * tokens * kv_heads
    if op == "rotary":
        return rotary
    if op == "cache":       # in, the cache, and out
        return {"bytes": chunk * (size + 1 + 2) + 4 * rows, "flops": 6 * chunk}
    keys, pairs = _pairs_seen(case)
    attend = {"bytes": 2 * keys * kv_heads * (dim + 4) + 2 * tokens * heads * dim * size + (4 * tokens * heads if op == "attend" else 0),
              "flops": 4 * dim * heads * pairs}
    if op == "attend":
        return attend
    # the new keys and values are read once, from the product's rows; turned queries and keys are an output
    return {"bytes": rotary["bytes"] + chunk // 2 * size + attend["bytes"] - tokens * heads * dim * size, "flops": rotary["flops"] + 6 * chunk + attend["flops"]}


def exact(case, seed):
    s = _inputs(case, seed)
    op, dim, heads, kv_heads, page = case["op"], case["dim"], case["heads"], case["kv_heads"], case["page"]
    dtype = TYPES[case["dtype"]]

    def turn(x, h):
        x = x[:, : h * dim].double().reshape(-1, h, dim)
        axis, p = _axis(case), case["pairs"]
        sign = -1.0 if case["inverse"] else 1.0
        y = x.clone()
        for j in range(p):
            a = s["positions"][axis[j]].double() * s["freq"][j].double()
            turned = torch.polar(torch.ones_like(a), sign * a)[:, None]
            i1, i2 = (2 * j, 2 * j + 1) if case["neighbours"] else (j, p + j)
            z = torch.complex(x[:, :, i1], x[:, :, i2]) * turned
            y[:, :, i1], y[:, :, i2] = z.real, z.imag
        return y.reshape(x.shape[0], -1)

    def to_8_bits(x):
        """Rows of heads as 8-bit steps, and their size, as 32 bits hold it."""
        x = x.double().reshape(-1, kv_heads, dim)
        step = torch.maximum(x.abs().max(2).values / 127, torch.full((), 2.0 ** -126, dtype=torch.float64, device=x.device))
        return torch.round(x / step.unsqueeze(2)), step.unsqueeze(2)

    if op == "rotary":
        return {"y": turn(s["x"], heads + kv_heads)}
    if op == "cache":
        return {name: torch.mul(*to_8_bits(s[name][:, : kv_heads * dim])).reshape(-1, kv_heads * dim) for name in ("k", "v")}
    table, group = s["table"].cpu().tolist(), heads // kv_heads
    answer = {}
    new = None
    if op == "step":
        y = turn(s["x"], heads + kv_heads)
        answer["y"] = y
        y = y.to(dtype)       # as it is stored
        end = (heads + kv_heads) * dim
        q = y[:, : heads * dim]
        new = [torch.mul(*to_8_bits(t)) for t in (y[:, heads * dim:], s["x"][:, end:end + kv_heads * dim])]
    else:
        q = s["q"][:, : heads * dim]
    q = q.double().reshape(-1, kv_heads, group, dim)
    o = torch.empty_like(q)
    lse = torch.empty(q.shape[:3], dtype=torch.float64, device=q.device)
    first = 0
    for b, (n, t) in enumerate(zip(*_lengths(case))):
        here = torch.tensor(table[b][: -(-t // page)], device=q.device, dtype=torch.long)
        token = torch.arange(t - n, t, device=q.device)
        for h in range(kv_heads):
            k, v = ((s["cache_" + c][here, h, :, :dim].double() * s["scale_" + c][here, h].double().unsqueeze(-1)).reshape(-1, dim)[:t].clone()
                    for c in ("k", "v"))
            if new is not None:
                k[t - n:], v[t - n:] = new[0][first:first + n, h], new[1][first:first + n, h]
            for r in range(0, n, 1024):
                rows = slice(first + r, first + min(n, r + 1024))
                at = token[r:r + 1024]
                x = torch.mm(q[rows, h].reshape(-1, dim), k.T.contiguous()).reshape(-1, group, t) / math.sqrt(dim)
                hidden = torch.arange(t, device=q.device) > at.unsqueeze(1)
                if case["window"]:
                    hidden |= torch.arange(t, device=q.device) + case["window"] <= at.unsqueeze(1)
                x = x.masked_fill(hidden.unsqueeze(1), -math.inf)
                lse[rows, h] = torch.logsumexp(x, 2)
                o[rows, h] = torch.mm(torch.softmax(x, 2).reshape(-1, t), v).reshape(-1, group, dim)
        first += n
    answer["o"] = o.reshape(o.shape[0], -1)
    if op == "attend":
        answer["lse"] = lse.reshape(o.shape[0], -1)
    return answer
