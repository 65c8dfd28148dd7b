"""Attentions that together reach every kernel and every way that keys are cut: dtype, (new, all) tokens of the sequences,
heads, heads of the cache, dim, page, longest; and what runs: kernel -> pieces, "join" where more than one."""

ROUTES = {
    "decoding": ("bf16", [(1, 300)] * 40, 8, 4, 128, 16, 1, {"few": 3}),
    "decoding, one piece": ("f16", [(1, 130), (1, 127)] * 80, 8, 8, 64, 16, 1, {"few": 1}),
    "one token over a long cache": ("f32", [(1, 9000)], 2, 1, 128, 16, 1, {"few": 71}),
    "as many rows as few takes": ("bf16", [(16, 700), (16, 300), (3, 40)], 4, 1, 128, 16, 16, {"few": 6}),
    "one row more": ("bf16", [(17, 700), (16, 300), (3, 40)], 4, 1, 128, 16, 17, {"few": 6, "many": 11}),
    "a chunk": ("f16", [(60, 900)], 2, 1, 96, 16, 60, {"many": 15}),
    "a chunk, FP32": ("f32", [(60, 900)], 2, 1, 128, 16, 60, {"many": 15}),
    "a chunk of wide heads": ("bf16", [(70, 500)], 2, 2, 200, 16, 70, {"many": 8}),
    "chunks of one piece": ("f16", [(40, 60), (50, 50), (33, 64)], 4, 2, 64, 64, 50, {"few": 1, "many": 1}),
    "a prompt": ("bf16", [(520, 520)], 8, 4, 128, 16, 520, {"prompt": 9}),
    "a prompt after others": ("f16", [(600, 1100)], 2, 1, 64, 16, 600, {"prompt": 9}),
    "a prompt in one piece": ("bf16", [(1030, 1100)], 32, 32, 80, 16, 1030, {"prompt": 1}),
    "prompts": ("f16", [(600, 700), (560, 560)], 4, 2, 80, 16, 600, {"few": 6, "prompt": 11}),
    "a prompt, FP32": ("f32", [(520, 520)], 4, 2, 64, 16, 520, {"many": 9}),
    "a prompt of wide heads": ("f16", [(520, 520)], 4, 2, 160, 16, 520, {"many": 9}),
    "not known": ("bf16", [(1, 300), (1, 40), (1, 7)], 8, 4, 128, 16, 0, {"few": 3}),
}


def width(sequences, page):
    return max(-(-t // page) for _, t in sequences)
