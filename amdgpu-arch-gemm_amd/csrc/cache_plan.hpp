// How an attention over the cache runs: kernels, pieces of the keys, workspace.  Host
// code without HIP.
#pragma once

#include <cstddef>
#include <cstdint>

namespace q8 {

// Rows of a tile: tokens of one sequence times the heads that share one of the cache's; keys of a step.
constexpr uint32_t kFewRows = 16, kFewKeys = 128;
constexpr uint32_t kManyKeys = 64;
// A sequence of so many rows still goes in tiles of few.  8 sequences of 64 rows over 4096 keys: 43 us, in one of many's
// tiles each 70; 16 of up to 132 rows: 121 and 116.
constexpr uint32_t kFewMost = 64;
// Tiles whose keys are taken in pieces, at the most: each has a ticket in the handle.
constexpr uint32_t kTickets = 1u << 16;
// Pieces: the grid's second dimension ends at 65535, the grid at 2^32 work-items (kMostGroups work-groups of 256); and their
// sums stay small beside a cache.
constexpr uint64_t kMostPieces = 4096, kMostGroups = (1u << 24) - 1, kMostSumBytes = 1ull << 28;

constexpr uint64_t up(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// Values of a head as the kernels hold them.
constexpr uint32_t held_dim(uint32_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
// Rows of a tile of many: 32 a wave, of eight waves, or of four that have the registers of two each.
constexpr uint32_t many_rows(bool f32, uint32_t dim) { return f32 || dim > 128 ? 128 : 256; }

// 64 keys and values as 16-bit values, and their scales.
constexpr uint32_t image_bytes(uint32_t held) { return 64 * (held * 2 + 16) + held * 144 + 1024; }
// Images are made beforehand from so many rows a sequence on, if they take no more workspace than this.  Over 8192 keys
// (bf16, 8 heads of the cache, 4 heads each): 64 tokens (256 rows) 74 us with images and 42 without, 128 tokens 77 and 70;
// 16 prompts of up to 300 tokens 90 and 69; 256 tokens over 32768 keys 210 and 226; 8192 tokens 628 and 719.  Their workspace, too, is
// by the table's width: 16 prompts of 2048 take 1053 us, and with a table for 32768 positions, without images, 1109.
constexpr uint64_t kImageRows = 1024, kMostImageBytes = 1ull << 30;

struct AttentionLaunch {
    uint32_t slots = 0;         // tiles there may be; 0: no launch
    uint32_t least = 0, most = UINT32_MAX;
    uint32_t piece = 0;         // keys of a piece
    uint32_t pieces = 1;        // of the longest sequence
    uint64_t most_groups = kMostGroups;
};
struct AttentionPlan {
    AttentionLaunch few, many;
    uint32_t images = 0;        // of a sequence and head of the cache, for `many`; 0: none
    size_t image_bytes = 0;     // workspace: images, then the pieces' sums
    size_t bytes = 0;
};

// The keys of a sequence in pieces: as many as make `groups` work-groups of `tiles`, and none longer than `longest` keys; at
// most `at_most`, and no more than a grid of the slots and the `heads` of the cache can hold.  `keys` is the table's width, as
// the host does not know the lengths, so a table far wider than they are makes pieces too long (a token over 4096 keys takes
// 13.5 us with a table for 4096 or 32768 positions and 28 with one for 131072; 8 such sequences 21, 46 and 61).
inline void cut(AttentionLaunch& l, uint64_t heads, uint64_t tiles, uint64_t keys, uint64_t step, uint64_t groups, uint64_t longest,
                uint64_t at_most) {
    const uint64_t steps = up(keys ? keys : 1, step);
    uint64_t most = groups / tiles ? groups / tiles : 1;
    const uint64_t limits[] = {steps, at_most, l.most_groups / (l.slots * heads), l.slots * heads > kTickets ? 1 : kMostPieces};
    if (most < up(keys, longest)) most = up(keys, longest);
    for (uint64_t limit : limits)
        if (most > limit) most = limit ? limit : 1;
    const uint64_t each = up(steps, most);
    l.piece = (uint32_t)(each * step);
    l.pieces = (uint32_t)up(steps, each);
}

inline AttentionPlan plan_attention(bool f32, uint64_t tokens, uint64_t seqs, uint64_t keys, uint64_t longest, uint64_t heads,
                                    uint64_t kv_heads, uint32_t dim) {
    AttentionPlan p;
    if (!tokens || !seqs) return p;
    const uint64_t group = heads / kv_heads, rows = tokens * group, filled = seqs < tokens ? seqs : tokens;
    if (!longest || longest > tokens) longest = tokens;
    const bool few = longest * group <= kFewMost || seqs > 1, many = longest * group > kFewMost;
    if (few) {
        p.few.slots = (uint32_t)(rows / kFewRows + filled);
        if (many) {
            p.few.most = p.many.least = kFewMost;
            if (p.few.slots > filled * up(kFewMost, kFewRows)) p.few.slots = (uint32_t)(filled * up(kFewMost, kFewRows));
        }
        // One sequence fills the card at once: 131072 keys of 8 heads take 64 us in 512 work-groups, in 256 93 and in 1024
        // 83.  Of several, whose lengths differ, the longest alone is left at the end: 64 of up to 8192 keys take 133 us in
        // pieces of at most 4096, of 2048 137, of 1024 142, and 183 whole.
        const uint64_t each = tokens * heads * (held_dim(dim) + 2) * 4;
        cut(p.few, kv_heads, p.few.slots * kv_heads, keys, kFewKeys, seqs > 1 ? 1024 : 512, 4096, kMostSumBytes / each);
    }
    if (many) {
        const uint32_t height = many_rows(f32, dim);
        const uint64_t own = rows / kFewMost < filled ? rows / kFewMost : filled;      // sequences of more rows than few
        p.many.slots = (uint32_t)(rows / height + (own ? own : 1));
        p.many.most_groups = kMostGroups * 128 / height;      // two work-items a row
        // One work-group a CU, two where their registers and images are small; twice that of several sequences, whose tiles
        // end at different times (4 of 512 tokens over up to 8192 keys: 311 us, in 1024 work-groups 346).  FP32, 512 tokens
        // over 2048 keys: 85 us in two pieces, 147 in one.  A piece costs its
        // sums' way through memory: 64 tokens over 8192 keys take 42 us in 16 pieces, 54 in 32.
        const uint64_t each_cu = !f32 && dim <= 64 ? 512 : 256;
        cut(p.many, kv_heads, (seqs > 1 ? p.many.slots : up(rows, height)) * kv_heads, keys, kManyKeys,
            seqs > 1 ? 2 * each_cu : each_cu, UINT32_MAX, 16);
    }
    const uint64_t each = up(keys, kManyKeys), image = each * kv_heads * seqs * image_bytes(held_dim(dim));
    if (many && !f32 && dim <= 128 && rows >= kImageRows * seqs && image && image <= kMostImageBytes && each <= kMostImageBytes) {
        p.images = (uint32_t)each;
        p.image_bytes = (size_t)image;
    }
    p.bytes = p.image_bytes;
    const uint64_t pieces = p.few.pieces > p.many.pieces ? p.few.pieces : p.many.pieces;
    if (pieces > 1) p.bytes += (size_t)pieces * tokens * heads * (held_dim(dim) + 2) * 4;
    return p;
}

}  // namespace q8
