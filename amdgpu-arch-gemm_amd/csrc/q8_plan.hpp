// How the products of the 8-bit operators run: tile, K ranges, workspace.  Host
// code without HIP.
#pragma once

#include <cstddef>
#include <cstdint>

namespace q8 {

constexpr uint32_t kComputeUnits = 256;
constexpr uint32_t kTileBytes = 128;         // of the summed index, a K tile
constexpr uint32_t kMaxSplits = 16;
// A tile's rows are addressed with 32-bit offsets from its first one.
constexpr uint64_t kMaxRowBytes = 1u << 22;
// Up to so many tokens the weights are streamed once, from rows that start anywhere.
constexpr uint32_t kFewTokens = 64;

struct Tile {
    uint32_t m, n;
};
// The kernels of a product: 256 x 256 tiles, one work-group a CU; 128 x 128 ones, two work-groups a
// CU with two buffers each; the same with three buffers, one work-group a CU.
enum Kind { K_LARGE = 0, K_SMALL = 1, K_SMALL_DEEP = 2, K_KINDS = 3 };
constexpr Tile kTiles[K_KINDS] = {{256, 256}, {128, 128}, {128, 128}};

struct ProductPlan {
    int kind = 0;
    uint32_t splits = 1;
    size_t partial_bytes = 0;
    double time = 0.0;
};

constexpr uint64_t div_up(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// Microseconds of `groups` work-groups of `tiles_k` K tiles each on a kernel, fitted to launches
// back to back: a K tile's time and a fixed one for each round of work-groups.  The large
// tiles take 1.47 us a K tile whether one or all CUs have one (4096^3 in 8-bit integers: 59
// us).  Of the small ones, a CU with two takes 1.0 us for a K tile of both; one alone waits for
// its loads, 0.57 us, and three buffers make that 0.36 (16384 x 128 x 4096 in 8-bit integers: 25.3 ->
// 17.8 us, 2048^3 in BF16: 24.8 -> 18.5; 1024^3, 8 K tiles: 8.0 -> 10.5, as launches overlap less).
inline double product_time(int kind, uint64_t groups, uint64_t tiles_k) {
    const double k = (double)tiles_k;
    if (kind == K_LARGE) return (double)div_up(groups, kComputeUnits) * (1.47 * k + 10.0);
    if (kind == K_SMALL_DEEP) return (double)div_up(groups, kComputeUnits) * (0.36 * k + 7.0);
    const uint64_t slots = 2 * kComputeUnits, rest = groups % slots;
    return (double)(groups / slots) * (1.0 * k + 6.0) + (!rest ? 0.0 : rest <= kComputeUnits ? 0.57 * k + 4.5 : 1.0 * k + 6.0);
}

// m x n outputs over kb bytes of the summed index.
inline ProductPlan plan_product(uint64_t m, uint64_t n, uint64_t kb) {
    ProductPlan best;
    double least = 1e300;
    const uint64_t tiles_k = div_up(kb ? kb : 1, kTileBytes);
    for (int kind = 0; kind < K_KINDS; ++kind) {
        const Tile& t = kTiles[kind];
        const uint64_t tiles = div_up(m, t.m) * div_up(n, t.n);
        for (uint32_t s = 1; s <= kMaxSplits; ++s) {
            // K ranges only where work-groups are idle
            if (s > 1 && (tiles * s > 2 * kComputeUnits || tiles_k / s < 4)) break;
            // the ranges' sums: written, read and finished by another kernel
            const double join = s > 1 ? 3.0 + (s + 1.0) * (double)m * (double)n * 4.0 / 3e6 : 0.0;
            const double time = product_time(kind, tiles * s, div_up(tiles_k, s)) + join;
            if (time < least * 0.999) {
                least = time;
                best.kind = kind;
                best.splits = s;
            }
        }
    }
    best.time = least;
    const Tile& t = kTiles[best.kind];
    const uint64_t tiles = div_up(m, t.m) * div_up(n, t.n);
    // whole ranges: none of the splits is empty
    best.splits = (uint32_t)div_up(tiles_k, div_up(tiles_k, best.splits));
    if (best.splits > 1) best.partial_bytes = (size_t)(tiles * best.splits * t.m * t.n * 4);
    return best;
}

// The direct kernel's tiles, 16 MT tokens x 16 NT channels a work-group of WAVES waves:
//   1 x 1, 16 waves  a small product: a work-group a CU (333 x 129 x 517: 4.2 us, 2 x 1 5.2)
//   1 x 1, 8 waves   up to 16 tokens (16 x 4096 x 4096: 6.9 us; 16 waves 7.2), and 16 waves over
//                    a deep K of few channels (1 x 4096 x 16384: 14.5 against 16.9)
//   1 x 4, 8 waves   up to 16 tokens into many channels: the tokens are read a quarter as often
//                    (16 x 16384 x 4096: 15.8 us, 1 x 1 19.0)
//   2 x 1, 2 x 4     the same up to 32 tokens (32 x 16384 x 4096: 18.4 us, 2 x 1 26.8)
//   2 x 2, 4 x 4     and up to 64 (64 x 4096 x 4096: 10.4 us, 2 x 1 14.1, 4 x 1 12.5;
//                    64 x 16384 x 4096: 25.2 us, 2 x 2 40.8)
enum Direct { D_1x1_16, D_1x1_8, D_1x4_8, D_2x1_8, D_2x4_8, D_2x2_8, D_4x4_4 };
inline Direct direct_kind(uint64_t m, uint64_t n, uint64_t k) {
    const bool wide = n >= 12288;
    if (m <= 16) return wide ? D_1x4_8 : n <= 4096 && k > 8192 ? D_1x1_16 : D_1x1_8;
    if (div_up(m, 16) * div_up(n, 16) <= kComputeUnits) return D_1x1_16;
    if (m <= 32) return wide ? D_2x4_8 : D_2x1_8;
    if (m <= kFewTokens) return wide ? D_4x4_4 : D_2x2_8;
    return D_2x1_8;
}
// Whether more tokens run on it too: a small product, which the tile kernels would spend on
// whole tiles and on copies of rows that are not theirs (`copies` launches, `copy_bytes` in all).
inline bool direct_for_many(uint64_t m, uint64_t n, uint64_t k, double tile_time, int copies, uint64_t copy_bytes) {
    // a grid's second dimension ends at 65535, all of it at 2^32 work-items
    if (m > (1u << 20) || div_up(m, 32) * div_up(n, 16) > (1u << 22)) return false;
    const uint64_t t = div_up(m, 16) * div_up(n, 16);
    const double rows = t <= kComputeUnits ? 32.0 * (double)t : 48.0 * (double)(div_up(m, 32) * div_up(n, 16));
    const double direct = 3.8 + rows * (double)k / 7e6;     // each work-group's rows, out of L2
    return direct < tile_time + 3.0 * copies + 2.0 * (double)copy_bytes / 3e6;
}

}  // namespace q8
