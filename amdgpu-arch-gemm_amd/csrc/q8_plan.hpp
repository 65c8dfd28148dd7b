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
// Fewest tokens that the tile kernels are used for; below, the weights are streamed once.
constexpr uint32_t kFewTokens = 64;

struct Tile {
    uint32_t m, n, resident;   // resident: work-groups of it on a CU
};
constexpr Tile kTiles[] = {{256, 256, 1}, {128, 128, 2}};
constexpr int kTileKinds = 2;

struct ProductPlan {
    int kind = 0;
    uint32_t splits = 1;
    size_t partial_bytes = 0;
};

constexpr uint64_t div_up(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// m x n outputs over kb bytes of the summed index.
inline ProductPlan plan_product(uint64_t m, uint64_t n, uint64_t kb) {
    ProductPlan best;
    double least = 1e300;
    const uint64_t tiles_k = div_up(kb ? kb : 1, kTileBytes);
    for (int kind = 0; kind < kTileKinds; ++kind) {
        const Tile& t = kTiles[kind];
        const uint64_t tiles = div_up(m, t.m) * div_up(n, t.n);
        const uint64_t slots = (uint64_t)kComputeUnits * t.resident;
        // a K tile of 256 x 256 takes a work-group about four times as long as one
        // of 128 x 128 on a CU of its own, and two of the latter share a CU
        const double step = kind == 0 ? 1.0 : 0.62;
        for (uint32_t s = 1; s <= kMaxSplits; ++s) {
            if (s > 1 && (tiles >= slots || tiles_k / s < 4)) break;
            const double rounds = (double)div_up(tiles * s, slots);
            const double fixed = 3.0 + (s > 1 ? 3.0 + 0.5 * s : 0.0);
            const double cost = rounds * ((double)div_up(tiles_k, s) + fixed) * step;
            if (cost < least * 0.999) {
                least = cost;
                best.kind = kind;
                best.splits = s;
            }
        }
    }
    const Tile& t = kTiles[best.kind];
    const uint64_t tiles = div_up(m, t.m) * div_up(n, t.n);
    // whole ranges: none of the splits is empty
    best.splits = (uint32_t)div_up(tiles_k, div_up(tiles_k, best.splits));
    if (best.splits > 1) {
        best.partial_bytes = (size_t)(tiles * best.splits * t.m * t.n * 4);
    }
    return best;
}

}  // namespace q8
