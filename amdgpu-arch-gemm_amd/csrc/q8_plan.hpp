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
// The longest sum of a gradient whose operands are laid out, of 16-bit values in `terms` terms each: a
// row holds a multiple of eight values.
constexpr uint64_t most_summed(uint32_t terms) { return kMaxRowBytes / (2 * terms) / 8 * 8; }
// Up to so many tokens the weights are streamed once, from rows that start anywhere.
constexpr uint32_t kFewTokens = 64;
// So many scales are looked through by every work-group that needs their largest, which costs
// less than a launch.
constexpr uint32_t kFewScales = 4096;

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

// The next column, after c < cols, of a thread that takes one of every `step`; `cols` after its last.  (A
// plain sum of 32 bits passes 2^32 in the widest rows, starts again below `cols` and never ends.)
constexpr uint32_t next_column(uint32_t c, uint32_t step, uint32_t cols) { return cols - c > step ? c + step : cols; }

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

// K tiles of a work-group, and whether it asks L2 for the next ones' lines (256 x 256 tiles): a second round of work-groups
// finds its lines in memory, and in a deep K they drift apart; one round of few K tiles is 2% faster unasked.
constexpr uint64_t tiles_per_split(uint64_t kb, uint32_t splits) { return div_up(div_up(kb, kTileBytes), splits); }
constexpr bool asks_ahead(uint64_t groups, uint64_t tiles) { return groups > kComputeUnits || tiles > 32; }

// The direct kernel's tiles, 16 MT tokens x 16 NT channels a work-group of WAVES waves.  Times in us at the sizes named, with
// 400 MB of weights and more in turn, as a model's layers follow one another; weights that the last-level cache
// holds favour other tiles in places (1 x 4 at 1 x 12288 x 4096 by 5%, 16 waves at 1 x 4096 x 16384 by 11%).
//   1 x 1, 8 waves   up to 16 tokens (16 x 4096 x 4096 6.5, one token 5.6); 16 waves gain 4% at most and cost
//                    up to 14% (1 x 4096 x 10240 10.0 against 9.8, x 12288 13.0 against 11.3)
//   1 x 4, 8 waves   the same into many channels: four times the tokens' operands for a work-group's weights, a quarter of the
//                    work-groups, so it pays where the tokens weigh and where K is short.  16 x 16384 x 4096 19.3
//                    against 21.2, x 12288 16.4 and 16.9, x 11264 15.7 and 15.9; 1 x 12288 x 1024 5.6 and
//                    6.0, x 2048 7.8 and 8.1, x 3000 18.9 and 15.5, x 8192 27.2 and 19.1; x 4096 of 8, 12 and 16 tokens into 16384
//                    18.3 and 18.1, 18.9 and 19.7, 19.3 and 21.2
//   1 x 1, 16 waves  a small product of more tokens: a work-group a CU (333 x 129 x 517: 4.2, 2 x 1 5.2)
//   2 x 1, 2 x 4     up to 32 tokens.  2 x 4 once 2 x 1 has more than two work-groups a CU: 32 x 8704 x 4096 17.3 against
//                    20.4, x 16384 22.2 and 29.5, but x 8192 17.0 and 15.4
//   2 x 2, 4 x 4     and up to 64, with the same bound: 64 x 8704 x 4096 23.9 against 28.3, x 16384 28.8 and
//                    42.0, but x 8192 23.5 and 21.5 (64 x 4096 x 4096: 2 x 1 14.1, 4 x 1 12.5, 2 x 2 10.4)
enum Direct { D_1x1_16, D_1x1_8, D_1x4_8, D_2x1_8, D_2x4_8, D_2x2_8, D_4x4_4 };
inline Direct direct_kind(uint64_t m, uint64_t n, uint64_t k) {
    if (m <= 16) return n >= 12288 && (m >= 12 || k <= 2048) ? D_1x4_8 : D_1x1_8;
    if (div_up(m, 16) * div_up(n, 16) <= kComputeUnits) return D_1x1_16;
    const bool wide = n > 2 * kComputeUnits * 16;
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

// The kernel that takes a gradient from operands as they are: rows of a work-group without and
// with a turn of the 16-bit operand, and 64 columns.
constexpr uint32_t kGradientRows[2] = {64, 128};
inline uint64_t gradient_groups(bool turned, uint64_t rows, uint64_t cols) {
    return div_up(rows, kGradientRows[turned]) * div_up(cols, 64);
}
// Its waves, which share the summed index: eight where no work-group waits and each still has
// two steps (BF16, not turned, 64 x 4224 x 924: 8.3 us, four 9.1; 874 x 128 x 106: 4.7 and 4.2).  Turned FP32
// operands are three terms of 64 values a lane, and 512 registers: four.
inline uint32_t gradient_waves(bool turned, bool f32, uint64_t rows, uint64_t cols, uint64_t sum) {
    return gradient_groups(turned, rows, cols) <= kComputeUnits && sum > 512 && !(turned && f32) ? 8 : 4;
}
// Its time in microseconds, fitted to launches back to back: a fixed one and, for each 32 values that a
// wave takes of the summed index, one; with more work-groups than CUs one for each round of
// them, of which a short last one (half a round and less) overlaps the one before where a CU has
// two.  Rows of 16-bit values that start between dwords (odd) take more loads: 1024 x 1024 x 1024 9.0 us, 1024 x
// 1024 x 1025 10.6 (by loads from where they start 3000 x 1003 x 1001 34 us, so 27).
inline double gradient_time(bool turned, bool f32, bool odd, uint64_t rows, uint64_t cols, uint64_t sum) {
    const uint64_t groups = gradient_groups(turned, rows, cols);
    const uint32_t waves = gradient_waves(turned, f32, rows, cols, sum);
    const double k = (double)div_up(sum, 32 * waves);
    const double fixed = turned ? 4.2 : 3.0, pieces = !odd ? 1.0 : turned ? 1.15 : 1.35;
    if (groups <= kComputeUnits) {
        constexpr double step[2][2][2] = {{{0.75, 1.2}, {1.45, 2.4}}, {{1.0, 1.65}, {2.25, 2.25}}};
        return fixed + pieces * step[turned][f32][waves == 8] * k;
    }
    const uint64_t slots = turned && f32 ? kComputeUnits : 2 * kComputeUnits, rest = groups % slots;
    const double rounds = (double)(groups / slots) + (!rest ? 0.0 : rest > slots / 2 || (turned && f32) ? 1.0 : turned ? 0.7 : 0.4);
    const double round = turned ? fixed + (f32 ? 2.25 : 1.75) * k : f32 ? 1.9 + 2.2 * k : 1.4 + 1.32 * k;
    return (turned ? 0.0 : fixed) + pieces * rounds * round;
}
// Whether a gradient is taken so, rather than laid out (`packed_bytes` read and written) and multiplied by the
// kernels above in `tile_time`: it has no fewer values than a lane's loads take, and in F16 the scales
// are few.  (BF16, turned / not, direct and laid out: 512^3 8.0 and 12.5 us / 6.0 and 12.0, 1024^3 11.1 and 17.6 /
// 9.0 and 15.8, 2048 x 2048 x 1024 17.3 and 21.9 / 24.8 and 19.0; FP32 512^3 13.1 and 20.0 / 8.9 and 17.7,
// 300 x 300 x 2000 40 and 25 / 22 and 24.  Over 80 random sizes that the fit has not seen the choice costs 0.3% more
// than the better one on average, 16% at most.)
inline bool gradient_direct(bool turned, bool f32, bool f16, bool odd, uint64_t rows, uint64_t cols, uint64_t sum, double tile_time,
                            uint64_t packed_bytes) {
    if (cols < 4 || sum < (turned ? 1u : 32u) || (turned && rows < 8) || (f16 && sum > kFewScales)) return false;
    // 2^32 work-items are one grid's end
    if (rows > (1u << 22) || gradient_groups(turned, rows, cols) >= (1u << 22)) return false;
    return 1.05 * gradient_time(turned, f32, odd, rows, cols, sum) < tile_time + 3.0 + (double)packed_bytes / 3e6;
}

constexpr uint64_t round_up(uint64_t x, uint64_t to) { return (x + to - 1) / to * to; }

// A call's parts of the workspace, one after the other.
struct Layout {
    size_t a = 0, b = 0, pair = 0, partial = 0, total = 0;
    void add(size_t& at, size_t bytes) {
        at = total;
        total += piece(bytes);
    }
    static constexpr size_t piece(size_t bytes) { return (bytes + 255) & ~(size_t)255; }
};

// How an 8-bit product runs: on the direct kernel, or on tiles, of rows that are copied first where copy_a
// and copy_b say so.
struct GemmPlan {
    bool direct = false, copy_a = false, copy_b = false;
    uint64_t ldc = 0;   // bytes of a copied row
    ProductPlan plan;
    Layout at;
};
inline GemmPlan plan_gemm(uint64_t m, uint64_t n, uint64_t k, bool copy_a, bool copy_b) {
    GemmPlan g;
    g.ldc = round_up(k, 16);
    g.plan = plan_product(m, n, k);
    g.direct = m <= kFewTokens || direct_for_many(m, n, k, g.plan.time, (int)copy_a + (int)copy_b,
                                                  (copy_a ? m * g.ldc : 0) + (copy_b ? n * g.ldc : 0));
    if (g.direct) return g;
    g.copy_a = copy_a;
    g.copy_b = copy_b;
    if (copy_a) g.at.add(g.at.a, m * g.ldc);
    if (copy_b) g.at.add(g.at.b, n * g.ldc);
    if (g.plan.partial_bytes) g.at.add(g.at.partial, g.plan.partial_bytes);
    return g;
}

// How the gradient D (rows x cols) summed over `sum` runs.
struct GradPlan {
    bool direct = false;    // from the operands as they are; else:
    uint64_t cp = 0;        // values of the summed index in a laid-out row
    uint32_t terms = 1;
    uint64_t kb = 0;        // its bytes
    uint64_t pitch = 0;     // and those from one row to the next
    ProductPlan plan;
    Layout at;
};
constexpr uint32_t grad_terms(bool f32) { return f32 ? 3 : 1; }
// copy_a: the 16-bit operand would be laid out too, turned: it has the summed index from row to row, odd: its
// rows start between dwords.  sum <= most_summed(terms).
inline GradPlan plan_grad(bool f32, bool f16, bool turned, bool odd, uint64_t rows, uint64_t cols, uint64_t sum, bool copy_a) {
    GradPlan g;
    g.cp = round_up(sum, 8);
    g.terms = grad_terms(f32);
    g.kb = g.cp * g.terms * 2;
    // whole lines, and not a multiple of 4096 bytes (F16, 4096 x 4096 x 16384: 396 us as it is, 386 with 512
    // bytes more; 1024 x 1024 x 16384 in four ranges: 46 and 47, but 60 with 128)
    g.pitch = round_up(g.kb, 128);
    if (g.pitch % 4096 == 0) g.pitch += 512;
    g.plan = plan_product(rows, cols, g.kb);
    copy_a = copy_a || f32;
    const uint64_t bytes = cols * (sum + g.kb) + (copy_a ? rows * (sum * (f32 ? 4 : 2) + g.kb) : 0);
    g.direct = gradient_direct(turned, f32, f16, odd, rows, cols, sum, g.plan.time, bytes);
    if (g.direct) return g;
    if (copy_a) g.at.add(g.at.a, rows * g.pitch);
    g.at.add(g.at.b, cols * g.pitch);
    if (f16) g.at.add(g.at.pair, 8);
    if (g.plan.partial_bytes) g.at.add(g.at.partial, g.plan.partial_bytes);
    return g;
}

}  // namespace q8
