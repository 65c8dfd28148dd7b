"""Launches of an attention over the cache (csrc/cache_plan.hpp) have a tile for every row, whatever the chunks, on the CPU."""
import os
import subprocess

import pytest

from shim import q8_cache as C
from shim import sgemm_shim as S

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "amdgpu-arch-gemm_amd", "csrc")

# Chunks of `seqs` sequences with `tokens` rows in all, and the tiles that the kernels find in them: of a sequence of rows in
# (least, most] as many as its rows fill.  Every sequence that has rows is one launch's, and no launch has fewer slots than tiles.
PROGRAM = r"""
#include "cache_plan.hpp"
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>
using namespace q8;
typedef std::vector<uint64_t> Chunks;
static uint64_t plans = 0;
static void check(bool f32, uint64_t group, uint64_t kv, uint32_t dim, uint64_t keys, const Chunks& chunks, uint64_t spare) {
    uint64_t tokens = spare, most = 0;
    for (uint64_t n : chunks) { tokens += n; most = std::max(most, n); }
    for (uint64_t longest : {most, (uint64_t)0, (uint64_t)1, most / 2, most + 1, tokens, (uint64_t)UINT32_MAX}) {
        const AttentionPlan p = plan_attention(f32, tokens, chunks.size(), keys, longest, kv * group, kv, dim);
        uint64_t tiles[2] = {0, 0};
        for (uint64_t n : chunks) {
            int launches = 0;
            for (int i = 0; i < 2; ++i) {
                const AttentionLaunch& l = i ? p.many : p.few;
                const uint64_t rows = n * group, height = i ? many_rows(f32, dim) : kFewRows;
                if (!l.slots || rows <= l.least || rows > l.most) continue;
                tiles[i] += up(rows, height);
                ++launches;
            }
            if (n && launches != 1) { std::printf("a sequence of %llu tokens has %d launches\n", (unsigned long long)n, launches); std::exit(1); }
        }
        if (tiles[0] > p.few.slots || tiles[1] > p.many.slots) {
            std::printf("%llu and %llu tiles in %u and %u slots: %llu tokens, %zu sequences, longest %llu, group %llu, %u values%s\n",
                        (unsigned long long)tiles[0], (unsigned long long)tiles[1], p.few.slots, p.many.slots, (unsigned long long)tokens,
                        chunks.size(), (unsigned long long)longest, (unsigned long long)group, dim, f32 ? ", FP32" : "");
            std::exit(1);
        }
        ++plans;
    }
}
int main() {
    std::mt19937 rng(1);
    auto any = [&](uint64_t lo, uint64_t hi) { return lo + rng() % (hi - lo + 1); };
    for (uint64_t group : {1, 3, 4, 7, 16, 64, 65, 128}) for (uint32_t dim : {64, 128, 256}) for (int f32 = 0; f32 < 2; ++f32)
        for (uint64_t kv : {1, 8}) for (uint64_t seqs : {1, 2, 5, 64, 65, 300}) {
        std::vector<Chunks> cases;
        // all alike, on both sides of each tile's height and of the most rows of few
        for (uint64_t rows : {1, 15, 16, 17, 63, 64, 65, 79, 80, 81, 127, 128, 129, 255, 256, 257, 1024, 5000})
            for (uint64_t n : {rows / group, up(rows, group), rows / group + 1}) cases.push_back(Chunks(seqs, n));
        // one long, the others of one token, none or just past the most rows of few
        for (uint64_t other : {(uint64_t)0, (uint64_t)1, kFewMost / group, kFewMost / group + 1}) for (uint64_t n : {65, 300, 8192}) {
            cases.push_back(Chunks(seqs, other));
            cases.back()[any(0, seqs - 1)] = n;
        }
        // by turns two kinds; at random, many of them empty
        Chunks turns(seqs);
        for (uint64_t b = 0; b < seqs; ++b) turns[b] = b % 2 ? kFewMost / group + 1 : 1;
        cases.push_back(turns);
        for (int i = 0; i < 20; ++i) {
            Chunks c(seqs);
            const uint64_t hi = 1ull << any(0, 10);
            for (uint64_t& n : c) n = any(0, 3) ? any(0, hi) : 0;
            cases.push_back(c);
        }
        for (const Chunks& c : cases)
            for (uint64_t keys : {0, 300, 8192, 131072}) check(f32, group, kv, dim, keys, c, any(0, 1) * any(0, 40));
    }
    std::printf("ok %d\n", plans > 100000);
}
"""


def test_every_row_has_a_tile(tmp_path):
    source = tmp_path / "tiles.cpp"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", CSRC, str(source),
                    "-o", str(tmp_path / "tiles")], check=True)
    out = subprocess.run([str(tmp_path / "tiles")], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "ok 1", out.stdout + out.stderr


def test_no_grid_passes_2_to_the_32_work_items():
    """A tile of many rows has eight waves, 2^23 of them are more than a grid holds: such sizes are refused before a launch."""
    cache = C.Cache(None, None, None, None, 4, 16, 64, 1)
    for seqs in (1, 2):
        C.attention_workspace(C.BF16, cache, C.Batch(None, None, None, seqs, 2 ** 24, 8), 64)
        with pytest.raises(S.SgemmError) as e:
            C.attention_workspace(C.BF16, cache, C.Batch(None, None, None, seqs, 2 ** 25 - 1, 8), 64)
        assert e.value.code == -4 and "grid" in e.value.message
