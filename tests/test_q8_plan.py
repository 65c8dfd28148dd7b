"""How the 8-bit operators' products are planned (csrc/q8_plan.hpp), on the CPU."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "q8_plan.hpp"
#include <cstdio>
#include <cstdlib>
using namespace q8;
static void need(bool ok, const char* what, uint64_t m, uint64_t n, uint64_t k) {
    if (!ok) { std::printf("%s: %llu x %llu x %llu\n", what, (unsigned long long)m, (unsigned long long)n, (unsigned long long)k); std::exit(1); }
}
int main() {
    const uint64_t sizes[] = {0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 333, 1000, 1024, 4096, 4097, 16384,
                              100000, 1000000, 1u << 22, 4294967295u};
    int n_split = 0, n_kind[K_KINDS] = {};
    for (uint64_t m : sizes) for (uint64_t n : sizes) for (uint64_t k : sizes) {
        if (!m || !n || k > kMaxRowBytes) continue;
        const ProductPlan p = plan_product(m, n, k);
        ++n_kind[p.kind];
        need(p.kind >= 0 && p.kind < K_KINDS && p.splits >= 1 && p.splits <= kMaxSplits, "kind and splits", m, n, k);
        const uint64_t tiles_k = div_up(k ? k : 1, kTileBytes), per = div_up(tiles_k, p.splits);
        need(per * (p.splits - 1) < tiles_k, "no range is empty", m, n, k);
        const uint64_t tiles = div_up(m, kTiles[p.kind].m) * div_up(n, kTiles[p.kind].n);
        const uint64_t bytes = tiles * p.splits * kTiles[p.kind].m * kTiles[p.kind].n * 4;
        need(p.partial_bytes == (p.splits > 1 ? bytes : 0), "the ranges' sums fit", m, n, k);
        if (p.splits > 1) { ++n_split; need(tiles * p.splits <= 2 * kComputeUnits, "splits only fill idle CUs", m, n, k); }
        const bool many = direct_for_many(m, n, k, p.time, 2, (m + n) * (k + 16));
        if (m > kFewTokens && many) need(div_up(m, 32) <= 65535, "a grid's second dimension", m, n, k);
        if (m <= kFewTokens || many) {
            const Direct d = direct_kind(m, n, k);
            need(d >= D_1x1_16 && d <= D_4x4_4, "a kernel", m, n, k);
            // work-items of the grid
            const uint64_t mt = d == D_2x1_8 || d == D_2x4_8 || d == D_2x2_8 ? 2 : d == D_4x4_4 ? 4 : 1;
            const uint64_t nt = d == D_1x4_8 || d == D_2x4_8 || d == D_4x4_4 ? 4 : d == D_2x2_8 ? 2 : 1;
            const uint64_t threads = d == D_1x1_16 ? 1024 : d == D_4x4_4 ? 256 : 512;
            if (n < (1u << 28)) need(div_up(n, 16 * nt) * div_up(m, 16 * mt) * threads < (1ull << 32), "a grid", m, n, k);
        }
    }
    need(n_split > 0 && n_kind[0] && n_kind[1] && n_kind[2], "every kernel is reached", 0, 0, 0);
    std::puts("ok");
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    d = tmp_path_factory.mktemp("q8_plan")
    source = d / "plan.cpp"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-I", os.path.join(ROOT, "amdgpu-arch-gemm_amd", "csrc"), str(source), "-o", str(d / "plan")], check=True)
    return str(d / "plan")


def test_plans_hold_over_all_sizes(program):
    out = subprocess.run([program], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr


GRADIENTS = r"""
#include "q8_plan.hpp"
#include <cstdio>
using namespace q8;
int main() {
    const uint64_t sizes[] = {1, 3, 4, 7, 8, 31, 32, 33, 64, 128, 129, 512, 513, 1000, 4096, 4097, 16384, 1000000, 2000000,
                              1u << 22, 1u << 28, 4294967295u};
    int direct = 0, eight = 0;
    for (int turned = 0; turned < 2; ++turned) for (int type = 0; type < 3; ++type)
        for (uint64_t r : sizes) for (uint64_t c : sizes) for (uint64_t s : sizes) {
            if (s > 2000000 || !gradient_direct(turned, type == 0, type == 1, false, r, c, s, 1e300, 0)) continue;
            ++direct;
            // what the kernel takes for granted
            bool ok = c >= 4 && (turned ? r >= 8 : s >= 32) && (type != 1 || s <= kFewScales);
            const uint64_t groups = gradient_groups(turned, r, c), waves = gradient_waves(turned, type == 0, r, c, s);
            ok = ok && groups * waves * 64 < (1ull << 32) && (waves == 4 || waves == 8);
            ok = ok && div_up(r, kGradientRows[turned]) * kGradientRows[turned] + 512 < (1ull << 32);
            ok = ok && div_up(c, 64) * 64 < (1ull << 32) && s + 8 * 64 < (1ull << 32);
            ok = ok && !(turned && type == 0 && waves == 8);
            eight += waves == 8;
            if (!ok) { std::printf("%d %d %llu %llu %llu\n", turned, type, (unsigned long long)r, (unsigned long long)c, (unsigned long long)s); return 1; }
        }
    std::puts(direct && eight ? "ok" : "no case");
}
"""


def test_gradients_from_operands_as_they_are(tmp_path):
    source = tmp_path / "gradients.cpp"
    source.write_text(GRADIENTS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-I", os.path.join(ROOT, "amdgpu-arch-gemm_amd", "csrc"), str(source), "-o", str(tmp_path / "gradients")],
                   check=True)
    out = subprocess.run([str(tmp_path / "gradients")], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr
