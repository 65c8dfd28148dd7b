"""How attentions over the cache are planned (csrc/cache_plan.hpp), and that the kernels' sources are all prepared, on the CPU."""
import glob
import os
import re
import subprocess

import pytest

from cache_routes import ROUTES, width
from shim import q8_cache as C

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "amdgpu-arch-gemm_amd", "csrc")

PROGRAM = r"""
#include "cache_plan.hpp"
#include <cstdio>
#include <cstdlib>
#include <initializer_list>
using namespace q8;
static void need(bool ok, const char* what, uint64_t tokens, uint64_t seqs, uint64_t keys, uint64_t heads, uint64_t kv, uint64_t dim) {
    if (ok) return;
    std::printf("%s: %llu tokens, %llu sequences, %llu keys, %llu / %llu heads of %llu\n", what, (unsigned long long)tokens,
                (unsigned long long)seqs, (unsigned long long)keys, (unsigned long long)heads, (unsigned long long)kv, (unsigned long long)dim);
    std::exit(1);
}
int main(int argc, char** argv) {
    if (argc > 1) {
        uint64_t v[8];
        for (int i = 0; i < 8; ++i) v[i] = std::strtoull(argv[1 + i], nullptr, 10);
        const AttentionPlan p = plan_attention(v[0], v[1], v[2], v[3], v[4], v[5], v[6], (uint32_t)v[7]);
        std::printf("%u %u %u %u %u %zu\n", p.few.slots, p.few.pieces, p.many.slots, p.many.pieces, p.images, p.bytes);
        return 0;
    }
    int n = 0;
    typedef std::initializer_list<uint64_t> List;
    for (uint64_t dim : List{1, 64, 65, 128, 129, 256}) for (uint64_t kv : List{1, 3, 8, 64}) for (uint64_t group : List{1, 4, 7})
        for (uint64_t seqs : List{1, 2, 7, 64, 65, 4096, 1000000}) for (uint64_t tokens : List{1, 2, 16, 64, 300, 8192, 1000000})
            for (uint64_t keys : List{0, 1, 64, 129, 5000, 131072, (1ull << 31) - (1u << 16) - 1})
                for (uint64_t longest : List{0, 1, 17, 5000}) for (int f32 = 0; f32 < 2; ++f32) {
        const uint64_t heads = kv * group;
        const AttentionPlan p = plan_attention(f32, tokens, seqs, keys, longest, heads, kv, (uint32_t)dim);
        auto check = [&](bool ok, const char* what) { need(ok, what, tokens, seqs, keys, heads, kv, dim); };
        const uint64_t known = longest && longest < tokens ? longest : tokens;
        check(p.few.slots || p.many.slots, "a launch");
        check(p.few.slots || known * group > kFewMost, "few rows have a launch");
        check(p.many.slots || known * group <= kFewMost, "many rows have a launch");
        if (p.few.slots && p.many.slots) check(p.few.most == p.many.least, "every sequence has one launch");
        size_t sums = 0;
        for (const AttentionLaunch* l : {&p.few, &p.many}) {
            if (!l->slots) continue;
            ++n;
            const uint32_t step = l == &p.few ? kFewKeys : kManyKeys;
            check(l->pieces >= 1 && l->pieces <= kMostPieces && l->piece && l->piece % step == 0, "pieces");
            check((uint64_t)l->piece * l->pieces >= keys && (uint64_t)l->piece * (l->pieces - 1) < (keys ? keys : 1), "pieces cover the keys, none empty");
            check(l->pieces == 1 || (uint64_t)l->slots * kv <= kTickets, "tickets");
            check(l->pieces == 1 || (uint64_t)l->slots * kv * l->pieces <= kMostGroups, "the grid");
            // tiles of sequences that this launch takes: at the most, each sequence has one that is not full
            const uint64_t height = l == &p.few ? kFewRows : many_rows(f32, (uint32_t)dim), rows = tokens * group;
            const uint64_t all = seqs < tokens ? seqs : tokens;
            if (l == &p.few && !p.many.slots) check(l->slots >= rows / height + all, "tiles");
            const size_t own = l->pieces > 1 ? (size_t)l->pieces * tokens * heads * (held_dim((uint32_t)dim) + 2) * 4 : 0;
            check(own <= kMostSumBytes, "the sums are small");
            if (own > sums) sums = own;
        }
        check(p.bytes == sums + p.image_bytes && p.image_bytes <= kMostImageBytes && (!p.images || p.many.slots), "workspace");
    }
    std::printf("ok %d\n", n > 1000);
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    d = tmp_path_factory.mktemp("cache_plan")
    source = d / "plan.cpp"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-I", CSRC, str(source), "-o", str(d / "plan")], check=True)
    return str(d / "plan")


def test_plans_hold_over_all_sizes(program):
    out = subprocess.run([program], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "ok 1", out.stdout + out.stderr


@pytest.mark.parametrize("name", list(ROUTES))
def test_the_sizes_reach_every_kernel(program, name):
    dtype, sequences, heads, kv_heads, dim, page, longest, want = ROUTES[name]
    tokens, keys = sum(n for n, _ in sequences), width(sequences, page) * page
    out = subprocess.run([program] + [str(a) for a in (int(dtype == "f32"), tokens, len(sequences), keys, longest, heads, kv_heads, dim)],
                         capture_output=True, text=True, check=True).stdout
    few, few_pieces, many, many_pieces, images, size = map(int, out.split())
    got = {}
    if few:
        got["few"] = few_pieces
    if many:
        got["prompt" if images else "many"] = many_pieces
    assert got == want
    cache, batch = C.Cache(None, None, None, None, 4, page, kv_heads, dim), C.Batch(None, None, None, len(sequences), tokens, keys // page, longest=longest)
    assert C.attention_workspace({"f32": C.F32, "f16": C.F16, "bf16": C.BF16}[dtype], cache, batch, heads) == size


def test_the_sizes_cover_all_routes():
    ways = {(kernel, dtype == "f32", held, pieces > 1) for dtype, _, _, _, dim, _, _, want in ROUTES.values()
            for kernel, pieces in want.items() for held in [dim > 128]}
    assert {("few", False, False, True), ("few", False, False, False), ("few", True, False, True), ("many", False, False, True),
            ("many", False, False, False), ("many", True, False, True), ("many", False, True, True), ("prompt", False, False, True),
            ("prompt", False, False, False)} <= ways


def test_a_long_bound_on_the_keys_is_served():
    """A table as wide as positions go: fewer and longer pieces, not a refusal, and a workspace that stays small."""
    cache = C.Cache(None, None, None, None, 4, 16, 8, 128)
    for seqs in (1, 64, 500):
        batch = C.Batch(None, None, None, seqs, seqs, (2 ** 31 - 2 ** 16) // 16 - 1, longest=1)
        assert C.attention_workspace(C.BF16, cache, batch, 32) <= 2 ** 28
    batch = C.Batch(None, None, None, 1, 8192, (2 ** 31 - 2 ** 16) // 16 - 1)
    assert C.attention_workspace(C.BF16, cache, batch, 32) <= 2 ** 28


def test_every_kernel_source_is_loaded_when_a_handle_opens():
    host = open(os.path.join(CSRC, "q8_shim.cpp")).read()
    opening = re.search(r"int q8_open\(.*?\n}\n", host, re.S).group(0)
    sources = glob.glob(os.path.join(CSRC, "cache_*.hip"))
    assert len(sources) == 4
    for path in sources:
        names = re.findall(r"hipError_t (prepare_\w+)\(\)", open(path).read())
        assert len(names) == 1 and f"{names[0]}()" in opening, path
