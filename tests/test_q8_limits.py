"""Index arithmetic of the 8-bit operators at the ends of their range, on the CPU."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run(tmp_path, program):
    source = tmp_path / "program.cpp"
    source.write_text(program)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-I", os.path.join(ROOT, "amdgpu-arch-gemm_amd", "csrc"), str(source), "-o", str(tmp_path / "program")],
                   check=True)
    out = subprocess.run([str(tmp_path / "program")], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr


def test_columns_of_a_thread_end(tmp_path):
    """A thread meets each of its columns once and comes to an end, in rows of every width."""
    run(tmp_path, r"""
#include "q8_plan.hpp"
#include <cstdio>
#include <initializer_list>
using namespace q8;
int main() {
    const uint32_t widths[] = {1, 7, 8, 9, 511, 512, 513, 2048, 2049, 8191, 8192, 8193, 100000, 1u << 27, 2147483647u, 1u << 31,
                               4294959104u, 4294959105u, 4294965248u, 4294965249u, 4294967288u, 4294967294u, 4294967295u};
    for (uint32_t step : {512u, 2048u, 8192u})
        for (uint32_t cols : widths)
            for (uint32_t first : {0u, 8u, step / 2, step - 8}) {
                uint64_t want = first;
                for (uint32_t c = first; c < cols; c = next_column(c, step, cols), want += step)
                    if (c != want) { std::printf("%u of %u: %u\n", step, cols, c); return 1; }
                if (want < cols) { std::printf("%u of %u ends before %llu\n", step, cols, (unsigned long long)want); return 1; }
            }
    std::puts("ok");
}
""")
