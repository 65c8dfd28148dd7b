"""Index arithmetic of the 8-bit operators at the ends of their range, on the CPU."""
import inspect
import os
import re
import subprocess

import pytest

from shim import q8_shim as Q
from shim import sgemm_shim as S

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


@pytest.mark.parametrize("call", [Q.CALL_GRAD_INPUT, Q.CALL_GRAD_WEIGHT])
@pytest.mark.parametrize("dtype,most", [(Q.F32, Q.MAX_SUM_F32), (Q.F16, Q.MAX_SUM), (Q.BF16, Q.MAX_SUM)])
def test_longest_sums_of_the_gradients(call, dtype, most):
    """The longest sum is taken, the next one refused with a message that says which is the longest."""
    def size(summed):
        return Q.workspace_size(call, dtype, *((200, summed, 200) if call == Q.CALL_GRAD_INPUT else (summed, 200, 200)))

    assert size(most) > 0
    with pytest.raises(S.SgemmError) as e:
        size(most + 1)
    assert e.value.code == -4 and f"at most {most}" in e.value.message


def test_longest_sums_match_the_header():
    text = open(os.path.join(ROOT, "include", "q8_shim.h")).read()
    values = {k: int(v) for k, v in re.findall(r"#define (Q8_MAX_\w+) (\d+)u", text)}
    assert values == {"Q8_MAX_K": Q.MAX_K, "Q8_MAX_SUM": Q.MAX_SUM, "Q8_MAX_SUM_F32": Q.MAX_SUM_F32}


class _Memory:
    ptr = 4096


@pytest.mark.parametrize("size", [-1, 2 ** 32, 2 ** 32 + 5, -2 ** 40])
@pytest.mark.parametrize("name", ["quantize", "dequantize", "rmsnorm", "rmsnorm_backward", "gemm", "grad_input", "grad_weight"])
def test_sizes_past_32_bits_reach_no_call(name, size):
    """They would be cut: 2^32 + 5 rows to five, -1 to 2^32 - 1."""
    ops = Q.Ops.__new__(Q.Ops)       # without a handle every call that reaches the library is refused there
    ops.handle, ops._lib = None, Q.load_library()
    parameters = list(inspect.signature(getattr(Q.Ops, name)).parameters)[1:]
    sizes = [p for p in parameters if p in ("rows", "cols", "m", "n", "k")]
    given = {**{p: Q.F32 for p in parameters if p.endswith("dtype")}, **{p: 8 for p in sizes}}
    given.update({p: _Memory() for p in parameters if p not in given and not p.startswith("ld") and p not in ("eps", "accumulate")})
    with pytest.raises(S.SgemmError):
        getattr(ops, name)(**given)
    for p in sizes + [p for p in parameters if p.startswith("ld")]:
        with pytest.raises(ValueError, match="q8_" + name):
            getattr(ops, name)(**{**given, p: size})


def test_workspace_of_sizes_past_32_bits():
    for bad in ((-1, 8, 8), (8, 2 ** 32, 8), (8, 8, 2 ** 33 + 1)):
        with pytest.raises(ValueError):
            Q.workspace_size(Q.CALL_GEMM, Q.F32, *bad)
