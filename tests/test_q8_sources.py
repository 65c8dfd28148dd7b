"""What the sources of the 8-bit operators have to keep among themselves, on the CPU."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "amdgpu-arch-gemm_amd", "csrc")


def read(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


def test_opening_a_handle_loads_every_code_object():
    """One a kernel source: else the first call that needs it loads it, under capture too."""
    opening = re.search(r"int q8_open\(.*?\n}\n", read("q8_shim.cpp"), re.S).group()
    called = set(re.findall(r"\b(prepare_\w+)\(\)", opening))
    sources = [os.path.basename(p) for p in glob.glob(os.path.join(CSRC, "q8_*.hip"))]
    assert len(sources) == 4
    for name in sources:
        defined = re.findall(r"^hipError_t (prepare_\w+)\(\) {", read(name), re.M)
        assert len(defined) == 1 and defined[0] in called, name


def test_widths_of_the_row_tests_are_those_of_the_kernels():
    from test_gpu_q8_widths import HELD, HELD_BACKWARD

    text = read("q8_rows.hip")
    for function, held in (("quantize_any", HELD), ("backward_any", HELD_BACKWARD)):
        body = re.search(r"hipError_t %s\(.*?\n}\n" % function, text, re.S).group()
        assert [int(n) for n in re.findall(r"pieces <= (\d+)\) return", body)] == held, function
