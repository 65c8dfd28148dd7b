"""The row operators at the widths at which each of their kernels takes over (test_q8_sources.py checks that these are
all of them), against float64 as in test_gpu_q8_rows.py."""
import pytest

import test_gpu_q8_rows as rows
from q8_reference import TYPES
from shim import q8_shim as Q

pytestmark = pytest.mark.gpu

# pieces of eight values that the kernels of a row hold at most: of the norm and the quantisation, and of the norm's gradient
HELD = [64, 128, 192, 256, 384, 512, 768, 1024, 1536, 2048, 4096]
HELD_BACKWARD = [64, 128, 256, 512, 1024, 2048]


def widths(held):
    """A kernel's first width, an odd one in its middle, and its last one."""
    out, least = [], 8
    for pieces in held:
        out += [least, (least + 8 * pieces) // 2 | 1, 8 * pieces]
        least = 8 * pieces + 1
    return out + [least]


@pytest.fixture(scope="module")
def ops():
    with Q.Ops() as o:
        yield o


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cols", widths(HELD))
def test_norm_and_quantize(ops, cols, dtype):
    print(f"norm of {cols} {dtype}", flush=True)
    rows.test_norm(ops, dtype, cols, 0, 0, True, True)
    rows.test_norm(ops, dtype, cols, 1, 1, False, False)
    rows.test_quantize_and_restore(ops, dtype, cols, 0, 0)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cols", widths(HELD_BACKWARD))
def test_norm_backward(ops, cols, dtype):
    print(f"norm's gradient of {cols} {dtype}", flush=True)
    rows.test_norm_backward(ops, dtype, 7, cols, 0, 0, True)
    rows.test_norm_backward(ops, dtype, 2, cols, 3, 1, False)
