"""The sizes of test_gpu_q8_routes.py reach every kernel and every way that operands get to it, on the CPU."""
import pytest

from q8_routes import (DIRECT_TILES, DIRECTS, GEMM_ROUTES, GEMMS, GRADIENTS, direct_tile, gemm_route, grad_routes,
                       grad_wanted)


def test_products_reach_every_route():
    reached = {gemm_route(m, n, k, k + pad, shift) for m, n, k, pad, shift in GEMMS}
    assert GEMM_ROUTES <= reached, GEMM_ROUTES - reached


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_gradients_reach_every_route(dtype):
    routes = [grad_routes(m, n, k, dtype, n + pad, shift) for m, n, k, pad, shift in GRADIENTS]
    for turned in (0, 1):
        reached = {r[turned][:2] for r in routes}
        assert grad_wanted(dtype, turned) <= reached, (turned, grad_wanted(dtype, turned) - reached)
    # the input's gradient reads dy as it is, or laid out
    if dtype != "f32":
        copies = {r[0][2] for r in routes if r[0][0] != "direct"}
        assert copies == {"copies-0", "copies-1"}


def test_few_tokens_reach_every_tile():
    assert {direct_tile(*size) for size in DIRECTS} == set(DIRECT_TILES)


@pytest.mark.parametrize("m,n,k,tile", [
    # one token's weights are streamed by as many work-groups as there are, unless K is short
    (1, 12288, 8192, "1x1"), (1, 65536, 4096, "1x1"), (8, 16384, 4096, "1x1"), (1, 12288, 1024, "1x4"), (8, 16384, 2048, "1x4"),
    (16, 16384, 4096, "1x4"), (12, 32768, 8192, "1x4"), (16, 10240, 4096, "1x1"), (1, 4096, 12288, "1x1"), (1, 4096, 28672, "1x1"),
    # wide tiles from the first size on that gives narrow ones more than two work-groups a CU
    (32, 8192, 4096, "2x1"), (32, 8704, 4096, "2x4"), (17, 10240, 8192, "2x4"), (64, 8192, 4096, "2x2"), (64, 8704, 4096, "4x4"),
    (33, 11264, 1024, "4x4"), (64, 4096, 4096, "2x2")])
def test_few_tokens_take_the_faster_tile(m, n, k, tile):
    """Each of these was measured against the other tile of its tokens."""
    assert direct_tile(m, n, k) == tile
