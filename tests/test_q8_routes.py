"""The sizes of test_gpu_q8_routes.py reach every kernel and every way that operands get to it, on the CPU."""
import pytest

from q8_routes import GEMM_ROUTES, GEMMS, GRADIENTS, gemm_route, grad_routes, grad_wanted


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
