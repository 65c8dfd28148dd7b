"""The example that trains and serves a layer with the 8-bit operators."""
import importlib.util
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    path = os.path.join(ROOT, "amdgpu-arch-gemm_amd", "examples", "q8_layer.py")
    spec = importlib.util.spec_from_file_location("q8_layer", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("tokens,features,channels", [(512, 256, 192), (300, 129, 77)])
def test_layer_learns_and_decodes(tokens, features, channels):
    losses, worst = _example().train(tokens, features, channels, steps=20, report=lambda line: print(line, flush=True))
    assert np.all(np.isfinite(losses)) and losses[-1] < 0.5 * losses[0]
    # a row's norm does not depend on the other rows, and the product's integer sums are exact
    assert worst == 0.0
