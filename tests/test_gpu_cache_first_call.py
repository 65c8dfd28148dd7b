"""The first calls of a process, captured: nothing that they need is loaded by a call before them."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import os, sys
import numpy as np
for d in ("amdgpu-arch-gemm_amd", "tests"):
    sys.path.insert(0, os.path.join(os.getcwd(), d))
from cache_reference import Case
from test_gpu_cache_together import COLS, DIM, HEADS, KV, PAGE, Block
from test_gpu_noalloc_streams import _Hip, _ok
from shim import q8_cache as C

rng = np.random.default_rng(1)
case = Case(rng, eval(sys.argv[1]), HEADS, KV, DIM, PAGE)
kind = getattr(C, sys.argv[2])
hip = _Hip()
stream = hip.stream()
cache, batch = case.upload()
block = Block(C.Rotation(DIM, [0] * 32), kind, cache, batch, case.tokens)
x, positions = rng.normal(0, 1, (case.tokens, COLS)), np.arange(case.tokens)[None]
block.fill(x, positions)
o = C.Ops()
o.set_stream(stream.value)
o.reserve(C.attention_workspace(kind, cache, batch, HEADS))
hip.begin(stream, 0)
block.run(o)
exe = hip.end(stream)
print("captured", flush=True)
block.run(o)
o.synchronize()
want = block.out.numpy().copy()
assert np.all(np.isfinite(want)) and np.any(want != 0)
for _ in range(3):
    block.fill(x, positions)
    _ok(hip.lib.hipGraphLaunch(exe, stream))
    o.synchronize()
    assert np.array_equal(block.out.numpy(), want)
    block.fill(x, positions)
    block.run(o)
    o.synchronize()
    assert np.array_equal(block.out.numpy(), want)
_ok(hip.lib.hipGraphExecDestroy(exe))
o.set_stream(None)
o.close()
hip.lib.hipStreamDestroy(stream)
print("done", flush=True)
"""


# few rows; few and many; from images
@pytest.mark.parametrize("sequences,kind", [([(1, 900)], "F16"), ([(100, 300), (1, 500)], "F32"), ([(600, 700)], "BF16")])
def test_first_calls_captured(sequences, kind):
    out = subprocess.run([sys.executable, "-c", PROGRAM, repr(sequences), kind], cwd=ROOT, capture_output=True, text=True, timeout=100)
    print(out.stdout, flush=True)
    assert out.returncode == 0 and out.stdout.split("\n")[-2] == "done", out.stdout + out.stderr
