"""The first calls of a process, captured: nothing that they need is loaded by a call before them."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import os, sys, time
import numpy as np
for d in ("amdgpu-arch-gemm_amd", "tests"):
    sys.path.insert(0, os.path.join(os.getcwd(), d))
from q8_reference import random_q
from test_gpu_noalloc_streams import _Hip, _ok
from shim import q8_shim as Q, sgemm_shim as S

m, n, k = (int(a) for a in sys.argv[1:4])
rng = np.random.default_rng(1)
hip = _Hip()
stream = hip.stream()
x, g = Q.Array.of(rng.normal(0, 1, (m, k)), Q.BF16), Q.Array.of(np.ones(k), Q.BF16)
w, dy = Q.Array.of(rng.normal(0, 1, (n, k)), Q.BF16), Q.Array.of(rng.normal(0, 1, (m, n)), Q.BF16)
qx, sx, rstd, qw, sw = Q.Array(m, k, "int8"), Q.Array(1, m, Q.F32), Q.Array(1, m, Q.F32), Q.Array(n, k, "int8"), Q.Array(1, n, Q.F32)
y, dn, dw, dx, dg = Q.Array(m, n, Q.BF16), Q.Array(m, k, Q.BF16), Q.Array(n, k, Q.BF16), Q.Array(m, k, Q.BF16), Q.Array(1, k, Q.F32)
outs = (qw, sw, qx, sx, y, dw, dn, dx, dg)
o = Q.Ops()
o.set_stream(stream.value)
o.reserve(max(Q.workspace_size(c, Q.BF16, m, n, k) for c in range(4)))

def step():
    o.quantize(Q.BF16, w, qw, sw, n, k)
    o.rmsnorm(Q.BF16, x, None, g, None, qx, sx, rstd, m, k)
    o.gemm(Q.BF16, qx, sx, qw, sw, None, y, m, n, k)
    o.grad_weight(Q.BF16, dy, qx, sx, Q.BF16, dw, m, n, k)
    o.grad_input(Q.BF16, dy, qw, sw, dn, m, n, k)
    o.rmsnorm_backward(Q.BF16, dn, x, g, rstd, None, dx, dg, m, k)

hip.begin(stream, 0)
start = time.perf_counter()
step()
print(f"captured in {1e3 * (time.perf_counter() - start):.2f} ms", flush=True)
exe = hip.end(stream)
step()
o.synchronize()
want = [a.numpy().copy() for a in outs]
assert all(np.any(a != 0) and np.all(np.isfinite(a)) for a in want)
for _ in range(3):
    for a in outs:
        S._check("sgemm_memset", S.load_library().sgemm_memset(a.ptr, 0x11, a.nbytes))
    _ok(hip.lib.hipGraphLaunch(exe, stream))
    o.synchronize()
    assert all(np.array_equal(a.numpy(), b) for a, b in zip(outs, want))
    step()
    o.synchronize()
_ok(hip.lib.hipGraphExecDestroy(exe))
o.set_stream(None)
o.close()
hip.lib.hipStreamDestroy(stream)
print("done", flush=True)
"""


# gradients from the operands as they are, and laid out; the product on the direct and on a tile kernel
@pytest.mark.parametrize("m,n,k", [(100, 72, 66), (2701, 2203, 1301)])
def test_first_calls_captured(m, n, k):
    out = subprocess.run([sys.executable, "-c", PROGRAM, str(m), str(n), str(k)], cwd=ROOT, capture_output=True, text=True,
                         timeout=100)
    print(out.stdout, flush=True)
    assert out.returncode == 0 and out.stdout.split("\n")[-2] == "done", out.stdout + out.stderr
