"""What the 8-bit operators refuse, and that a refused call leaves its outputs alone."""
import numpy as np
import pytest

from shim import q8_shim as Q
from shim import sgemm_shim as S

pytestmark = pytest.mark.gpu

INVALID, SHAPE = -1, -4
M, N, K = 8, 16, 32


@pytest.fixture(scope="module")
def env():
    with Q.Ops() as ops:
        a = {"x": Q.Array(M, K, Q.F32), "n": Q.Array(M, K, Q.F32), "g": Q.Array(1, K, Q.F32), "h": Q.Array(M, K, Q.F32),
             "q": Q.Array(M, K, "int8"), "s": Q.Array(1, M, Q.F32), "r": Q.Array(1, M, Q.F32), "w": Q.Array(N, K, "int8"),
             "sw": Q.Array(1, N, Q.F32), "y": Q.Array(M, N, Q.F32), "dw": Q.Array(N, K, Q.F32), "dg": Q.Array(1, K, Q.F32)}
        for b in a.values():
            S._check("sgemm_memset", S.load_library().sgemm_memset(b.ptr, 0x3c, b.nbytes))
        yield ops, a


class At:
    def __init__(self, ptr):
        self.ptr = ptr


def refused(env, code, what, call):
    ops, a = env
    with pytest.raises(S.SgemmError) as e:
        call(ops, a)
    assert e.value.code == code and what in e.value.message, e.value.message
    ops.synchronize()
    for b in a.values():
        raw = S.DeviceView(b, 0, b.nbytes // 4 * 4).download().view(np.uint32)
        assert np.all(raw == 0x3c3c3c3c)


CALLS = {
    "quantize: type": (INVALID, "type", lambda o, a: o.quantize(7, a["x"], a["q"], a["s"], M, K)),
    "quantize: null x": (INVALID, "x is null", lambda o, a: o.quantize(Q.F32, None, a["q"], a["s"], M, K)),
    "quantize: null scale": (INVALID, "scale is null", lambda o, a: o.quantize(Q.F32, a["x"], a["q"], None, M, K)),
    "quantize: ld": (SHAPE, "leading dimension", lambda o, a: o.quantize(Q.F32, a["x"], a["q"], a["s"], M, K, ldx=K - 1)),
    "quantize: alignment": (INVALID, "aligned", lambda o, a: o.quantize(Q.F32, At(a["x"].ptr + 2), a["q"], a["s"], 1, 4)),
    "quantize: overlap": (INVALID, "overlaps", lambda o, a: o.quantize(Q.F32, a["x"], At(a["x"].ptr + 64), a["s"], M, K)),
    "quantize: empty rows": (SHAPE, "no values", lambda o, a: o.quantize(Q.F32, a["x"], a["q"], a["s"], M, 0)),
    "dequantize: null q": (INVALID, "q is null", lambda o, a: o.dequantize(Q.F32, None, a["s"], a["x"], M, K)),
    "dequantize: overlap": (INVALID, "overlaps", lambda o, a: o.dequantize(Q.F32, a["q"], a["s"], a["q"], 1, 8)),
    "rmsnorm: null gain": (INVALID, "gain is null",
                           lambda o, a: o.rmsnorm(Q.F32, a["x"], None, None, None, a["q"], a["s"], None, M, K)),
    "rmsnorm: eps": (INVALID, "eps", lambda o, a: o.rmsnorm(Q.F32, a["x"], None, a["g"], None, a["q"], a["s"], None, M, K, -1.0)),
    "rmsnorm: eps no number": (INVALID, "eps", lambda o, a: o.rmsnorm(Q.F32, a["x"], None, a["g"], None, a["q"], a["s"], None,
                                                                      M, K, float("nan"))),
    "rmsnorm: hidden part of x": (INVALID, "hidden overlaps x", lambda o, a: o.rmsnorm(
        Q.F32, a["x"], None, a["g"], At(a["x"].ptr + 4 * K), a["q"], a["s"], None, M - 1, K)),
    "rmsnorm: scale is rstd": (INVALID, "overlaps", lambda o, a: o.rmsnorm(Q.F32, a["x"], None, a["g"], None, a["q"], a["s"],
                                                                          a["s"], M, K)),
    "backward: null rstd": (INVALID, "rstd is null", lambda o, a: o.rmsnorm_backward(
        Q.F32, a["n"], a["h"], a["g"], None, None, a["x"], None, M, K)),
    "backward: dx is hidden": (INVALID, "dx overlaps hidden", lambda o, a: o.rmsnorm_backward(
        Q.F32, a["n"], a["h"], a["g"], a["r"], None, a["h"], None, M, K)),
    "backward: dgain is gain": (INVALID, "dgain overlaps gain", lambda o, a: o.rmsnorm_backward(
        Q.F32, a["n"], a["h"], a["g"], a["r"], None, a["x"], a["g"], M, K)),
    "gemm: null weights": (INVALID, "qw is null", lambda o, a: o.gemm(Q.F32, a["q"], a["s"], None, a["sw"], None, a["y"], M, N, K)),
    "gemm: ld of y": (SHAPE, "y: leading", lambda o, a: o.gemm(Q.F32, a["q"], a["s"], a["w"], a["sw"], None, a["y"], M, N, K,
                                                              ldy=N - 1)),
    "gemm: too long a sum": (SHAPE, "131071", lambda o, a: o.gemm(Q.F32, a["q"], a["s"], a["w"], a["sw"], None, a["y"], 1, 1,
                                                                 131072)),
    "gemm: y is a scale": (INVALID, "y overlaps sw", lambda o, a: o.gemm(Q.F32, a["q"], a["s"], a["w"], a["sw"], None, a["sw"],
                                                                        1, N, K)),
    "grad_input: null dy": (INVALID, "dy is null", lambda o, a: o.grad_input(Q.F32, None, a["w"], a["sw"], a["x"], M, N, K)),
    "grad_input: type": (INVALID, "type", lambda o, a: o.grad_input(-1, a["y"], a["w"], a["sw"], a["x"], M, N, K)),
    "grad_input: overlap": (INVALID, "dx overlaps dy", lambda o, a: o.grad_input(Q.F32, a["x"], a["w"], a["sw"], a["x"], M, N, K)),
    "grad_weight: out type": (INVALID, "type", lambda o, a: o.grad_weight(Q.F32, a["y"], a["q"], a["s"], Q.BF16, a["dw"], M, N, K)),
    "grad_weight: too long a sum": (SHAPE, "too long", lambda o, a: o.grad_weight(
        Q.F32, a["y"], a["q"], a["s"], Q.F32, a["dw"], 3_000_000, N, K)),
    "grad_weight: ld": (SHAPE, "qx: leading", lambda o, a: o.grad_weight(Q.F32, a["y"], a["q"], a["s"], Q.F32, a["dw"], M, N, K,
                                                                        ldx=K - 1)),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_refused(env, name):
    refused(env, *CALLS[name])


def test_windows_of_one_buffer_are_apart(env):
    """Columns of one buffer next to one another are no overlap."""
    ops, _ = env
    both = Q.Array(M, 2 * K, Q.F32)
    host = np.zeros((M, 2 * K), np.float32)
    host[:, :K] = np.arange(M * K).reshape(M, K) - 100
    S._check("sgemm_memcpy_h2d", S.load_library().sgemm_memcpy_h2d(both.ptr, host.ctypes.data, host.nbytes))
    q, s = Q.Array(M, K, "int8"), Q.Array(1, M, Q.F32)
    g = Q.Array.of(np.ones(K))
    ops.rmsnorm(Q.F32, both, None, g, At(both.ptr + 4 * K), q, s, None, M, K, ldx=2 * K, ldh=2 * K)
    ops.synchronize()
    got = both.numpy()
    assert np.array_equal(got[:, K:], host[:, :K]) and np.array_equal(got[:, :K], host[:, :K])
    with pytest.raises(S.SgemmError):
        ops.rmsnorm(Q.F32, both, None, g, At(both.ptr + 4 * K - 4), q, s, None, M, K, ldx=2 * K, ldh=2 * K)
