"""The C-ABI of the 8-bit operators without a GPU."""
import ctypes
import os
import re

import numpy as np
import pytest

from shim import q8_shim as Q
from shim import sgemm_shim as S

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "q8_shim.h")


def _text():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


def test_every_declared_symbol_is_exported_and_bound():
    names = set(re.findall(r"\b(q8_[a-z0-9_]+)\s*\(", _text()))
    lib = Q.load_library()
    assert names == set(Q.SIGNATURES)
    for name in names:
        assert hasattr(lib, name), name


def test_constants_match_the_header():
    values = dict(re.findall(r"\b(Q8_[A-Z0-9_]+) = (\d+)", _text()))
    want = {"Q8_F32": Q.F32, "Q8_F16": Q.F16, "Q8_BF16": Q.BF16, "Q8_CALL_RMSNORM_BACKWARD": Q.CALL_RMSNORM_BACKWARD,
            "Q8_CALL_GEMM": Q.CALL_GEMM, "Q8_CALL_GRAD_INPUT": Q.CALL_GRAD_INPUT, "Q8_CALL_GRAD_WEIGHT": Q.CALL_GRAD_WEIGHT}
    assert {k: int(v) for k, v in values.items()} == want
    assert int(re.search(r"#define Q8_MAX_K (\d+)u", _text()).group(1)) == Q.MAX_K


def test_no_device_is_an_error_code_not_a_crash():
    if os.path.exists("/dev/kfd"):
        pytest.skip("a GPU is visible here")
    h = ctypes.c_void_p()
    assert Q.load_library().q8_open(ctypes.byref(h)) == -5
    assert b"device" in S.load_library().sgemm_last_error()
    with pytest.raises(S.SgemmError):
        Q.Ops()


def test_calls_without_a_handle_are_refused():
    lib = Q.load_library()
    assert lib.q8_open(None) == -1
    lib.q8_close(None)
    for name, (_, args) in Q.SIGNATURES.items():
        if name in ("q8_open", "q8_close", "q8_workspace_size"):
            continue
        assert getattr(lib, name)(None, *[a() for a in args[1:]]) == -1, name
        assert b"handle" in S.load_library().sgemm_last_error()


def test_workspace_sizes():
    with pytest.raises(S.SgemmError) as e:
        Q.workspace_size(9, Q.F32, 1, 1, 1)
    assert e.value.code == -1
    with pytest.raises(S.SgemmError):
        Q.workspace_size(Q.CALL_GEMM, 3, 1, 1, 1)
    # few tokens need none; more tokens need their copies at the most, or K ranges
    assert Q.workspace_size(Q.CALL_GEMM, Q.BF16, 64, 4096, 4096) == 0
    assert Q.workspace_size(Q.CALL_GEMM, Q.BF16, 2000, 1000, 1000) >= (2000 + 1000) * 1008
    # the gradients' operands in 16 bits, three terms for 32
    for call in (Q.CALL_GRAD_INPUT, Q.CALL_GRAD_WEIGHT):
        one, three = (Q.workspace_size(call, t, 8192, 4096, 4096) for t in (Q.BF16, Q.F32))
        assert 0 < one < three
    with pytest.raises(S.SgemmError) as e:      # a row of the laid-out operand is too long
        Q.workspace_size(Q.CALL_GRAD_WEIGHT, Q.BF16, 3_000_000, 8, 8)
    assert e.value.code == -4
    assert Q.workspace_size(Q.CALL_RMSNORM_BACKWARD, Q.F32, 1, 0, 1000) >= 4000


def test_bfloat16_conversions():
    x = np.array([0.0, -0.0, 1.0, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, 1 + 2.0 ** -9, 3.4e38, np.inf, -np.inf, 1e-40], np.float32)
    want = [0.0, -0.0, 1.0, 1.0, 1 + 2.0 ** -6, 1.0, np.inf, np.inf, -np.inf, np.float32(1e-40)]
    got = Q.from_bf16(Q.to_bf16(x))
    assert np.array_equal(got[:-1], np.array(want[:-1], np.float32)) and abs(got[-1] - want[-1]) <= 2.0 ** -134   # half a step there
    assert np.signbit(got[1]) and np.isnan(Q.from_bf16(Q.to_bf16(np.array([np.nan], np.float32))))[0]


def test_row_bytes():
    assert [Q.row_bytes(c) for c in (1, 16, 17, 4096)] == [16, 16, 32, 4096]
