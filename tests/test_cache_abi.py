"""The C-ABI of the rotary, cache and attention operators without a GPU."""
import ctypes
import os
import re

import numpy as np
import pytest

from shim import q8_cache as C
from shim import q8_shim as Q
from shim import sgemm_shim as S

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "q8_cache.h")


def _text():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


def test_every_declared_symbol_is_exported_and_bound():
    names = set(re.findall(r"\bint (q8_[a-z0-9_]+)\s*\(", _text()))
    lib = C.load_library()
    assert names == set(C.SIGNATURES) and not names & set(Q.SIGNATURES)
    for name in names:
        assert hasattr(lib, name), name


def test_structures_match_the_header():
    """The fields' order and types, and that the compiler lays them out the same (natural alignment, no tail)."""
    sizes = {"uint32_t": 4, "uint8_t": 1}
    for struct, name in ((C._Rotation, "q8_rotation"), (C._Cache, "q8_cache"), (C._Batch, "q8_batch")):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), _text(), re.S).group(1)
        fields = re.findall(r"(?:const )?(\w+)(\*?) (\w+)(?:\[(\d+)\])?;", body)
        assert [f[2] for f in fields] == [f[0] for f in struct._fields_]
        offset = 0
        for kind, pointer, field, count in fields:
            size = 8 if pointer else sizes[kind]
            offset = -(-offset // size) * size
            assert getattr(struct, field).offset == offset and getattr(struct, field).size == size * int(count or 1)
            offset += size * int(count or 1)
    values = dict(re.findall(r"#define (Q8_MAX_[A-Z]+) (\d+)u", _text()))
    assert {k: int(v) for k, v in values.items()} == {"Q8_MAX_DIM": C.MAX_DIM, "Q8_MAX_AXES": C.MAX_AXES}


def test_calls_without_a_handle_are_refused():
    lib = C.load_library()
    for name, (_, args) in C.SIGNATURES.items():
        if name == "q8_attention_workspace":
            continue
        assert getattr(lib, name)(None, *[a() for a in args[1:]]) == -1, name
        assert b"handle" in S.load_library().sgemm_last_error()


def workspace(code, what, cache=(4, 16, 2, 64), batch=(2, 2, 4), heads=4, dtype=C.BF16):
    with pytest.raises(S.SgemmError) as e:
        C.attention_workspace(dtype, C.Cache(None, None, None, None, *cache), C.Batch(None, None, None, *batch), heads)
    assert e.value.code == code and what in e.value.message, e.value.message


def test_sizes_that_are_refused():
    """The checks of sizes that all calls share, through the one that needs no handle."""
    workspace(-1, "type", dtype=5)
    workspace(-4, "257 values", cache=(4, 16, 2, 257))
    workspace(-4, "0 values", cache=(4, 16, 2, 0))
    workspace(-4, "no heads", cache=(4, 16, 0, 64))
    workspace(-4, "no tokens", cache=(4, 0, 2, 64))
    workspace(-4, "2^31 bytes", cache=(4, 1 << 24, 2, 64))
    workspace(-4, "2^31 bytes", cache=(4, 2 ** 32 - 1, 65535, 256))
    workspace(-4, "2^48 bytes", cache=(2 ** 31 - 1, 1 << 16, 16, 64), batch=(2, 2, 4))
    workspace(-4, "31 bits", cache=(2 ** 31, 1, 1, 16))
    workspace(-4, "31 bits", batch=(2, 2 ** 31, 4))
    workspace(-4, "31 bits", batch=(2 ** 31, 2, 4))
    workspace(-4, "positions", batch=(2, 2, 2 ** 27 - 4096))
    workspace(-4, "no multiple", heads=3)
    workspace(-4, "no multiple", heads=0)
    workspace(-4, "2^24", heads=2 ** 18)
    workspace(-4, "2^24", cache=(4, 1, 2 ** 18, 64), heads=2 ** 18)
    lib = C.load_library()
    n = ctypes.c_size_t(7)
    cache, batch = C.Cache(None, None, None, None, 4, 16, 2, 64), C.Batch(None, None, None, 2, 2, 4)
    assert lib.q8_attention_workspace(C.BF16, cache.at, batch.at, 4, None) == -1
    assert lib.q8_attention_workspace(C.BF16, None, batch.at, 4, ctypes.byref(n)) == -1 and n.value == 0
    assert lib.q8_attention_workspace(C.BF16, cache.at, None, 4, ctypes.byref(n)) == -1


def test_binding_refuses_what_32_bits_do_not_hold():
    for make in (lambda: C.Cache(None, None, None, None, 2 ** 32, 16, 2, 64), lambda: C.Batch(None, None, None, 2, -1, 4),
                 lambda: C.Rotation(2 ** 32, [0]), lambda: C.Rotation(64, [0] * 129), lambda: C.Rotation(64, [-1])):
        with pytest.raises(ValueError):
            make()


def test_division_by_a_page():
    """n / d as the kernels take it (a product's upper bits) for all kinds of d and the n where it could be off."""
    for d in [1, 2, 3, 5, 7, 16, 24, 100, 4095, 4097, 2 ** 16 - 1, 2 ** 16 + 1, 2 ** 30 - 1, 2 ** 30, 2 ** 30 + 1, 2 ** 31 - 1]:
        s = 0
        while s < 31 and 1 << s < d:
            s += 1
        mul = ((1 << (31 + s)) + d - 1) // d
        assert mul < 2 ** 32
        for q in {0, 1, 2, (2 ** 31 - 1) // d, (2 ** 31 - 1) // d // 2}:
            for n in (q * d - 1, q * d, q * d + d - 1, 2 ** 31 - 1):
                if 0 <= n < 2 ** 31:
                    assert n * mul >> (31 + s) == n // d
