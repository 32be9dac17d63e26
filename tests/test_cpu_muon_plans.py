"""How Newton-Schulz calls are launched (mms_muon_plan, a host function): a way is not left to a float's last bit."""
from __future__ import annotations

import ctypes
import math

import pytest


@pytest.fixture(scope="module")
def L():
    from multimodalstudio_amd import _lib, build
    if not _lib.LIB_PATH.exists():
        build.build()
    return _lib.lib()


def _tables(shapes):
    n = len(shapes)
    I64 = ctypes.c_int64 * n
    return n, I64(*[math.prod(s[:-2]) for s in shapes]), I64(*[s[-2] for s in shapes]), I64(*[s[-1] for s in shapes])


def plan(L, shapes, prec):
    out, tables = (ctypes.c_int64 * 48)(), ctypes.c_int64(-1)
    assert L.mms_muon_plan(*_tables(shapes), prec, 8, out, ctypes.addressof(tables)) == 0
    return [tuple(out[6 * i:6 * i + 6]) for i in range(tables.value)]


def test_equal_estimates_go_to_whole_sums(L):
    """8 x 1024 x 4096 with single fp16 operands: A whole and in two parts are estimated alike; no room for parts."""
    need = ctypes.c_int64(-1)
    assert L.mms_muon_workspace(*_tables([(8, 1024, 4096)]), 1, ctypes.addressof(need)) == 0
    # the launches' table, then partial sums of the norm, X, the next X and its low half, A, B for each matrix
    assert need.value == 8704 + 8 * (8192 + 3 * 1024 * 4096 * 2 + 2 * 1024 * 1024 * 2)


def test_plan(L):
    assert plan(L, [], 0) == [] and plan(L, [(0, 5), (3, 0, 4)], 0) == []
    (a,) = plan(L, [(40, 70), (5, 2, 3)], 0)
    assert a[:2] == (2, 2)
    # 60 matrices: two tables; prec 1 keeps split operands up to 128 rows
    assert [p[0] for p in plan(L, [(40, 70)] * 60, 0)] == [48, 12]
    assert [p[1] for p in plan(L, [(40, 700), (200, 300)], 1)] == [1, 2]
    # no more than `max` groups are written
    out, tables = (ctypes.c_int64 * 12)(*[-7] * 12), ctypes.c_int64(-1)
    assert L.mms_muon_plan(*_tables([(40, 70)] * 60), 0, 1, out, ctypes.addressof(tables)) == 0
    assert tables.value == 2 and list(out[6:]) == [-7] * 6 and out[0] == 48
    assert L.mms_muon_plan(*_tables([(40, 70)]), 0, 1, None, ctypes.addressof(tables)) != 0
    assert L.mms_muon_plan(*_tables([(40, 70)]), 0, 1, out, None) != 0
    assert L.mms_muon_plan(*_tables([(40, 70)]), 3, 1, out, ctypes.addressof(tables)) != 0
