"""How Newton-Schulz calls are launched (mms_muon_plan, a host function): the GPU tests take every way that ordinary sizes
do, and a way is not left to a float's last bit."""
from __future__ import annotations

import ctypes
import math
import random

import pytest

from test_gpu_muon_plans import CASES


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


def ways(L, shapes, prec):
    """{(operands' width, product, tile, in parts)}, and the same for a matrix of at most 64 rows that shares them."""
    found = set()
    groups = plan(L, shapes, prec)
    for n, w, a, chunk, b, x in groups:
        kinds = {w}
        if len(groups) == 1 and w == 2 and any(min(s[-2:]) <= 64 for s in shapes):
            kinds.add("narrow")
        for k in kinds:
            found |= {(k, "A", a, chunk > 0), (k, "B", b, False), (k, "X", x, False)}
    return found


def test_gpu_tests_take_every_way(L):
    tested = set()
    for prec in (0, 1):
        for shapes in CASES:
            tested |= ways(L, shapes, prec)
    rng = random.Random(3)

    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    taken = {}
    for _ in range(12000):
        shapes = [(rng.choice([1, 1, 1, 2, 4, 8, 16, 32]), log(1, 6000), log(8, 12000)) for _ in range(rng.choice([1, 1, 1, 2, 3]))]
        if sum(b * min(r, c) ** 2 * max(r, c) for b, r, c in shapes) <= 6e11:
            for prec in (0, 1):
                for w in ways(L, shapes, prec):
                    taken.setdefault(w, (shapes, prec))
    assert len(taken) >= 40
    assert {w: s for w, s in taken.items() if w not in tested} == {}


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
