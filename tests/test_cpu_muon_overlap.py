"""Matrices that a Muon or Newton-Schulz call writes and that share memory with others of the call are refused: the blocks
of one would run beside those of the other.  Host checks, before any launch: the addresses here are made up, and a call
that passes the check ends at its workspace of no bytes."""
from __future__ import annotations

import ctypes
import random

import pytest

BASE = 1 << 20


@pytest.fixture(scope="module")
def L():
    from multimodalstudio_amd import _lib, build
    if not _lib.LIB_PATH.exists():
        build.build()
    return _lib.lib()


class Mat:
    """[batch, rows, cols] at element `at` of one made-up buffer."""

    def __init__(self, at, rows, cols, ld=None, batch=1, bs=0):
        self.at, self.rows, self.cols, self.ld, self.batch, self.bs = at, rows, cols, ld or cols, batch, bs

    def elements(self):
        return {self.at + k * self.bs + r * self.ld + c
                for k in range(self.batch) for r in range(self.rows) for c in range(self.cols)}


def far(i, like):
    return Mat((1 << 24) + (i << 18), like.rows, like.cols, batch=like.batch, bs=like.rows * like.cols)


def _arrays(ms, es=4):
    n = len(ms)
    I64, VP = ctypes.c_int64 * n, ctypes.c_void_p * n
    return (VP(*[BASE + es * m.at for m in ms]), I64(*[m.ld for m in ms]), I64(*[m.bs for m in ms]))


def step(L, weights, grads=None, momenta=None, bf16=0):
    n = len(weights)
    grads = grads or [far(i, w) for i, w in enumerate(weights)]
    momenta = momenta or [far(n + i, w) for i, w in enumerate(weights)]
    I64 = ctypes.c_int64 * n
    es = 2 if bf16 else 4
    p, ldp, bsp = _arrays(weights, es)
    g, ldg, bsg = _arrays(grads, es)
    rc = L.mms_muon_step(n, I64(*[w.batch for w in weights]), I64(*[w.rows for w in weights]),
                         I64(*[w.cols for w in weights]), p, ldp, bsp, g, ldg, bsg, _arrays(momenta)[0],
                         (ctypes.c_float * n)(*[1.0] * n), bf16, 0, 5, 3.4445, -4.7750, 2.0315, 1e-7, 0.95, 1, None,
                         0.0, None, 1.0, -0.1, 256, 0, None)
    assert rc != 0
    text = L.mms_last_error().decode()
    assert "overlap" in text or "workspace" in text, text
    return "overlap" in text


def test_weights(L):
    for bf16 in (0, 1):
        def bad(*ws):
            return step(L, list(ws), bf16=bf16)
        assert not bad(Mat(0, 4, 8), Mat(32, 4, 8)) and not bad(Mat(32, 4, 8), Mat(0, 4, 8))
        assert bad(Mat(0, 4, 8), Mat(31, 4, 8)) and bad(Mat(0, 4, 8), Mat(0, 2, 16))
        # w[:4] and w[2:]; a stack and one of its matrices; the same rows
        assert bad(Mat(0, 4, 8), Mat(16, 4, 8)) and bad(Mat(0, 4, 8, batch=3, bs=32), Mat(32, 4, 8))
        # columns of one buffer: side by side, sharing one; every second row
        assert not bad(Mat(0, 6, 5, 16), Mat(5, 6, 11, 16)) and bad(Mat(0, 6, 6, 16), Mat(5, 6, 11, 16))
        assert not bad(Mat(0, 3, 16, 32), Mat(16, 3, 16, 32)) and not bad(Mat(5, 6, 11, 16), Mat(0, 6, 5, 16))
        # a small matrix in the gap between a stack's matrices, or not quite
        assert not bad(Mat(0, 2, 4, batch=3, bs=20), Mat(8, 3, 4)) and bad(Mat(0, 2, 4, batch=3, bs=20), Mat(9, 3, 4))
        # three: only the first and the last meet
        assert bad(Mat(0, 100, 4, 10), Mat(4, 3, 3, 10), Mat(992, 1, 1)) and not bad(Mat(0, 100, 4, 10), Mat(4, 3, 3, 10),
                                                                                  Mat(996, 1, 1))


def test_momenta_and_gradients(L):
    w = [Mat(0, 4, 8), Mat(100, 4, 8)]
    assert step(L, w, momenta=[Mat(500, 4, 8), Mat(516, 4, 8)])
    assert step(L, w, momenta=[Mat(16, 4, 8), Mat(500, 4, 8)]) and step(L, w, momenta=[Mat(500, 4, 8), Mat(16, 4, 8)])
    g = [Mat(500, 4, 8), Mat(600, 4, 8)]
    assert step(L, w, g, [Mat(500, 4, 8), Mat(900, 4, 8)]) and step(L, w, g, [Mat(610, 4, 8), Mat(900, 4, 8)])
    # a weight where another's gradient lies; where its own lies, which is read before; one gradient for both
    assert step(L, w, [Mat(300, 4, 8), Mat(0, 4, 8)])
    assert not step(L, w, w) and not step(L, w, [g[0], g[0]])
    # a repeated gradient
    stack = [Mat(0, 2, 4, batch=3, bs=8)]
    assert not step(L, stack, [Mat(300, 2, 4, batch=3, bs=0)]) and not step(L, stack, [Mat(0, 2, 4, batch=3, bs=0)])


def test_any_layout(L):
    """Random layouts in a small buffer against the sets of their elements."""
    rng = random.Random(7)
    seen = set()
    for _ in range(4000):
        ws = []
        for _ in range(rng.choice([2, 2, 3])):
            rows, cols = rng.randint(1, 4), rng.randint(1, 5)
            ld = rng.choice([cols, cols + rng.randint(0, 9), 10, 20])
            ld = max(ld, cols)
            batch = rng.choice([1, 1, 2, 3])
            bs = (rows - 1) * ld + cols + rng.randint(0, 12) if batch > 1 else 0
            if batch > 1 and bs < rows * ld - (ld - cols):
                bs = rows * ld
            ws.append(Mat(rng.randint(0, 60), rows, cols, ld, batch, bs))
        want = any(a.elements() & b.elements() for i, a in enumerate(ws) for b in ws[:i])
        assert step(L, ws) == want
        seen.add(want)
    assert seen == {True, False}


def test_newton_schulz(L):
    def ns(out, src):
        n = len(out)
        I64 = ctypes.c_int64 * n
        p, ldp, bsp = _arrays(out)
        g, ldg, bsg = _arrays(src)
        rc = L.mms_newton_schulz(n, I64(*[w.batch for w in out]), I64(*[w.rows for w in out]), I64(*[w.cols for w in out]),
                                 g, ldg, bsg, p, ldp, bsp, 0, 0, 5, 3.4445, -4.7750, 2.0315, 1e-7, 256, 0, None)
        assert rc != 0
        return "overlap" in L.mms_last_error().decode()
    a, b = Mat(0, 4, 8), Mat(100, 4, 8)
    assert not ns([a, b], [a, b]) and ns([a, b], [b, a]) and ns([a, a], [b, b]) and not ns([a], [b])
