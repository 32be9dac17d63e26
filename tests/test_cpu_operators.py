"""Refusals of the parameter operators' entry points (Muon's update, learned row tables), without a device: the C-ABI
checks its arguments before any launch, the Python entry points before any call."""
from __future__ import annotations

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def L():
    from multimodalstudio_amd import _lib, build
    if not _lib.LIB_PATH.exists():
        build.build()
    return _lib.lib()


def _err(L):
    return L.mms_last_error().decode()


def _tables(shapes):
    n = len(shapes)
    I64 = ctypes.c_int64 * n
    return n, I64(*[s[0] for s in shapes]), I64(*[s[1] for s in shapes]), I64(*[s[2] for s in shapes])


def _workspace(L, shapes, prec=0):
    need = ctypes.c_int64(-1)
    rc = L.mms_muon_workspace(*_tables(shapes), prec, ctypes.addressof(need))
    return rc, need.value


def test_muon_workspace(L):
    assert _workspace(L, []) == (0, 0)
    assert _workspace(L, [(0, 4, 4), (1, 0, 9), (2, 7, 0)]) == (0, 0)
    rc, one = _workspace(L, [(1, 60, 100)])
    # 64 x 128 padded: X and the next X (hi and lo, 2 bytes each), A and A's polynomial 64 x 64, the norm's partial sums,
    # the launches' table
    assert rc == 0 and one - 8704 == 2 * 64 * 128 * 4 + 2 * 64 * 64 * 4 + 8192
    assert _workspace(L, [(1, 100, 60)]) == (0, one)
    assert _workspace(L, [(3, 60, 100)]) == (0, 8704 + 3 * (one - 8704))
    # two matrices of one table; long rows: whole parts of 64 x 64 sums of A besides
    assert _workspace(L, [(1, 60, 100), (1, 100, 60)]) == (0, 8704 + 2 * (one - 8704))
    rc, long = _workspace(L, [(1, 60, 8192)])
    parts = long - (8704 + 2 * 64 * 8192 * 4 + 2 * 64 * 64 * 4 + 8192)
    assert rc == 0 and parts > 0 and parts % (64 * 64 * 4) == 0
    for shapes, word in (([(-1, 4, 4)], "sizes"), ([(1, 1 << 21, 4)], "sizes"), ([(1 << 20, 1 << 20, 1 << 20)], "sizes")):
        assert _workspace(L, shapes)[0] != 0 and word in _err(L)
    assert _workspace(L, [(1, 4, 4)], prec=2)[0] != 0 and "prec" in _err(L)
    assert L.mms_muon_workspace(1, None, None, None, 0, ctypes.addressof(ctypes.c_int64(0))) != 0
    assert L.mms_muon_workspace(*_tables([(1, 4, 4)]), 0, None) != 0


def _ns(L, shape=(1, 8, 8), ptr=4096, ld=8, steps=5, eps=1e-7, ws=4096, ws_bytes=1 << 40, bs=64):
    n, b, r, c = _tables([shape])
    VP, I64 = ctypes.c_void_p * 1, ctypes.c_int64 * 1
    return L.mms_newton_schulz(n, b, r, c, VP(ptr), I64(ld), I64(bs), VP(ptr), I64(ld), I64(bs), 0, 0, steps, 3.4, -4.8,
                               2.0, eps, ws, ws_bytes, None)


def test_newton_schulz_refusals(L):
    for kw, word in (({"steps": 0}, "steps"), ({"steps": 65}, "steps"), ({"eps": 0.0}, "eps"), ({"ld": 7}, "leading"),
                     ({"ptr": None}, "null"), ({"ws": None}, "workspace"), ({"ws_bytes": 1000}, "workspace"),
                     ({"ws": 4096 + 128}, "workspace"), ({"shape": (2, 8, 8), "bs": 63}, "overlap")):
        assert _ns(L, **kw) != 0 and word in _err(L), kw
    # nothing to do is a success
    assert _ns(L, shape=(1, 0, 8), ptr=None, ws=None, ws_bytes=0) == 0


def test_muon_step_refusals(L):
    n, b, r, c = _tables([(1, 8, 8)])
    VP, I64, F = ctypes.c_void_p * 1, ctypes.c_int64 * 1, ctypes.c_float * 1

    def step(m=4096, scale=F(1.0), momentum=0.95):
        return L.mms_muon_step(n, b, r, c, VP(4096), I64(8), I64(64), VP(4096), I64(8), I64(64), VP(m), scale, 0, 0, 5,
                               3.4, -4.8, 2.0, 1e-7, momentum, 1, None, 0.0, None, 1.0, -0.1, None, 0, None)
    assert step(m=None) != 0 and "momentum" in _err(L)
    assert step(scale=None) != 0 and "scale" in _err(L)
    assert step(momentum=1.0) != 0 and "momentum" in _err(L)
    assert step() != 0 and "workspace" in _err(L)


def test_embedding_refusals(L):
    def fwd(ids=4096, stride=1, n=4, table=4096, ldt=8, rows=5, dim=8, dtype=0, out=4096, ldo=8):
        return L.mms_embedding_fwd(ids, 1, stride, n, table, ldt, rows, dim, dtype, 1.0, out, ldo, None)

    for kw, word in (({"ids": None}, "indices"), ({"stride": -1}, "stride"), ({"n": -1}, "indices"),
                     ({"n": 1 << 24}, "indices"), ({"rows": 0}, "rows"), ({"dim": 0}, "rows"), ({"dtype": 3}, "dtype"),
                     ({"table": None}, "table"), ({"ldt": 7}, "fit"), ({"ldo": 7}, "fit")):
        assert fwd(**kw) != 0 and word in _err(L), kw
    assert fwd(n=0, ids=None, table=None, out=None) == 0

    def bwd(ids=4096, n=400, dout=4096, ldd=8, rows=5, dim=8, dtype=0, pad=-1, dtable=4096, ldg=8, acc=0, ws=4096,
            ws_bytes=1 << 40):
        return L.mms_embedding_bwd(ids, 1, 1, n, dout, ldd, rows, dim, dtype, 1.0, pad, dtable, ldg, acc, ws, ws_bytes,
                                   None)
    for kw, word in (({"ids": None}, "indices"), ({"rows": 1 << 29}, "rows"), ({"dim": (1 << 20) + 1}, "rows"),
                     ({"dtype": -1}, "dtype"), ({"dout": None}, "null"), ({"ldd": 7}, "fit"), ({"dtable": None}, "null"),
                     ({"ldg": 7}, "fit"), ({"ws": None}, "workspace"), ({"ws_bytes": 8}, "workspace"),
                     ({"ws": 4224}, "workspace")):
        assert bwd(**kw) != 0 and word in _err(L), kw
    # nothing to add into the table
    assert bwd(n=0, ids=None, dout=None, acc=1, ws=None, ws_bytes=0) == 0
    need = ctypes.c_int64(-1)
    assert L.mms_embedding_bwd_workspace(0, 5, 8, 0, ctypes.addressof(need)) == 0
    assert L.mms_embedding_bwd_workspace(1000, 5, 8, 0, None) != 0
    # few positions: none; many rows: two lists of (row, position); few: a sum per row and 256 positions
    assert L.mms_embedding_bwd_workspace(128, 500, 8, 0, ctypes.addressof(need)) == 0 and need.value == 0
    assert L.mms_embedding_bwd_workspace(1000, 500, 8, 0, ctypes.addressof(need)) == 0 and need.value > 2 * 8000
    assert L.mms_embedding_bwd_workspace(1000, 5, 8, 0, ctypes.addressof(need)) == 0 and need.value >= 4 * 5 * 8 * 4


def test_python_entry_points_refuse_host_tensors():
    from multimodalstudio_amd import hip_ops
    g = torch.randn(4, 6)
    with pytest.raises(RuntimeError, match="device"):
        hip_ops.newton_schulz(g)
    with pytest.raises(RuntimeError, match="device"):
        hip_ops.muon_step([g], [g], [g], lr=0.1)
    with pytest.raises(RuntimeError, match="device"):
        hip_ops.embedding(torch.zeros(3, dtype=torch.int64), g)
    with pytest.raises(RuntimeError, match="device"):
        hip_ops.embedding_backward(torch.zeros(3, dtype=torch.int64), torch.zeros(3, 6), 4)
    hip_ops.muon_step([], [], [], lr=0.1)       # no weights: nothing to do
    with pytest.raises(ValueError):
        hip_ops.muon_step([g], [], [], lr=0.1)


def test_matrix_layouts():
    """Which layouts are read in place: rows contiguous and not overlapping; a transposed or expanded one is copied
    where it is read and refused where it is written."""
    from multimodalstudio_amd import hip_ops
    base = torch.arange(6 * 70 * 130, dtype=torch.float32).reshape(6, 70, 130)
    for v, want in ((base, (6, 70, 130, 130, 9100)), (base[0], (1, 70, 130, 130, 0)),
                    (base[0][:, 3:100], (1, 70, 97, 130, 0)), (base[::2], (3, 70, 130, 130, 18200)),
                    (base[0][::2, :5], (1, 35, 5, 260, 0)), (base[0][:1, ::1], (1, 1, 130, 130, 0)),
                    (base[0][:, :1], (1, 70, 1, 130, 0))):
        t, *got = hip_ops._matrices(v, "m", False)
        assert tuple(got) == want and t.data_ptr() == v.data_ptr()
    for v in (base[0].mT, base[0][:, ::2], base[0][:1].expand(5, 130), base[:1].expand(3, 70, 130)):
        with pytest.raises(ValueError):
            hip_ops._matrices(v, "m", False)
        t, batch, rows, cols, ld, bs = hip_ops._matrices(v, "m", True)
        assert torch.equal(t.reshape(v.shape), v) and ld >= cols and (batch == 1 or bs >= rows * cols)
    with pytest.raises(ValueError):
        hip_ops._matrices(base[0, 0], "m", True)


def test_muon_scale():
    from multimodalstudio_amd import hip_ops
    assert hip_ops.muon_scale(256, 64) == 2.0 and hip_ops.muon_scale(64, 256) == 1.0
    assert hip_ops.muon_scale(25, 100, "match_rms_adamw") == 2.0
    with pytest.raises(ValueError):
        hip_ops.muon_scale(4, 4, "other")


def test_flat_indices():
    """A column of a coordinate tensor is read where it lies, other layouts are copied."""
    from multimodalstudio_amd import hip_ops
    c = torch.arange(30, dtype=torch.int32).reshape(10, 3)
    t, st = hip_ops._flat_ids(c[:, :1])
    assert st == 3 and t.data_ptr() == c.data_ptr()
    t, st = hip_ops._flat_ids(c[:, 1])
    assert st == 3 and t.data_ptr() == c.data_ptr() + 4
    t, st = hip_ops._flat_ids(c[:, :2])
    assert st == 1 and t.is_contiguous() and torch.equal(t, c[:, :2])
    t, st = hip_ops._flat_ids(c[:1, :1].expand(7, 1))
    assert st == 1 and t.is_contiguous() and t.numel() == 7
