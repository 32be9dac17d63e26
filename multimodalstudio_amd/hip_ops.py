"""torch.autograd bridges onto the C-ABI HIP kernels (libmms_hip.so).

Tensors are PyTorch-owned device memory; kernels receive raw pointers and the current HIP stream.
Every function here requires CUDA(HIP) tensors and raises otherwise: there is no CPU fallback.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import os
from typing import Optional

import torch

from . import _lib

ACT_IDS = {None: 0, "None": 0, "Identity": 0, "ReLU": 1, "Softplus": 2, "Sigmoid": 3}
NT, NN, TN = 0, 1, 2


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _check_dev(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError("MMS HIP ops require device (cuda/hip) tensors; no CPU fallback exists")


# ----------------------------------------------------------------------------------------------
# hash grid
# ----------------------------------------------------------------------------------------------
def _f32_array(vals):
    arr = (ctypes.c_float * len(vals))(*[float(v) for v in vals])
    return arr


INTERP = {None: 0, "Linear": 0, "Smoothstep": 1}   # HashEncodingConfig.interpolation (encodings.py:64-67)


def hashgrid_forward(pos: torch.Tensor, table: torch.Tensor, scales, log2T: int, radius: float,
                     active_levels: int, out: Optional[torch.Tensor] = None, interp: int = 0) -> torch.Tensor:
    """Raw forward launch; pos [M, >=3] (row stride pos.stride(0)), out [M, >=2L]; interp 0 Linear, 1 Smoothstep."""
    _check_dev(pos, table)
    L = len(scales)
    M = pos.shape[0]
    if out is None:
        out = torch.empty(M, 2 * L, device=pos.device, dtype=torch.float32)
    assert pos.stride(1) == 1 and out.stride(1) == 1 and table.is_contiguous()
    sc = _f32_array(scales)
    _lib.call("mms_hashgrid_fwd", pos.data_ptr(), M, pos.stride(0), table.data_ptr(), L, log2T, table.shape[1],
              int(interp), ctypes.cast(sc, ctypes.c_void_p), float(radius), int(active_levels), out.data_ptr(), out.stride(0),
              _stream())
    return out


def hashgrid_backward(pos, table, scales, log2T, radius, active_levels, dout, dtable=None, dpos=None, interp: int = 0):
    _check_dev(pos, table, dout)
    L = len(scales)
    sc = _f32_array(scales)
    assert dout.stride(1) == 1
    _lib.call("mms_hashgrid_bwd", pos.data_ptr(), pos.shape[0], pos.stride(0), table.data_ptr(), L, log2T,
              table.shape[1], int(interp), ctypes.cast(sc, ctypes.c_void_p), float(radius), int(active_levels),
              dout.data_ptr(), dout.stride(0), _ptr(dtable), _ptr(dpos), 0 if dpos is None else dpos.stride(0),
              _stream())


class HashGridFunction(torch.autograd.Function):
    """FeatureGrid(HashEncoding) forward/backward on the HIP kernels."""

    @staticmethod
    def forward(ctx, pos, table, scales, log2T, radius, active_levels, interp: int = 0):
        pos_c = pos.contiguous()
        out = hashgrid_forward(pos_c, table, scales, log2T, radius, active_levels, interp=interp)
        ctx.save_for_backward(pos_c, table)
        ctx.cfg = (scales, log2T, radius, active_levels, interp)
        return out

    @staticmethod
    def backward(ctx, dout):
        pos, table = ctx.saved_tensors
        scales, log2T, radius, active_levels, interp = ctx.cfg
        dtable = torch.zeros_like(table) if ctx.needs_input_grad[1] else None
        dpos = torch.zeros_like(pos) if ctx.needs_input_grad[0] else None
        hashgrid_backward(pos, table, scales, log2T, radius, active_levels, dout.contiguous(), dtable, dpos,
                          interp=interp)
        return dpos, dtable, None, None, None, None, None


# ----------------------------------------------------------------------------------------------
# GEMM
# ----------------------------------------------------------------------------------------------
_MODE_TRANS = {NT: (0, 0), NN: (0, 1), TN: (1, 1)}
PREC_IDS = {"fp32": 0, "bf16": 1, "bf16x3": 2}


def gemm(mode: int, M: int, N: int, K: int, A: torch.Tensor, lda: int, B: torch.Tensor, ldb: int,
         C: torch.Tensor, ldc: int, bias=None, Z=None, ldz=0, aux=None, ldaux=0, act=0, dact=0,
         beta=1.0, thr=20.0, accumulate=False, splits=1, prec: int = 0, ones_col: int = -1, colsum=None):
    """NT: C = A B^T (A [M,K], B [N,K]); NN: C = A B (B [K,N]); TN: C = A^T B (A [K,M], B [K,N]).

    ``colsum`` (TN only): colsum[m] += sum_k A[k, m] fused into the same pass (bias gradients)."""
    ta, tb = _MODE_TRANS[mode]
    _lib.call("mms_gemm", int(prec), ta, tb, int(M), int(N), int(K), A.data_ptr(), int(lda), B.data_ptr(), int(ldb),
              C.data_ptr(), int(ldc), _ptr(bias), _ptr(Z), int(ldz), _ptr(aux), int(ldaux), int(act), int(dact),
              float(beta), float(thr), int(bool(accumulate)), int(splits), int(ones_col), _ptr(colsum), _stream())


def weight_norm_fwd(g, v, W, norms):
    N, K = v.shape
    _lib.call("mms_weight_norm_fwd", g.data_ptr(), v.data_ptr(), N, K, W.data_ptr(), W.stride(0), norms.data_ptr(),
              _stream())


def weight_norm_bwd(g, v, norms, dW, dg, dv):
    N, K = v.shape
    _lib.call("mms_weight_norm_bwd", g.data_ptr(), v.data_ptr(), norms.data_ptr(), N, K, dW.data_ptr(), dW.stride(0),
              dg.data_ptr(), dv.data_ptr(), _stream())


def colsum_(A, out):
    M, N = A.shape
    _lib.call("mms_colsum", A.data_ptr(), M, N, A.stride(0), out.data_ptr(), _stream())


def act_bwd(dY, Z, act, beta, thr, dZ):
    M, N = dY.shape
    _lib.call("mms_act_bwd", dY.data_ptr(), dY.stride(0), Z.data_ptr(), Z.stride(0), M, N, int(act), float(beta),
              float(thr), dZ.data_ptr(), dZ.stride(0), _stream())


# split-K target: blocks per weight-gradient GEMM (measured, scripts/tn_sweep.py): one 128x128-tile block per CU for
# bf16 operands (more splits only add float atomics), two for split-bf16x3 (3 MFMAs per product), four for fp32
_SPLIT_BLOCKS = {0: 1024, 1: 256, 2: 512}


def _splits_for(M_rows: int, tiles: int, prec: int = 0) -> int:
    """K slices of a split-K weight gradient: a multiple of 8 (mms_gemm spreads each tile's slices over the 8 XCDs and
    pads the count to a multiple of 8: a padded count loads some XCDs with one slice more) within the block target."""
    target = max(1, _SPLIT_BLOCKS.get(int(prec), 1024) // max(1, tiles))
    if target >= 8:
        target = target // 8 * 8
    return int(max(1, min(target, M_rows // 512)))


# grouped weight-gradient launches (mms_gemm_tn_grouped): blocks per launch for all the MLP's layers together
_GROUP_BLOCKS = {0: 1024, 1: 256, 2: 512}


# weight-gradient engine of the bf16 modes: "wide" (mms_gemm_tn_wide: 256 x 256 tiles, operand rows read once per
# slice; SDF MLP 0.52 -> 0.36 ms alone, scripts/tn_wide_bench.py) or "tiled" (mms_gemm_tn_grouped: 128 x 128 tiles);
# MMS_TN_ENGINE overrides (A/B measurement)
TN_ENGINE = os.environ.get("MMS_TN_ENGINE", "wide")
_WIDE_BLOCKS = 256
TN_STAGE_ROWS = int(os.environ.get("MMS_TN_STAGE", "16"))
TN_WORKSPACE = os.environ.get("MMS_TN_WS", "0") == "1"


def _aligned_item(it) -> bool:
    A, B = it[3], it[4]
    return all(t.data_ptr() % 16 == 0 and t.stride(0) % 4 == 0 and t.stride(1) == 1 for t in (A, B))


def gemm_tn_grouped(items, prec: int, target_blocks: Optional[int] = None, engine: Optional[str] = None,
                    stage_rows: Optional[int] = None):
    """items = [(N_out, K_in, rows, dZ [rows, >=N_out], X [rows, >=K_in], dW [N_out, K_in], db [N_out] or None)]:
    dW += dZ^T X and db += colsum(dZ) for every item in one launch (<= 5 items)."""
    n = len(items)
    I64 = ctypes.c_int64 * n
    VP = ctypes.c_void_p * n
    engine = engine or TN_ENGINE
    # the wide engine's 256-row tiles pay for MLPs with 256-wide layers; the 64-wide modality heads stay on 128 tiles
    wide = engine == "wide" and int(prec) in (1, 2) and all(_aligned_item(it) for it in items) and \
        max(it[0] for it in items) >= 128
    if wide:
        entry = "mms_gemm_tn_wide"
        target = int(os.environ.get("MMS_TN_BLOCKS", "0")) or target_blocks or _WIDE_BLOCKS
    else:
        entry = "mms_gemm_tn_grouped"
        target = int(os.environ.get("MMS_TN_BLOCKS", "0")) or target_blocks or _GROUP_BLOCKS.get(int(prec), 512)
    extra = ()
    if wide:
        # the slices' partial tiles go through a scratch buffer and a deterministic reduce launch (plain stores instead
        # of 256 KB of float atomics per block); MMS_TN_WS=0 keeps the atomics
        ws = torch.empty((target + 16) * 65536, device=items[0][3].device) if TN_WORKSPACE else None
        extra = (int(stage_rows or TN_STAGE_ROWS), None if ws is None else ws.data_ptr(),
                 0 if ws is None else ws.numel())
    _lib.call(entry, int(prec), n, I64(*[it[0] for it in items]), I64(*[it[1] for it in items]),
              I64(*[it[2] for it in items]), VP(*[it[3].data_ptr() for it in items]),
              I64(*[it[3].stride(0) for it in items]), VP(*[it[4].data_ptr() for it in items]),
              I64(*[it[4].stride(0) for it in items]), VP(*[it[5].data_ptr() for it in items]),
              I64(*[it[5].stride(0) for it in items]),
              VP(*[(it[6].data_ptr() if it[6] is not None else None) for it in items]), target, *extra, _stream())


def gemm_tn_wide16(items, target_blocks: Optional[int] = None):
    """items = [(N_out, K_in, rows, dZ, rinv or None, emax or None, X, dW, db or None)] in ONE launch
    (mms_gemm_tn_wide16): dW += dZ^T X and db += colsum(dZ).  dZ fp16 row-scaled with rinv / emax (mms_mlp_chain prec
    6 with rinv; emax a 1-element int32 view): one fp16 MFMA per product; dZ fp32 (rinv None): split bf16x3.  X fp32 or
    fp16 rows (its dtype).  <= 5 items."""
    n = len(items)
    I64 = ctypes.c_int64 * n
    VP = ctypes.c_void_p * n
    target = int(os.environ.get("MMS_TN_BLOCKS", "0")) or target_blocks or _WIDE_BLOCKS
    _lib.call("mms_gemm_tn_wide16", n, I64(*[it[0] for it in items]), I64(*[it[1] for it in items]),
              I64(*[it[2] for it in items]), VP(*[it[3].data_ptr() for it in items]),
              I64(*[it[3].stride(0) for it in items]), VP(*[_ptr(it[4]) for it in items]),
              VP(*[_ptr(it[5]) for it in items]), VP(*[it[6].data_ptr() for it in items]),
              I64(*[it[6].stride(0) for it in items]),
              (ctypes.c_int * n)(*[int(it[6].dtype == torch.float16) for it in items]),
              VP(*[it[7].data_ptr() for it in items]), I64(*[it[7].stride(0) for it in items]),
              VP(*[_ptr(it[8]) for it in items]), target, _stream())


def _ptr(t):
    return None if t is None else t.data_ptr()


# ----------------------------------------------------------------------------------------------
# Muon: orthogonalised updates of weight matrices
# ----------------------------------------------------------------------------------------------
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)   # torch.optim.Muon's quintic
_MATRIX_DTYPES = {torch.float32: 0, torch.bfloat16: 1}


_HERE = contextlib.nullcontext()


def _stream_of(t: torch.Tensor) -> int:
    """The current stream of ``t``'s device (torch.cuda.current_stream's handle at a fifth of its host time)."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _on_device(t: torch.Tensor):
    """The device of ``t`` as the current one (nothing to do if it is already): streams and launches go to it."""
    return _HERE if t.get_device() == torch.cuda.current_device() else torch.cuda.device(t.device)


def _matrices(t: torch.Tensor, what: str, copy: bool):
    """(tensor, batch, rows, cols, leading dimension, distance of a stack's matrices) of [..., rows, cols]; a layout
    that the kernels do not read in place is copied if ``copy``, else refused."""
    if t.dim() == 2 and t.is_contiguous():     # the common case, at a few hundred ns of host time
        rows, cols = t.shape
        return t, 1, rows, cols, cols, 0
    if t.dim() < 2:
        raise ValueError(f"{what} must have at least two dimensions, got shape {tuple(t.shape)}")
    rows, cols = t.shape[-2:]

    def in_place(x):
        return x.numel() == 0 or ((cols == 1 or x.stride(-1) == 1) and (rows == 1 or x.stride(-2) >= cols))
    if not in_place(t):
        if not copy:
            raise ValueError(f"{what}: rows must be contiguous and not overlap, got strides {t.stride()}")
        t = t.contiguous()
    if t.dim() > 3:
        t = t.reshape(-1, rows, cols) if copy else t.view(-1, rows, cols)
    ld = cols if rows == 1 else t.stride(-2)
    batch = t.shape[0] if t.dim() == 3 else 1
    bs = 0 if batch <= 1 else t.stride(0)
    if batch > 1 and t.numel() and bs < (rows - 1) * ld + cols:
        if not copy:
            raise ValueError(f"{what}: stacked matrices must not overlap, got strides {t.stride()}")
        t = t.contiguous()
        ld, bs = cols, rows * cols
    return t, batch, rows, cols, ld, bs


class _MatrixTable:
    """Host tables of several matrices for mms_newton_schulz / mms_muon_step."""

    def __init__(self, mats):
        n = self.n = len(mats)
        I64, VP = ctypes.c_int64 * n, ctypes.c_void_p * n
        self.keep, batch, rows, cols, ld, bs = zip(*mats)
        self.batch, self.rows, self.cols, self.ld, self.bs = I64(*batch), I64(*rows), I64(*cols), I64(*ld), I64(*bs)
        self.ptr = VP(*[t.data_ptr() for t in self.keep])


def _muon_workspace(tab: _MatrixTable, prec: int, device) -> torch.Tensor:
    need = ctypes.c_int64(0)
    _lib.call("mms_muon_workspace", tab.n, tab.batch, tab.rows, tab.cols, prec, ctypes.addressof(need))
    return torch.empty(max(1, need.value), dtype=torch.uint8, device=device)


def _check_matrices(ts, what: str):
    _check_dev(*ts)
    device = ts[0].device if ts else None
    for t in ts:
        if t.dtype not in _MATRIX_DTYPES:
            raise TypeError(f"{what} must be float32 or bfloat16, got {t.dtype}")
        if t.device != device:
            raise ValueError(f"{what} must be on one device, got {device} and {t.device}")


def _written(*ts: torch.Tensor):
    """The kernels wrote these tensors: a backward pass that saved one of them before is to notice."""
    torch.autograd.graph.increment_version(ts)


def newton_schulz(mats, steps: int = 5, coefficients=NS_COEFFICIENTS, eps: float = 1e-7, prec: Optional[int] = None):
    """The nearest semi-orthogonal matrix, approximately, of each matrix by Newton-Schulz products:
    X = G / max(|G|_F, eps), then ``steps`` times X <- a X + (b A + c A A) X with A = X X^T (X^T X for tall G) -- the
    iteration of torch.optim.Muon.

    ``mats``: a tensor [..., rows, cols] (a stack of matrices) or a list of such; float32 or bfloat16; returns the
    same structure, contiguous and without autograd history.  A zero matrix gives zeros, one with NaN or infinities NaN.
    All matrices share the same few launches.  Coefficients with which a singular value of X before the last step, of A or
    of b A + c A A can pass 60000 are refused.

    ``prec``: 0 (or None) fp32's accuracy whatever the type -- a bfloat16 result is off by its own rounding alone; 1
    bfloat16's accuracy for matrices of more than 128 rows and columns in about half of the time (8 x 1024 x 4096
    bfloat16: 1.00 ms for 1.92, off by 1.84e-3 of the result's norm for 1.66e-3)."""
    if isinstance(mats, torch.Tensor):
        return newton_schulz([mats], steps, coefficients, eps, prec)[0]
    mats = list(mats)
    _check_matrices(mats, "newton_schulz: matrices")
    prec = int(prec or 0)
    a, b, c = (float(x) for x in coefficients)
    outs = [torch.empty_like(m, memory_format=torch.contiguous_format) for m in mats]   # (half of torch.empty's time)
    for dtype, bf16 in _MATRIX_DTYPES.items():
        pick = [i for i, m in enumerate(mats) if m.dtype == dtype]
        if not pick:
            continue
        with _on_device(mats[0]):
            g = _MatrixTable([_matrices(mats[i], "newton_schulz: matrix", True) for i in pick])
            o = _MatrixTable([_matrices(outs[i], "newton_schulz: result", False) for i in pick])
            ws = _muon_workspace(g, prec, mats[0].device)
            _lib.call("mms_newton_schulz", g.n, g.batch, g.rows, g.cols, g.ptr, g.ld, g.bs, o.ptr, o.ld, o.bs, bf16,
                      prec, int(steps), a, b, c, float(eps), ws.data_ptr(), ws.numel(), _stream_of(mats[0]))
    return outs


def muon_scale(rows: int, cols: int, adjust: Optional[str] = None) -> float:
    """The learning rate's factor for a rows x cols matrix (torch.optim.Muon's adjust_lr_fn)."""
    if adjust in (None, "original"):
        return max(1.0, rows / max(1, cols)) ** 0.5
    if adjust == "match_rms_adamw":
        return 0.2 * max(rows, cols) ** 0.5
    raise ValueError(f"adjust must be 'original' or 'match_rms_adamw', got {adjust!r}")


def muon_step(params, grads, momenta, lr: float, momentum: float = 0.95, nesterov: bool = True,
              weight_decay: float = 0.1, steps: int = 5, coefficients=NS_COEFFICIENTS, eps: float = 1e-7,
              adjust: Optional[str] = None, prec: Optional[int] = None, sumsq: Optional[torch.Tensor] = None,
              max_norm: float = 0.0, hyper: Optional[torch.Tensor] = None) -> None:
    """One Muon step of weight matrices, in place:
    m <- m + (1 - momentum)(g - m), u = g + momentum (m - g) (``nesterov``) or m,
    p <- (1 - lr weight_decay) p - lr scale newton_schulz(u), scale = ``muon_scale(rows, cols, adjust)``.

    ``params`` / ``grads``: lists of [..., rows, cols] tensors of one type each, float32 or bfloat16; ``momenta``:
    float32, contiguous, zeros before the first step.  Weights or momenta that overlap others of the call are refused (a
    list's types are stepped one after the other, each by itself).  ``sumsq`` (device, one float) with ``max_norm``: the gradients
    are clipped by min(1, max_norm / (sqrt(sumsq) + 1e-6)).  ``hyper`` (device): [1 - lr weight_decay, -lr] read by the
    kernels in place of the arguments (graph replays).  ``coefficients``, ``prec``: as newton_schulz's."""
    params, grads, momenta = list(params), list(grads), list(momenta)
    if not len(params) == len(grads) == len(momenta):
        raise ValueError(f"muon_step: {len(params)} weights, {len(grads)} gradients, {len(momenta)} momenta")
    if not params:
        return
    _check_matrices(params, "muon_step: weights")
    _check_dev(*grads, *momenta, sumsq, hyper)
    device = params[0].device
    for p, g, m in zip(params, grads, momenta):
        shape = p.shape
        if g.shape != shape or m.shape != shape:
            raise ValueError(f"muon_step: weights {tuple(p.shape)}, gradient {tuple(g.shape)}, momentum "
                             f"{tuple(m.shape)} must have one shape")
        if g.dtype != p.dtype or m.dtype != torch.float32 or not m.is_contiguous():
            raise ValueError("muon_step: gradients have their weights' type, momenta are contiguous float32")
        if g.device != device or m.device != device:
            raise ValueError("muon_step: weights, gradients and momenta must be on one device")
    for t, k in ((sumsq, 1), (hyper, 2)):
        if t is not None and (t.dtype != torch.float32 or t.numel() < k or not t.is_contiguous()
                              or t.device != params[0].device):
            raise ValueError("muon_step: sumsq and hyper are contiguous float32 on the weights' device")
    if sumsq is not None and not max_norm > 0.0:
        raise ValueError(f"muon_step: clipping by sumsq needs a positive max_norm, got {max_norm}")
    prec = int(prec or 0)
    a, b, c = (float(x) for x in coefficients)
    for dtype, bf16 in _MATRIX_DTYPES.items():
        pick = [i for i, p in enumerate(params) if p.dtype == dtype]
        if not pick:
            continue
        with torch.no_grad(), _on_device(params[0]):
            w = _MatrixTable([_matrices(params[i], "muon_step: weights", False) for i in pick])
            g = _MatrixTable([_matrices(grads[i], "muon_step: gradient", True) for i in pick])
            m = (ctypes.c_void_p * w.n)(*[momenta[i].data_ptr() for i in pick])
            for what, ptrs in (("weights", w.ptr), ("momenta", m)):
                full = [q for q, b, r, c in zip(ptrs, w.batch, w.rows, w.cols) if b * r * c]
                if len(set(full)) < len(full):
                    raise ValueError(f"muon_step: the same {what} twice")
            scale = (ctypes.c_float * w.n)(*[muon_scale(w.rows[k], w.cols[k], adjust) for k in range(w.n)])
            ws = _muon_workspace(w, prec, params[0].device)
            _lib.call("mms_muon_step", w.n, w.batch, w.rows, w.cols, w.ptr, w.ld, w.bs, g.ptr, g.ld, g.bs, m, scale,
                      bf16, prec, int(steps), a, b, c, float(eps), float(momentum), int(bool(nesterov)), _ptr(sumsq),
                      float(max_norm), _ptr(hyper), 1.0 - float(lr) * float(weight_decay), -float(lr), ws.data_ptr(),
                      ws.numel(), _stream_of(params[0]))
        _written(*(params[i] for i in pick), *(momenta[i] for i in pick))


# ----------------------------------------------------------------------------------------------
# learned row tables
# ----------------------------------------------------------------------------------------------
_TABLE_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_MAX_INDICES = (1 << 24) - 1      # of one mms_embedding_* call


def _check_table(ids: torch.Tensor, rows: torch.Tensor, what: str) -> int:
    if not (ids.is_cuda and rows.is_cuda):
        _check_dev(ids, rows)
    if ids.dtype is not torch.int64 and ids.dtype is not torch.int32:
        raise TypeError(f"embedding: indices must be int32 or int64, got {ids.dtype}")
    dt = _TABLE_DTYPES.get(rows.dtype)
    if dt is None:
        raise TypeError(f"embedding: {what} must be float32, bfloat16 or float16, got {rows.dtype}")
    if ids.get_device() != rows.get_device():
        raise ValueError(f"embedding: indices on {ids.device}, {what} on {rows.device}")
    return dt


def _flat_ids(ids: torch.Tensor):
    """(tensor, elements between two indices): a column of a coordinate tensor is read where it lies."""
    if ids.is_contiguous():
        return ids, 1
    lead = [(s, st) for s, st in zip(ids.shape, ids.stride()) if s != 1]
    if ids.numel() and len(lead) == 1 and lead[0][1] > 0:
        return ids, lead[0][1]
    return ids.contiguous(), 1


def _rows2d(t: torch.Tensor, dim: int) -> torch.Tensor:
    t = t.reshape(-1, dim) if t.dim() != 2 else t
    return t if t.stride(1) == 1 and (t.shape[0] <= 1 or t.stride(0) >= dim) else t.contiguous()


def embedding(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """out[..., :] = scale * table[ids[...], :]; ids int32 / int64 of any shape, table [rows, dim] float32, bfloat16 or
    float16.  An index outside the table gives a row of zeros.  Without autograd history (EmbeddingFunction has it)."""
    dt = _check_table(ids, table, "the table")
    if table.dim() != 2 or table.shape[0] == 0 or table.shape[1] == 0:
        raise ValueError(f"embedding: the table must be [rows, dim], got {tuple(table.shape)}")
    rows, dim = table.shape
    t = table if table.is_contiguous() or (table.stride(1) == 1 and table.stride(0) >= dim) else table.contiguous()
    out = torch.empty(*ids.shape, dim, dtype=table.dtype, device=table.device)
    flat, stride = _flat_ids(ids)
    n = ids.numel()
    with _on_device(t):
        for i in range(0, n, _MAX_INDICES):
            _lib.call("mms_embedding_fwd", flat.data_ptr() + i * stride * ids.element_size(), ids.dtype is torch.int64,
                      stride, min(n - i, _MAX_INDICES), t.data_ptr(), dim if rows == 1 else t.stride(0), rows, dim, dt,
                      scale, out.data_ptr() + i * dim * t.element_size(), dim, _stream_of(t))
    return out


def _rows_overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Do two tensors of rows [..., dim] share memory?  Columns of one buffer, side by side, do not; rows of different
    strides whose ranges meet count as if they did."""
    if a.numel() == 0 or b.numel() == 0 or a.untyped_storage().data_ptr() != b.untyped_storage().data_ptr():
        return False

    def span(t):
        return t.data_ptr(), t.data_ptr() + (sum((s - 1) * st for s, st in zip(t.shape, t.stride())) + 1) * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    if a1 <= b0 or b1 <= a0:
        return False
    if a.dim() != 2 or b.dim() != 2 or a.stride(0) != b.stride(0) or a.stride(1) != 1 or b.stride(1) != 1 or a.stride(0) == 0:
        return True
    es = a.element_size()
    ld, d = a.stride(0) * es, (b0 - a0) % (a.stride(0) * es)
    return not (d >= a.shape[1] * es and d + b.shape[1] * es <= ld)


@functools.lru_cache(maxsize=256)
def _embedding_workspace(n: int, rows: int, dim: int, dt: int) -> int:
    need = ctypes.c_int64(0)
    _lib.call("mms_embedding_bwd_workspace", n, rows, dim, dt, ctypes.addressof(need))
    return need.value


def embedding_backward(ids: torch.Tensor, dout: torch.Tensor, rows: int, scale: float = 1.0,
                       padding_idx: Optional[int] = None, out: Optional[torch.Tensor] = None,
                       accumulate: bool = False) -> torch.Tensor:
    """The table's gradient [rows, dim] in ``dout``'s type: scale * the sum of dout over the positions of each row, in
    fp32 and in an order that ``ids`` alone fixes (the same bits on each call).  Positions whose index is
    ``padding_idx`` or outside the table add nothing, whatever ``dout`` holds there.  ``out``: written in place, or
    added into with ``accumulate``.  At most 2^24 - 1 positions (more: in parts, with ``accumulate``)."""
    dt = _check_table(ids, dout, "the gradient")
    dim = dout.shape[-1] if dout.dim() else 0
    if dim == 0 or dout.shape[:-1] != ids.shape or rows < 1:
        raise ValueError(f"embedding_backward: indices {tuple(ids.shape)} need a gradient [..., dim], got "
                         f"{tuple(dout.shape)} for {rows} rows")
    if out is None:
        if accumulate:
            raise ValueError("embedding_backward: accumulate needs out")
        out = torch.empty(rows, dim, dtype=dout.dtype, device=dout.device)
    elif tuple(out.shape) != (rows, dim) or out.dtype != dout.dtype or out.device != dout.device or \
            (dim > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < dim):
        raise ValueError(f"embedding_backward: out must be [{rows}, {dim}] {dout.dtype} with contiguous rows on "
                         f"{dout.device}")
    elif _rows_overlap(out, dout):
        raise ValueError("embedding_backward: out must not share memory with the gradient it is the sum of")
    pad = -1
    if padding_idx is not None:
        if not -rows <= padding_idx < rows:
            raise ValueError(f"embedding_backward: padding_idx {padding_idx} is outside the table's {rows} rows")
        pad = padding_idx % rows
    d = _rows2d(dout, dim)
    flat, stride = _flat_ids(ids)
    n = ids.numel()
    need = _embedding_workspace(n, rows, dim, dt)
    with _on_device(dout):
        ws = torch.empty(need, dtype=torch.uint8, device=dout.device) if need else None
        _lib.call("mms_embedding_bwd", flat.data_ptr(), ids.dtype is torch.int64, stride, n, d.data_ptr(),
                  dim if n <= 1 else d.stride(0), rows, dim, dt, scale, pad, out.data_ptr(),
                  dim if rows == 1 else out.stride(0), bool(accumulate), _ptr(ws), need, _stream_of(dout))
    _written(out)
    return out


class EmbeddingFunction(torch.autograd.Function):
    """Learned row table forward / backward on the HIP kernels: apply(ids, table, scale=1.0, padding_idx=None).  Once
    differentiable: a derivative of its gradient raises.  At most 2^24 - 1 indices where the table wants a gradient."""

    @staticmethod
    def forward(ctx, ids, table, scale: float = 1.0, padding_idx: Optional[int] = None):
        if ctx.needs_input_grad[1] and ids.numel() > _MAX_INDICES:
            raise ValueError(f"EmbeddingFunction: {ids.numel()} indices, the gradient takes up to {_MAX_INDICES}")
        ctx.save_for_backward(ids)
        ctx.cfg = (table.shape[0], float(scale), padding_idx)
        return embedding(ids, table, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        (ids,) = ctx.saved_tensors
        rows, scale, padding_idx = ctx.cfg
        dtable = embedding_backward(ids, dout, rows, scale, padding_idx) if ctx.needs_input_grad[1] else None
        return None, dtable, None, None
