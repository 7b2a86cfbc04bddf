"""Operators around a Linear layer whose activations are kept in 8 bits and
whose weights are served in 4 (include/mtlowbit.h):

  rms_norm, rms_norm_backward   RMS norm with the residual's addition, its rows
                                in fp32, in 8 bits, or both
  quantize_q8, dequantize_q8    rows kept in 8 bits for the backward pass
  linear_backward_q8            a Linear layer's gradients from such rows
  quantize_q4, dequantize_q4    a weight in 4 bits with a scale per group
  linear_q4                     F::linear over it, from fp32 or 8-bit rows

Like the rest of the package: GPU tensors, views read in place, work on the
current stream or on `stream`, ValueError for wrong shapes, types and devices,
RuntimeError where a launch fails.  None has a counterpart in the reference,
whose tensors are fp32 only.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Union

import torch

from . import (MatF32, _api, _check, _handle, _nbytes, _ptr, _require_gpu, _require_ws, _stream, lib,
               mat, native, workspace)


class Q8Rows(NamedTuple):
    """Rows in 8 bits: x[r, c] ~ q[r, c]·scale[r]; q int8 [R, C], scale float32 [R]."""
    q: torch.Tensor
    scale: torch.Tensor


class Q4Weight(NamedTuple):
    """A weight [N, K] in 4 bits: packed uint8 [N, 16·ceil(K/32)], input 2i in the
    low half of byte i and 2i + 1 in the high half, two's complement; scale float32
    [N, ceil(K/group)]; group 32, 64 or 128 inputs."""
    packed: torch.Tensor
    scale: torch.Tensor
    k: int
    group: int


class RmsNorm(NamedTuple):
    """What rms_norm gives: y (None unless asked for), h = x (+ residual), rstd [R],
    q8 = y in 8 bits (None unless asked for)."""
    y: Optional[torch.Tensor]
    h: torch.Tensor
    rstd: torch.Tensor
    q8: Optional[Q8Rows]


class RowsQ8(ctypes.Structure):
    _fields_ = [("q", ctypes.c_void_p), ("scale", ctypes.c_void_p), ("rows", ctypes.c_int64),
                ("cols", ctypes.c_int64), ("row_stride", ctypes.c_int64)]


class WeightQ4(ctypes.Structure):
    _fields_ = [("packed", ctypes.c_void_p), ("scale", ctypes.c_void_p), ("n", ctypes.c_int64),
                ("k", ctypes.c_int64), ("row_stride", ctypes.c_int64),
                ("scale_stride", ctypes.c_int64), ("group", ctypes.c_int32)]


class LowbitPlan(ctypes.Structure):
    _fields_ = [("tile_rows", ctypes.c_int32), ("splits", ctypes.c_int32),
                ("column_blocks", ctypes.c_int32)]


_P, _V, _I64, _F = ctypes.POINTER, ctypes.c_void_p, ctypes.c_int64, ctypes.c_float
_M, _Q, _W = _P(MatF32), _P(RowsQ8), _P(WeightQ4)
SIGS = {
    "mt_rms_norm_f32": (ctypes.c_int, [_M, _M, _V, _I64, _F, _M, _M, _Q, _V, _V]),
    "mt_rms_norm_backward_f32": (ctypes.c_int, [_M, _M, _V, _I64, _V, _M, _M, _V, _I64, _F, _V,
                                                ctypes.c_size_t, _V]),
    "mt_rms_norm_backward_workspace_f32": (ctypes.c_size_t, [_I64, _I64]),
    "mt_quantize_q8_f32": (ctypes.c_int, [_M, _Q, _V]),
    "mt_dequantize_q8_f32": (ctypes.c_int, [_Q, _M, _V]),
    "mt_linear_backward_q8_f32": (ctypes.c_int, [_M, _Q, _M, _M, _M, _F, _V, _I64, _F, _V,
                                                 ctypes.c_size_t, _V]),
    "mt_linear_backward_q8_workspace_f32": (ctypes.c_size_t, [_I64] * 3),
    "mt_quantize_q4_f32": (ctypes.c_int, [_M, _W, _V]),
    "mt_dequantize_q4_f32": (ctypes.c_int, [_W, _M, _V]),
    "mt_linear_q4_f32": (ctypes.c_int, [_M, _W, _V, _I64, _M, _V, ctypes.c_size_t, _V]),
    "mt_linear_q4_q8": (ctypes.c_int, [_Q, _W, _V, _I64, _M, _V, ctypes.c_size_t, _V]),
    "mt_linear_q4_workspace": (ctypes.c_size_t, [_I64] * 3),
    "mt_linear_q4_plan": (ctypes.c_int, [_I64] * 3 + [ctypes.c_int] * 2 + [_P(LowbitPlan)]),
    "mt_linear_backward_q8_plan": (ctypes.c_int, [_I64] * 3 + [_P(LowbitPlan)]),
}


def _bytes_on_gpu(t, dtype, what: str) -> None:
    if not isinstance(t, torch.Tensor) or t.device.type != "cuda" or t.dtype != dtype:
        raise ValueError(f"{what} must be a GPU tensor of {dtype}")


def _rows(xq: Q8Rows) -> RowsQ8:
    q, scale = xq
    _bytes_on_gpu(q, torch.int8, "Q8Rows.q")
    _require_gpu(scale)
    if q.dim() != 2 or (q.shape[1] > 1 and q.stride(1) != 1):
        raise ValueError("Q8Rows.q must be [R, C] with neighbouring elements in a row")
    if scale.shape != q.shape[:1] or (scale.numel() > 1 and scale.stride(0) != 1):
        raise ValueError("Q8Rows.scale must be [R], contiguous")
    return RowsQ8(q.data_ptr(), scale.data_ptr(), q.shape[0], q.shape[1],
                  q.stride(0) if q.shape[0] > 1 else q.shape[1])


def _weight(w: Q4Weight) -> WeightQ4:
    packed, scale, k, group = w
    _bytes_on_gpu(packed, torch.uint8, "Q4Weight.packed")
    _require_gpu(scale)
    if group not in (32, 64, 128):
        raise ValueError("Q4Weight.group must be 32, 64 or 128")
    if packed.dim() != 2 or scale.dim() != 2 or k < 0 or packed.shape[0] != scale.shape[0] or \
            packed.shape[1] != (k + 31) // 32 * 16 or scale.shape[1] != (k + group - 1) // group:
        raise ValueError("Q4Weight: expected packed [N, 16*ceil(k/32)] and scale [N, ceil(k/group)]")
    for t in (packed, scale):
        if t.shape[1] > 1 and t.stride(1) != 1:
            raise ValueError("Q4Weight: a row's elements must be neighbours")
    n = packed.shape[0]
    rs, ss = (packed.stride(0), scale.stride(0)) if n > 1 else packed.shape[1:] + scale.shape[1:]
    if packed.numel() and (packed.data_ptr() % 16 or rs % 16):
        raise ValueError("Q4Weight.packed: rows must start on multiples of 16 bytes")
    return WeightQ4(packed.data_ptr(), scale.data_ptr(), n, k, rs, ss, group)


def _vector(t: Optional[torch.Tensor], n: int, what: str):
    """(pointer, stride) of a float32 vector of n elements, or of none."""
    if t is None:
        return None, 0
    _require_gpu(t)
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{what} must be a vector of {n} elements")
    return t.data_ptr(), t.stride(0) if n > 1 else 1


def _matrix(t: Optional[torch.Tensor], shape, what: str):
    if t is None:
        return None
    _require_gpu(t)
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} must be {list(shape)}, not {list(t.shape)}")
    return ctypes.byref(mat(t))


def _empty(shape, like, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device=like.device)


def _ws(ws, need, like):
    _require_ws(ws)
    return ws if ws is not None else workspace(need, like.device)


@_api
def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
             residual: Optional[torch.Tensor] = None, eps: float = 1e-6, y: bool = True,
             q8: bool = False, h: Optional[torch.Tensor] = None, stream=None) -> RmsNorm:
    """h = x (+ residual); y = h / sqrt(mean(h²) + eps)·weight, row by row, in one pass.

    `y` and `q8` say whether the rows are wanted in fp32 and in 8 bits.  h is
    written where there is a residual or an `h` to write to, which may be x or
    residual itself; otherwise it is x."""
    r = native().rms_norm(x, weight, residual, eps, bool(y), bool(q8), h, _handle(stream))
    if r is None:
        _require_gpu(x, weight, residual, h)
        if x.dim() != 2:
            raise ValueError("rms_norm: expected x [R, C]")
        n, c = x.shape
        w, ws = _vector(weight, c, "rms_norm: weight")
        if h is None and residual is not None:
            h = _empty((n, c), x)
        out = _empty((n, c), x) if y else None
        rows = Q8Rows(_empty((n, c), x, torch.int8), _empty((n,), x)) if q8 else None
        rstd = _empty((n,), x)
        rc = lib().mt_rms_norm_f32(mat(x), _matrix(residual, x.shape, "rms_norm: residual"), w, ws,
                                   float(eps), _matrix(h, x.shape, "rms_norm: h"),
                                   _matrix(out, x.shape, "y"),
                                   ctypes.byref(_rows(rows)) if q8 else None, rstd.data_ptr(),
                                   _stream(stream))
        _check(rc, "mt_rms_norm_f32")
        return RmsNorm(out, x if h is None else h, rstd, rows)
    out, hh, rstd, q, scale = r
    return RmsNorm(out, hh, rstd, Q8Rows(q, scale) if q is not None else None)


@_api
def rms_norm_backward(dy: torch.Tensor, h: torch.Tensor, weight: Optional[torch.Tensor],
                      rstd: torch.Tensor, dh: Optional[torch.Tensor] = None, need_dh: bool = True,
                      need_dw: bool = True, out: Optional[torch.Tensor] = None,
                      dw: Optional[torch.Tensor] = None, beta: float = 0.0, ws=None, stream=None):
    """(gradient of h, gradient of the weight) from dy and the forward's h and rstd.

    `dh`: the gradient that arrives at h along the residual stream, added to the
    first (which may be written over it: out=dh); the gradient of the weight is
    beta·dw + ∂L/∂weight where a `dw` is passed."""
    r = native().rms_norm_backward(dy, h, weight, rstd, dh, bool(need_dh), bool(need_dw), out, dw,
                                   beta, ws, _handle(stream))
    if r is not None:
        return r
    _require_gpu(dy, h, weight, rstd, dh, out, dw)
    if dy.dim() != 2 or h.shape != dy.shape:
        raise ValueError("rms_norm_backward: expected dy and h [R, C]")
    n, c = dy.shape
    w, wst = _vector(weight, c, "rms_norm_backward: weight")
    rp, rst = _vector(rstd, n, "rms_norm_backward: rstd")
    if n > 1 and rst != 1:
        raise ValueError("rms_norm_backward: rstd must be contiguous")
    if need_dh and out is None:
        out = _empty((n, c), dy)
    if need_dw and dw is None:
        if beta != 0.0:
            raise ValueError("rms_norm_backward: beta without a dw to add to")
        dw = _empty((c,), dy)
    dwp, dws = _vector(dw if need_dw else None, c, "rms_norm_backward: dw")
    ws = _ws(ws, lib().mt_rms_norm_backward_workspace_f32(n, c) if need_dw else 0, dy)
    rc = lib().mt_rms_norm_backward_f32(
        mat(dy), mat(h), w, wst, rp, _matrix(dh, dy.shape, "rms_norm_backward: dh"),
        _matrix(out if need_dh else None, dy.shape, "rms_norm_backward: out"), dwp, dws, float(beta),
        _ptr(ws), _nbytes(ws), _stream(stream))
    _check(rc, "mt_rms_norm_backward_f32")
    return out if need_dh else None, dw if need_dw else None


@_api
def quantize_q8(x: torch.Tensor, out: Optional[Q8Rows] = None, stream=None) -> Q8Rows:
    """x [R, C] in 8 bits, a scale per row: scale = max(max|x[r]|/127, 2^-126), q to
    the nearest.  A row with an infinity or a NaN reads back as NaN."""
    if out is None:
        r = native().quantize_q8(x, _handle(stream))
        if r is not None:
            return Q8Rows(*r)
    _require_gpu(x)
    if x.dim() != 2:
        raise ValueError("quantize_q8: expected x [R, C]")
    if out is None:
        out = Q8Rows(_empty(x.shape, x, torch.int8), _empty(x.shape[:1], x))
    d = _rows(out)
    if out.q.shape != x.shape:
        raise ValueError("quantize_q8: out has the wrong shape")
    _check(lib().mt_quantize_q8_f32(mat(x), ctypes.byref(d), _stream(stream)), "mt_quantize_q8_f32")
    return out


@_api
def dequantize_q8(xq: Q8Rows, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """q·scale in float32."""
    r = native().dequantize_q8(xq[0], xq[1], out, _handle(stream))
    if r is not None:
        return r
    d = _rows(xq)
    if out is None:
        out = _empty(xq.q.shape, xq.q)
    m = _matrix(out, xq.q.shape, "dequantize_q8: out")
    _check(lib().mt_dequantize_q8_f32(ctypes.byref(d), m, _stream(stream)), "mt_dequantize_q8_f32")
    return out


@_api
def linear_backward_q8(dy: torch.Tensor, xq: Q8Rows, w: Optional[torch.Tensor] = None,
                       need_dw: bool = True, need_db: bool = True, dx=None, dw=None, db=None,
                       beta_w: float = 0.0, beta_b: float = 0.0, ws=None, stream=None):
    """linear_backward from an input that was kept in 8 bits: (dX = dY·W, dW = dYᵀ·x
    (+ beta_w·dw), db = Σ_rows dY (+ beta_b·db)).  dX is None without a `w` (a first
    layer needs none)."""
    r = native().linear_backward_q8(dy, xq[0], xq[1], w, bool(need_dw), bool(need_db), dx, dw, db,
                                    beta_w, beta_b, ws, _handle(stream))
    if r is not None:
        return r
    _require_gpu(dy, w, dx, dw, db)
    x = _rows(xq)
    if dy.dim() != 2 or dy.shape[0] != x.rows:
        raise ValueError("linear_backward_q8: expected dy [B, out] and rows [B, in]")
    n, fin, fout = x.rows, x.cols, dy.shape[1]
    wm = _matrix(w, (fout, fin), "linear_backward_q8: w")
    if w is None and dx is not None:
        raise ValueError("linear_backward_q8: a dx to write to without the w that gives it")
    if w is not None and dx is None:
        dx = _empty((n, fin), dy)
    if need_dw and dw is None:
        if beta_w != 0.0:
            raise ValueError("linear_backward_q8: beta_w without a dw to add to")
        dw = _empty((fout, fin), dy)
    if need_db and db is None:
        if beta_b != 0.0:
            raise ValueError("linear_backward_q8: beta_b without a db to add to")
        db = _empty((fout,), dy)
    dbp, dbs = _vector(db if need_db else None, fout, "linear_backward_q8: db")
    ws = _ws(ws, lib().mt_linear_backward_q8_workspace_f32(n, fin, fout), dy)
    rc = lib().mt_linear_backward_q8_f32(
        mat(dy), ctypes.byref(x), wm,
        _matrix(dx if w is not None else None, (n, fin), "linear_backward_q8: dx"),
        _matrix(dw if need_dw else None, (fout, fin), "linear_backward_q8: dw"), float(beta_w), dbp,
        dbs, float(beta_b), _ptr(ws), _nbytes(ws), _stream(stream))
    _check(rc, "mt_linear_backward_q8_f32")
    return dx if w is not None else None, dw if need_dw else None, db if need_db else None


@_api
def quantize_q4(w: torch.Tensor, group: int = 128, stream=None) -> Q4Weight:
    """A weight [N, K] in 4 bits: per group of inputs scale = max|w|/7, codes -7..7 to
    the nearest."""
    _require_gpu(w)
    if w.dim() != 2:
        raise ValueError("quantize_q4: expected w [N, K]")
    if group not in (32, 64, 128):
        raise ValueError("quantize_q4: group must be 32, 64 or 128")
    n, k = w.shape
    q = Q4Weight(_empty((n, (k + 31) // 32 * 16), w, torch.uint8),
                 _empty((n, (k + group - 1) // group), w), k, group)
    rc = lib().mt_quantize_q4_f32(mat(w), ctypes.byref(_weight(q)), _stream(stream))
    _check(rc, "mt_quantize_q4_f32")
    return q


@_api
def dequantize_q4(wq: Q4Weight, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """code·scale in float32, [N, K]."""
    d = _weight(wq)
    if out is None:
        out = _empty((d.n, d.k), wq.packed)
    m = _matrix(out, (d.n, d.k), "dequantize_q4: out")
    _check(lib().mt_dequantize_q4_f32(ctypes.byref(d), m, _stream(stream)), "mt_dequantize_q4_f32")
    return out


@_api
def linear_q4(x: Union[torch.Tensor, Q8Rows], wq: Q4Weight, b: Optional[torch.Tensor] = None,
              out: Optional[torch.Tensor] = None, ws=None, stream=None) -> torch.Tensor:
    """F::linear over a 4-bit weight: y = x·wᵀ + b, x in float32 or in 8 bits."""
    q8 = isinstance(x, Q8Rows)
    r = native().linear_q4(x[0] if q8 else x, x[1] if q8 else None, wq[0], wq[1], wq[2], wq[3], b,
                           out, ws, _handle(stream))
    if r is not None:
        return r
    d = _weight(wq)
    if q8:
        xd, rows, cols = _rows(x), x.q.shape[0], x.q.shape[1]
    else:
        _require_gpu(x)
        if x.dim() != 2:
            raise ValueError("linear_q4: expected x [B, in]")
        xd, (rows, cols) = mat(x), x.shape
    if cols != d.k:
        raise ValueError(f"linear_q4: x has {cols} inputs, the weight {d.k}")
    bp, bs = _vector(b, d.n, "linear_q4: bias")
    if out is None:
        out = _empty((rows, d.n), wq.packed)
    y = _matrix(out, (rows, d.n), "linear_q4: out")
    ws = _ws(ws, lib().mt_linear_q4_workspace(rows, d.k, d.n), wq.packed)
    fn = lib().mt_linear_q4_q8 if q8 else lib().mt_linear_q4_f32
    rc = fn(ctypes.byref(xd), ctypes.byref(d), bp, bs, y, _ptr(ws), _nbytes(ws), _stream(stream))
    _check(rc, "mt_linear_q4_q8" if q8 else "mt_linear_q4_f32")
    return out
