"""A gated feed-forward block and what a training step does with its gradients
(include/mtffn.h):

  gated_linear             h = act(x·Wgᵀ + bg) * (x·Wuᵀ + bu), in fp32 or from 8-bit rows
                           and weights
  gated_linear_backward    its gradients
  gate, gate_backward      the activation and product alone, for projections that another
                           operator gives (linear_q4)
  grad_norm                the norm of all tensors of a list
  clip_grad_norm           ... and the tensors scaled down to a largest norm

Like the rest of the package: GPU tensors, views read in place, work on the current stream
or on `stream`, ValueError for wrong shapes, types and devices, RuntimeError where a launch
fails.  None has a counterpart in the reference.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Sequence, Union

import torch

from . import (MT_ERR_WORKSPACE, MatF32, _api, _check, _handle, _nbytes, _ptr, _require_gpu,
               _stream, lib, linear_backward, mat, native)
from .lowbit import (Q8Plan, Q8Rows, RowsQ8, _empty, _matrix, _rows, _vector, _ws,
                     linear_backward_q8)

MAX_EXTENT = (1 << 31) - (1 << 16)   # of a view's rows and columns
ACTIVATIONS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")   # mt_activation


class GatedLinear(NamedTuple):
    """What gated_linear gives: h [R, F], and the projections gu [R, 2F] (None unless kept)."""
    h: torch.Tensor
    gu: Optional[torch.Tensor]


class GatePlan(ctypes.Structure):
    _fields_ = [("kind", ctypes.c_int32), ("tile_rows", ctypes.c_int32),
                ("tile_cols", ctypes.c_int32), ("splits", ctypes.c_int32),
                ("vector_rows", ctypes.c_int32)]


_P, _V, _I64, _F, _S = (ctypes.POINTER, ctypes.c_void_p, ctypes.c_int64, ctypes.c_float,
                        ctypes.c_size_t)
_M, _Q, _I = _P(MatF32), _P(RowsQ8), ctypes.c_int
SIGS = {
    "mt_gated_linear_f32": (_I, [_M, _M, _V, _I64, _I, _M, _M, _V, _S, _V]),
    "mt_gated_linear_workspace_f32": (_S, [_M, _M]),
    "mt_gated_linear_plan_f32": (_I, [_M, _M, _P(GatePlan)]),
    "mt_gated_linear_q8": (_I, [_Q, _Q, _V, _I64, _I, _M, _M, _V, _S, _V]),
    "mt_gated_linear_q8_workspace": (_S, [_Q, _Q]),
    "mt_gated_linear_q8_plan": (_I, [_I64] * 3 + [_P(Q8Plan)]),
    "mt_gate_f32": (_I, [_M, _I, _M, _V]),
    "mt_gate_backward_f32": (_I, [_M, _M, _I, _M, _V]),
    "mt_gate_backward_bias_f32": (_I, [_M, _M, _I, _M, _V, _I64, _F, _V, _S, _V]),
    "mt_gate_backward_bias_workspace_f32": (_S, [_I64, _I64]),
    "mt_grad_norm_f32": (_I, [_M, _I64, _V, _V, _S, _V]),
    "mt_clip_grad_norm_f32": (_I, [_M, _M, _I64, _F, _F, _V, _V, _S, _V]),
    "mt_grad_norm_workspace_f32": (_S, [_I64]),
}


def _act(name: str, what: str) -> int:
    if name not in ACTIVATIONS:
        raise ValueError(f"{what}: act must be one of {', '.join(ACTIVATIONS)}")
    return ACTIVATIONS.index(name)


def _here(*ts) -> None:
    """float32 tensors of the current device, whose stream the work goes to."""
    for t in ts:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise ValueError("minitensor_amd kernels take GPU tensors only")
        _require_gpu(t)
        if t.get_device() != torch.cuda.current_device():
            raise ValueError("tensors must be on the current device")


def _features(n: int, what: str) -> int:
    if n % 2:
        raise ValueError(f"{what}: expected gates and as many up columns, not {n} in all")
    return n // 2


@_api
def gated_linear(x: Union[torch.Tensor, Q8Rows], w: Union[torch.Tensor, Q8Rows],
                 b: Optional[torch.Tensor] = None, act: str = "silu", keep: bool = False,
                 out: Optional[torch.Tensor] = None, ws=None, stream=None) -> GatedLinear:
    """h = act(x·Wgᵀ + bg) * (x·Wuᵀ + bu) with w [2F, K] and b [2F], the gates first; x and w
    both in float32 or both in 8 bits.

    `keep`: the projections too, for gated_linear_backward."""
    a = _act(act, "gated_linear")
    q8 = isinstance(x, Q8Rows)
    if q8 != isinstance(w, Q8Rows):
        raise ValueError("gated_linear: x and w must both be float32 or both Q8Rows")
    r = native().gated_linear(x[0] if q8 else x, x[1] if q8 else None, w[0] if q8 else w,
                              w[1] if q8 else None, b, a, bool(keep), out, ws, _handle(stream))
    if r is not None:
        return GatedLinear(*r)
    if q8:
        xd, wd, like = _rows(x), _rows(w), x[0]
        _here(x[1], w[1])
        (n, k), (f2, wk) = x[0].shape, w[0].shape
    else:
        _here(x, w)
        if x.dim() != 2 or w.dim() != 2:
            raise ValueError("gated_linear: expected x [R, K] and w [2F, K]")
        xd, wd, like = mat(x), mat(w), x
        (n, k), (f2, wk) = x.shape, w.shape
    f = _features(f2, "gated_linear")
    if k != wk:
        raise ValueError(f"gated_linear: x has {k} inputs, the weight {wk}")
    _here(b, out)
    bp, bs = _vector(b, f2, "gated_linear: bias")
    if out is None:
        out = _empty((n, f), like)
    gu = _empty((n, f2), like) if keep else None
    query = lib().mt_gated_linear_q8_workspace if q8 else lib().mt_gated_linear_workspace_f32
    need = query(ctypes.byref(xd), ctypes.byref(wd))
    ws = _ws(ws, need, like)
    fn, name = ((lib().mt_gated_linear_q8, "mt_gated_linear_q8") if q8 else
                (lib().mt_gated_linear_f32, "mt_gated_linear_f32"))
    rc = fn(ctypes.byref(xd), ctypes.byref(wd), bp, bs, a, _matrix(out, (n, f), "gated_linear: out"),
            _matrix(gu, (n, f2), "gu"), _ptr(ws), _nbytes(ws), _stream(stream))
    _check(rc, name)
    return GatedLinear(out, gu)


@_api
def gate(gu: torch.Tensor, act: str = "silu", out: Optional[torch.Tensor] = None,
         stream=None) -> torch.Tensor:
    """act(gu[:, :F]) * gu[:, F:] of projections [R, 2F]."""
    a = _act(act, "gate")
    r = native().gate(gu, a, out, _handle(stream))
    if r is not None:
        return r
    _here(gu, out)
    if gu.dim() != 2:
        raise ValueError("gate: expected projections [R, 2F]")
    n, f = gu.shape[0], _features(gu.shape[1], "gate")
    if out is None:
        out = _empty((n, f), gu)
    rc = lib().mt_gate_f32(mat(gu), a, _matrix(out, (n, f), "gate: out"), _stream(stream))
    _check(rc, "mt_gate_f32")
    return out


@_api
def gate_backward(dh: torch.Tensor, gu: torch.Tensor, act: str = "silu",
                  out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """The gradient [R, 2F] at the projections, from that at h; out may be gu itself."""
    a = _act(act, "gate_backward")
    r = native().gate_backward(dh, gu, a, out, _handle(stream))
    if r is not None:
        return r
    _here(dh, gu, out)
    if dh.dim() != 2 or gu.dim() != 2 or gu.shape != (dh.shape[0], 2 * dh.shape[1]):
        raise ValueError("gate_backward: expected dh [R, F] and projections [R, 2F]")
    if out is None:
        out = _empty(gu.shape, gu)
    rc = lib().mt_gate_backward_f32(mat(dh), mat(gu), a, _matrix(out, gu.shape, "gate_backward: out"),
                                    _stream(stream))
    _check(rc, "mt_gate_backward_f32")
    return out


@_api
def gated_linear_backward(dh: torch.Tensor, gu: torch.Tensor, x: Union[torch.Tensor, Q8Rows],
                          w: Optional[torch.Tensor] = None, act: str = "silu",
                          need_dw: bool = True, need_db: bool = True,
                          dgu: Optional[torch.Tensor] = None, dx=None, dw=None, db=None,
                          beta_w: float = 0.0, beta_b: float = 0.0, ws=None, stream=None):
    """(dX, dW, db) of gated_linear from the gradient at h and the kept projections; x in
    float32, or kept in 8 bits.  dX is None without a `w` (a first layer needs none).

    `dgu` [R, 2F]: where the gradient at the projections goes, which may be gu itself.
    dW = beta_w·dw + ∂L/∂W and db = beta_b·db + ∂L/∂b where a dw, db is passed."""
    a, q8 = _act(act, "gated_linear_backward"), isinstance(x, Q8Rows)
    r = native().gated_linear_backward(dh, gu, x[0] if q8 else x, x[1] if q8 else None, w, a,
                                       bool(need_dw), bool(need_db), dgu, dx, dw, db, beta_w, beta_b,
                                       ws, _handle(stream))
    if r is not None:
        return r
    # (all checks first: dgu may be written over gu)
    _here(dh, gu, dgu, x[1] if q8 else x, w, dx, dw, db)
    rows = x[0] if q8 else x
    if dh.dim() != 2 or rows.dim() != 2 or rows.shape[0] != dh.shape[0]:
        raise ValueError("gated_linear_backward: expected dh [R, F] and x [R, K]")
    (n, f), k = dh.shape, rows.shape[1]
    for t, shape, what in ((gu, (n, 2 * f), "gu"), (dgu, (n, 2 * f), "dgu"), (w, (2 * f, k), "w"),
                           (dx, (n, k), "dx"), (dw, (2 * f, k), "dw")):
        _matrix(t, shape, f"gated_linear_backward: {what}")
    _vector(db, 2 * f, "gated_linear_backward: db")
    if w is None and dx is not None:
        raise ValueError("gated_linear_backward: a dx to write to without the w that gives it")
    if (need_dw and dw is None and beta_w != 0.0) or (need_db and db is None and beta_b != 0.0):
        raise ValueError("gated_linear_backward: a beta without a gradient to add to")
    for t in (dgu, dx, dw, db):
        if t is not None and any(e > 1 and at == 0 for e, at in zip(t.shape, t.stride())):
            raise ValueError("gated_linear_backward: an output must not be an expanded view")
    if q8:
        _rows(x)
    if k >= MAX_EXTENT:
        raise ValueError(f"gated_linear_backward: x has {k} inputs")
    sums = not q8 and need_db and native().sums_in_pass(n, 2 * f, k)
    if ws is not None or sums:
        need = (lib().mt_linear_backward_q8_workspace_f32 if q8 else lib().mt_linear_workspace_f32)(n, k, 2 * f)
        if sums:
            need = max(need, lib().mt_gate_backward_bias_workspace_f32(n, f))
        ws = _ws(ws, need, dh)
        if _nbytes(ws) < need:
            _check(MT_ERR_WORKSPACE, "gated_linear_backward")
    if sums:
        if db is None:
            db = _empty((2 * f,), dh)
        if dgu is None:
            dgu = _empty((n, 2 * f), dh)
        rc = lib().mt_gate_backward_bias_f32(mat(dh), mat(gu), a, mat(dgu), *_vector(db, 2 * f, "db"),
                                             float(beta_b), _ptr(ws), _nbytes(ws), _stream(stream))
        _check(rc, "mt_gate_backward_bias_f32")
    else:
        dgu = gate_backward(dh, gu, act, dgu)
    if q8:
        return linear_backward_q8(dgu, x, w, need_dw, need_db, dx, dw, db, beta_w, beta_b, ws)
    # (without a w there is no dx, and nothing reads the one that stands in for it)
    any_w = x.new_empty((1, 1)).expand(2 * f, k) if w is None else w
    dx, dw, own = linear_backward(dgu, x, any_w, w is not None, need_dw, need_db and not sums, dx,
                                  dw, db, beta_w, beta_b, ws)
    return dx, dw if need_dw else None, (db if sums else own) if need_db else None


def _axes(g: torch.Tensor, o: torch.Tensor):
    """The sizes and both strides of as few axes as hold g and o, element by element: axes in
    the order of g's strides, neighbouring ones that run on in both as one."""
    if 0 in g.shape:
        return [(0, 1, 1)]
    axes = []
    for n, a, b in sorted(((n, a, b) for n, a, b in zip(g.shape, g.stride(), o.stride()) if n > 1),
                          key=lambda x: (-x[1], -x[2])):
        if axes and axes[-1][1] == a * n and axes[-1][2] == b * n:
            axes[-1] = (axes[-1][0] * n, a, b)
        else:
            axes.append((n, a, b))
    return axes


def _tensors(ts, outs, what: str):
    """Descriptors of the lists' tensors."""
    n = len(ts)
    g, o = (MatF32 * max(n, 1))(), (MatF32 * max(n, 1))()
    for i, (a, b) in enumerate(zip(ts, outs)):
        if a is None or b is None:
            raise ValueError(f"{what}: expected tensors")
        _here(a, b)
        if a.shape != b.shape:
            raise ValueError(f"{what}: an output must have its tensor's shape")
        axes = _axes(a, b)
        if len(axes) > 3:
            raise ValueError(f"{what}: a view of more than three strided axes")
        axes = [(1, 0, 0)] * (3 - len(axes)) + axes
        for d, t, k in ((g[i], a, 1), (o[i], b, 2)):
            d.base, d.offset = t.data_ptr(), 0
            d.batch, d.rows, d.cols = (x[0] for x in axes)
            d.batch_stride, d.row_stride, d.col_stride = (x[k] for x in axes)
    return g, o, n


@_api
def grad_norm(grads: Sequence[torch.Tensor], ws=None, stream=None) -> torch.Tensor:
    """sqrt of the sum of all squares of all tensors, a float32 scalar on their device; the
    sum is held in 64 bits."""
    return _clip(grads, None, None, 0.0, ws, stream, "grad_norm")


@_api
def clip_grad_norm(grads: Sequence[torch.Tensor], max_norm: float,
                   out: Optional[Sequence[torch.Tensor]] = None, eps: float = 1e-6, ws=None,
                   stream=None) -> torch.Tensor:
    """Scales all tensors by min(1, max_norm/(norm + eps)), in place or into the tensors `out`,
    and returns the norm that they had, a float32 scalar on their device.  max_norm and eps are
    taken in float32; each product is rounded once."""
    if max_norm is None:
        raise ValueError("clip_grad_norm: no largest norm (grad_norm only measures)")
    return _clip(grads, max_norm, out, eps, ws, stream, "clip_grad_norm")


def _clip(grads, most, out, eps, ws, stream, what):
    grads = list(grads)
    if not grads:
        raise ValueError(f"{what}: no tensors")
    outs = grads if out is None else list(out)
    if len(outs) != len(grads):
        raise ValueError(f"{what}: as many outputs as tensors")
    r = native().clip(grads, None if out is None else outs, most is not None,
                      0.0 if most is None else most, eps, ws, _handle(stream))
    if r is not None:
        return r
    g, o, n = _tensors(grads, outs, what)
    norm = _empty((), grads[0])
    ws = _ws(ws, lib().mt_grad_norm_workspace_f32(n), grads[0])
    if most is None:
        rc = lib().mt_grad_norm_f32(g, n, norm.data_ptr(), _ptr(ws), _nbytes(ws), _stream(stream))
    else:
        rc = lib().mt_clip_grad_norm_f32(g, o, n, float(most), float(eps), norm.data_ptr(), _ptr(ws),
                                         _nbytes(ws), _stream(stream))
    _check(rc, f"mt_{what}_f32")
    return norm
