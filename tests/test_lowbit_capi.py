"""include/mtlowbit.h without a GPU: what the entry points refuse before they touch the
device, what they take as nothing to do, and the workspace queries."""
import ctypes

import pytest
import torch

import minitensor_amd as mt
from minitensor_amd.lowbit import RowsQ8, WeightQ4

OK, INVALID, WORKSPACE = mt.MT_OK, mt.MT_ERR_INVALID, mt.MT_ERR_WORKSPACE


def M(rows, cols, rs=None, cs=1, batch=1, bs=0, off=0, base=0x1000):
    return mt.MatF32(base, off, rows, cols, cols if rs is None else rs, cs, batch, bs)


def Q(rows, cols, rs=None, q=0x1000, scale=0x2000):
    return RowsQ8(q, scale, rows, cols, cols if rs is None else rs)


def W(n, k, group=128, rs=None, ss=None, packed=0x1000, scale=0x2000):
    return WeightQ4(packed, scale, n, k, (k + 31) // 32 * 16 if rs is None else rs,
                    -(-k // group) if ss is None else ss, group)


def R(x):
    return ctypes.byref(x) if x is not None else None


BAD_QUANTIZE = {
    "rows differ": (M(4, 8), Q(5, 8)),
    "columns differ": (M(4, 8), Q(4, 9)),
    "no codes": (M(4, 8), Q(4, 8, q=0)),
    "no scales": (M(4, 8), Q(4, 8, scale=0)),
    "rows over one another": (M(4, 8), Q(4, 8, rs=7)),
    "a batch": (M(4, 8, batch=2, bs=32), Q(4, 8)),
    "negative stride": (M(4, 8, rs=-8), Q(4, 8)),
    "no x": (M(4, 8, base=0), Q(4, 8)),
    "past 32 bits": (M(1 << 31, 8), Q(1 << 31, 8)),
    "blocks past 32 bits": (M(1, (1 << 31) - (1 << 16)), Q(1, (1 << 31) - (1 << 16))),
}


@pytest.mark.parametrize("case", sorted(BAD_QUANTIZE))
def test_quantize_q8_refuses(case):
    x, q = BAD_QUANTIZE[case]
    assert mt.lib().mt_quantize_q8_f32(R(x), R(q), None) == INVALID


def test_dequantize_q8_refuses():
    f = mt.lib().mt_dequantize_q8_f32
    assert f(R(Q(4, 8)), R(M(4, 9)), None) == INVALID
    assert f(R(Q(4, 8)), R(M(4, 8, rs=0)), None) == INVALID
    assert f(R(Q(4, 8)), R(M(4, 8, cs=0)), None) == INVALID
    assert f(R(Q(4, 8)), None, None) == INVALID
    assert f(R(Q(0, 8)), R(M(0, 8)), None) == OK


def rms(x=M(4, 8), r=None, w=0x3000, ws=1, eps=1e-6, h=None, y=None, q=None):
    return mt.lib().mt_rms_norm_f32(R(x), R(r), w, ws, eps, R(h), R(y), R(q), None, None)


def test_rms_norm_refuses():
    assert rms(r=M(4, 9)) == INVALID
    assert rms(y=M(3, 8)) == INVALID
    assert rms(y=M(4, 8, cs=0)) == INVALID
    assert rms(h=M(4, 8, rs=0)) == INVALID
    assert rms(q=Q(4, 9)) == INVALID
    assert rms(eps=-1.0) == INVALID
    assert rms(eps=float("nan")) == INVALID
    assert rms(ws=-1) == INVALID
    assert rms(x=M(4, 8, base=0)) == INVALID
    assert rms(x=None) == INVALID
    assert rms(x=M(0, 8)) == OK and rms(x=M(4, 0)) == OK


def test_rms_norm_backward_refuses():
    def call(dy=M(4, 8), h=M(4, 8), rstd=0x3000, dh0=None, dh=M(4, 8), dw=0x4000, dws=1, ws=None,
             n=0):
        return mt.lib().mt_rms_norm_backward_f32(R(dy), R(h), None, 0, rstd, R(dh0), R(dh), dw, dws,
                                                 0.0, ws, n, None)
    assert call(h=M(4, 9)) == INVALID
    assert call(rstd=None) == INVALID
    assert call(dh0=M(3, 8)) == INVALID
    assert call(dh=M(4, 8, cs=0)) == INVALID
    assert call(dws=0) == INVALID
    assert call() == WORKSPACE
    assert call(ws=0x5000, n=4) == WORKSPACE
    assert call(dh=None, dw=None) == OK
    assert mt.lib().mt_rms_norm_backward_workspace_f32(0, 8) == 0
    assert mt.lib().mt_rms_norm_backward_workspace_f32(100, 8) >= 32


BAD_WEIGHT = {
    "group": W(4, 64, group=16, ss=4),
    "packed off 16 bytes": W(4, 64, packed=0x1008),
    "row stride off 16 bytes": W(4, 64, rs=40),
    "rows over one another": W(4, 64, rs=16),
    "scales over one another": W(4, 256, ss=1),
    "no codes": W(4, 64, packed=0),
    "no scales": W(4, 64, scale=0),
    "negative n": W(-1, 64),
    "n past 2^26": W(1 << 26, 64),
    "k past 32 bits": W(4, (1 << 31) - 1),
    "scales far apart": W(4, 64, ss=1 << 22),
}


@pytest.mark.parametrize("case", sorted(BAD_WEIGHT))
def test_weights_are_checked(case):
    w = BAD_WEIGHT[case]
    n, k = max(w.n, 0), w.k
    assert mt.lib().mt_quantize_q4_f32(R(M(n, k)), R(w), None) == INVALID
    assert mt.lib().mt_dequantize_q4_f32(R(w), R(M(n, k)), None) == INVALID
    assert mt.lib().mt_linear_q4_f32(R(M(3, k)), R(w), None, 0, R(M(3, n)), None, 0, None) == INVALID
    assert mt.lib().mt_linear_q4_q8(R(Q(3, k)), R(w), None, 0, R(M(3, n)), None, 0, None) == INVALID


def test_linear_q4_refuses():
    f, g = mt.lib().mt_linear_q4_f32, mt.lib().mt_linear_q4_q8
    assert f(R(M(3, 65)), R(W(4, 64)), None, 0, R(M(3, 4)), None, 0, None) == INVALID
    assert f(R(M(3, 64)), R(W(4, 64)), None, 0, R(M(3, 5)), None, 0, None) == INVALID
    assert f(R(M(3, 64)), R(W(4, 64)), None, 0, R(M(3, 4, cs=0)), None, 0, None) == INVALID
    assert f(R(M(3, 64)), R(W(4, 64)), 0x100, -1, R(M(3, 4)), None, 0, None) == INVALID
    assert g(R(Q(3, 64, rs=10)), R(W(4, 64)), None, 0, R(M(3, 4)), None, 0, None) == INVALID
    many = 1 << 30                    # more tiles than a grid has threads
    assert f(R(M(many, 64)), R(W(4, 64)), None, 0, R(M(many, 4)), None, 0, None) == INVALID
    assert g(R(Q(many, 64)), R(W(4, 64)), None, 0, R(M(many, 4)), None, 0, None) == INVALID
    assert f(R(M(0, 64)), R(W(4, 64)), None, 0, R(M(0, 4)), None, 0, None) == OK
    assert g(R(Q(0, 64)), R(W(4, 64)), None, 0, R(M(0, 4)), None, 0, None) == OK
    assert f(R(M(3, 64)), R(W(0, 64)), None, 0, R(M(3, 0)), None, 0, None) == OK


def test_workspace_queries():
    lib = mt.lib()
    assert lib.mt_linear_q4_workspace(0, 64, 64) == 0
    assert lib.mt_linear_q4_workspace(-1, 64, 64) == 0
    assert lib.mt_linear_backward_q8_workspace_f32(-1, 4, 4) == 0
    # what a call needs it refuses to go without, and the query covers it
    need = lib.mt_linear_q4_workspace(100, 1 << 16, 128)
    if need:
        assert lib.mt_linear_q4_f32(R(M(100, 1 << 16)), R(W(128, 1 << 16)), None, 0, R(M(100, 128)),
                                    0x100, 16, None) == WORKSPACE
    need = lib.mt_linear_backward_q8_workspace_f32(1 << 16, 64, 64)
    assert need > 0
    assert lib.mt_linear_backward_q8_f32(R(M(1 << 16, 64)), R(Q(1 << 16, 64)), None, None, R(M(64, 64)),
                                         0.0, None, 0, 0.0, None, 0, None) == WORKSPACE


def test_linear_backward_q8_refuses():
    def call(dy=M(4, 8), x=Q(4, 16), w=None, dx=None, dw=None, db=None, dbs=1):
        return mt.lib().mt_linear_backward_q8_f32(R(dy), R(x), R(w), R(dx), R(dw), 0.0, db, dbs, 0.0,
                                                  None, 0, None)
    assert call(dy=M(5, 8)) == INVALID
    assert call(dx=M(4, 16)) == INVALID                       # dX without W
    assert call(dx=M(4, 16), w=M(9, 16)) == INVALID
    assert call(dx=M(4, 15), w=M(8, 16)) == INVALID
    assert call(dw=M(8, 15)) == INVALID
    assert call(dw=M(8, 16, cs=0)) == INVALID
    assert call(db=0x100, dbs=0) == INVALID
    assert call(x=Q(4, 16, scale=0)) == INVALID
    assert call() == OK


def test_python_refuses_cpu_tensors():
    x = torch.ones(4, 64)
    rows = mt.Q8Rows(torch.zeros(4, 64, dtype=torch.int8), torch.ones(4))
    wq = mt.Q4Weight(torch.zeros(8, 32, dtype=torch.uint8), torch.ones(8, 1), 64, 128)
    for f in (lambda: mt.quantize_q8(x), lambda: mt.dequantize_q8(rows), lambda: mt.rms_norm(x),
              lambda: mt.rms_norm_backward(x, x, None, torch.ones(4)), lambda: mt.quantize_q4(x),
              lambda: mt.dequantize_q4(wq), lambda: mt.linear_q4(x, wq),
              lambda: mt.linear_q4(rows, wq), lambda: mt.linear_backward_q8(x, rows)):
        with pytest.raises(ValueError):
            f()
