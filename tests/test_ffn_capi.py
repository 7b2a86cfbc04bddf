"""include/mtffn.h and mt_linear_q8 without a GPU: what the entry points refuse before they
touch the device, what they take as nothing to do, and the queries."""
import ctypes

import pytest

import minitensor_amd as mt
from minitensor_amd.ffn import GatePlan
from minitensor_amd.lowbit import Q8Plan, RowsQ8

OK, INVALID, WORKSPACE = mt.MT_OK, mt.MT_ERR_INVALID, mt.MT_ERR_WORKSPACE


def M(rows, cols, rs=None, cs=1, batch=1, bs=0, off=0, base=0x1000):
    return mt.MatF32(base, off, rows, cols, cols if rs is None else rs, cs, batch, bs)


def Q(rows, cols, rs=None, q=0x1000, scale=0x2000):
    return RowsQ8(q, scale, rows, cols, cols if rs is None else rs)


def R(x):
    return ctypes.byref(x) if x is not None else None


def plan_q8(m, k, n, gated=False):
    """(rows and columns of a tile or 0, splits) that linear_q8 (gated_linear of 8-bit rows) takes."""
    p = Q8Plan()
    f = mt.lib().mt_gated_linear_q8_plan if gated else mt.lib().mt_linear_q8_plan
    assert f(m, k, n, R(p)) == OK
    return (p.tile_rows, p.tile_cols), p.splits


def plan_gate(x, w):
    """(kind, (rows and columns of a tile), splits) of gated_linear in fp32."""
    p = GatePlan()
    assert mt.lib().mt_gated_linear_plan_f32(R(x), R(w), R(p)) == OK
    return p.kind, (p.tile_rows, p.tile_cols), p.splits


def test_gate_plans():
    assert plan_gate(M(1, 4096), M(8192, 4096))[0] == 0
    assert plan_gate(M(8, 64), M(64, 64))[0] == 0
    assert plan_gate(M(16, 64), M(32, 64))[0] == 0 and plan_gate(M(16, 65), M(32, 65))[0] == 0
    assert plan_gate(M(9, 5000), M(2200, 5000))[0] == 1 and plan_gate(M(9, 1000), M(2200, 1000))[0] == 0
    assert plan_gate(M(48, 64), M(128, 64))[0] == 0 and plan_gate(M(48, 5000), M(128, 5000))[0] == 1
    assert plan_gate(M(49, 64), M(128, 64)) == (0, (16, 0), 1)
    assert plan_gate(M(512, 1024), M(1024, 1024)) == (0, (32, 0), 1)
    assert plan_gate(M(500, 64), M(2048, 64))[0] == 0 and plan_gate(M(4096, 64), M(2048, 64))[0] == 1
    assert plan_gate(M(8, 64, rs=1, cs=8), M(64, 64))[0] == 1          # x across its rows
    assert plan_gate(M(100, 64), M(64, 64, rs=1, cs=64))[0] == 1
    assert plan_gate(M(100, 64, rs=128, cs=2), M(64, 64))[0] == 2
    assert plan_gate(M(100, 64), M(64, 64, rs=128, cs=2))[0] == 2
    assert plan_gate(M(100, 64), M(64, 64, rs=1 << 25))[0] == 0        # past 32-bit offsets
    assert plan_gate(M(2000, 64), M(2048, 64, rs=1 << 25))[0] == 2
    assert plan_gate(M(100, 0), M(64, 0))[0] == 2
    assert plan_gate(M(4096, 2048), M(8192, 2048)) == (1, (128, 256), 1)
    assert plan_gate(M(64, 2048), M(512, 2048))[2] > 1


def test_plans_of_most_columns():
    """A grid holds fewer than 2^23 workgroups of 512 threads, one for every 4 or 16 features (64
    columns) of few rows at least: past them, tiles."""
    for m in (1, 4):
        assert plan_gate(M(m, 1), M((1 << 26) - 8, 1)) == (0, (0, 0), 1)
        assert plan_gate(M(m, 1), M(1 << 26, 1)) != (0, (0, 0), 1)
        assert plan_gate(M(m, 1), M(1 << 28, 1))[0] == 1
    assert plan_q8(1, 1, (1 << 29) - 64)[0] == (0, 0) and plan_q8(1, 1, 1 << 29)[0] != (0, 0)
    assert plan_q8(1, 1, (1 << 28) - 32, True)[0] == (0, 0) and plan_q8(1, 1, 1 << 28, True)[0] != (0, 0)


def test_linear_q8_refuses():
    def call(x=Q(4, 64), w=Q(8, 64), y=M(4, 8), b=None, bs=0, ws=None, n=0):
        return mt.lib().mt_linear_q8(R(x), R(w), b, bs, R(y), ws, n, None)
    assert call(w=Q(8, 63)) == INVALID
    assert call(y=M(4, 9)) == INVALID
    assert call(y=M(5, 8)) == INVALID
    assert call(y=M(4, 8, cs=0)) == INVALID
    assert call(x=Q(4, 64, q=0)) == INVALID
    assert call(w=Q(8, 64, scale=0)) == INVALID
    assert call(w=Q(8, 64, rs=63)) == INVALID
    assert call(b=0x3000, bs=-1) == INVALID
    assert call(x=None) == INVALID and call(w=None) == INVALID and call(y=None) == INVALID
    assert call(x=Q(1 << 31, 64), y=M(1 << 31, 8)) == INVALID
    assert call(x=Q(0, 64), y=M(0, 8)) == OK
    assert call(w=Q(0, 64), y=M(4, 0)) == OK
    assert plan_q8(65, 65536, 64)[1] > 1
    assert call(x=Q(65, 65536), w=Q(64, 65536), y=M(65, 64)) == WORKSPACE


def test_gated_linear_refuses():
    f32, q8 = mt.lib().mt_gated_linear_f32, mt.lib().mt_gated_linear_q8

    def call(f, x, w, h=M(4, 4), gu=None, act=0, b=None, bs=0, ws=None, n=0):
        return f(R(x), R(w), b, bs, act, R(h), R(gu), ws, n, None)
    for f, X in ((f32, M), (q8, Q)):
        assert call(f, X(4, 64), X(7, 64)) == INVALID
        assert call(f, X(4, 64), X(8, 60)) == INVALID
        assert call(f, X(4, 64), X(8, 64), act=5) == INVALID
        assert call(f, X(4, 64), X(8, 64), act=-1) == INVALID
        assert call(f, X(4, 64), X(8, 64), h=M(4, 8)) == INVALID
        assert call(f, X(4, 64), X(8, 64), h=M(4, 4, rs=0)) == INVALID
        assert call(f, X(4, 64), X(8, 64), gu=M(4, 4)) == INVALID
        assert call(f, X(4, 64), X(8, 64), gu=M(4, 8, cs=0)) == INVALID
        assert call(f, X(4, 64), X(8, 64), b=0x3000, bs=-1) == INVALID
        assert call(f, None, X(8, 64)) == INVALID
        assert call(f, X(0, 64), X(8, 64), h=M(0, 4)) == OK
        assert call(f, X(4, 64), X(0, 64), h=M(4, 0)) == OK


def test_gate_refuses():
    g, b = mt.lib().mt_gate_f32, mt.lib().mt_gate_backward_f32
    assert g(R(M(4, 8)), 0, R(M(4, 5)), None) == INVALID
    assert g(R(M(4, 8)), 9, R(M(4, 4)), None) == INVALID
    assert g(R(M(4, 8)), 0, R(M(4, 4, cs=0)), None) == INVALID
    assert g(R(M(4, 8, base=0)), 0, R(M(4, 4)), None) == INVALID
    assert g(R(M(0, 8)), 0, R(M(0, 4)), None) == OK
    assert b(R(M(4, 4)), R(M(4, 8)), 0, R(M(4, 6)), None) == INVALID
    assert b(R(M(4, 3)), R(M(4, 8)), 0, R(M(4, 8)), None) == INVALID
    assert b(R(M(4, 4)), R(M(4, 8)), 0, R(M(4, 8, rs=0)), None) == INVALID
    assert b(R(M(4, 0)), R(M(4, 0)), 0, R(M(4, 0)), None) == OK


def test_gate_backward_bias_refuses():
    def b(dh=M(4, 4), gu=M(4, 8), act=0, dgu=M(4, 8), db=0x5000, stride=1, ws=None, n=0):
        return mt.lib().mt_gate_backward_bias_f32(R(dh), R(gu), act, R(dgu), db, stride, 0.0, ws, n, None)
    assert b(gu=M(4, 7)) == INVALID and b(gu=M(3, 8)) == INVALID and b(dgu=M(4, 9)) == INVALID
    assert b(act=5) == INVALID and b(act=-1) == INVALID
    assert b(dgu=M(4, 8, rs=0)) == INVALID and b(dgu=None) == INVALID
    assert b(db=None) == INVALID and b(stride=0) == INVALID and b(stride=-1) == INVALID
    assert b(ws=0x10002, n=64) == INVALID
    assert b(M(4, 0), M(4, 0), 0, M(4, 0), None, 0) == OK
    big = dict(dh=M(1000, 400), gu=M(1000, 800), dgu=M(1000, 800))
    need = mt.lib().mt_gate_backward_bias_workspace_f32(1000, 400)
    assert need >= 800 * 4 and b(**big) == WORKSPACE and b(**big, ws=0x10000, n=need - 4) == WORKSPACE
    f = mt.lib().mt_gate_backward_bias_workspace_f32
    assert f(0, 8) == 0 and f(8, 0) == 0 and f(-1, 8) == 0 and f(16, 1 << 29) == 0 and f(4, 1 << 31) == 0


def test_clip_refuses():
    def call(g, o=None, n=None, most=1.0, eps=1e-6, norm=0x9000, ws=0x10000, size=1 << 30, alone=False):
        a = (mt.MatF32 * max(len(g), 1))(*g)
        b = (mt.MatF32 * max(len(o), 1))(*o) if o is not None else None
        n = len(g) if n is None else n
        if alone:
            return mt.lib().mt_grad_norm_f32(a, n, norm, ws, size, None)
        return mt.lib().mt_clip_grad_norm_f32(a, b, n, most, eps, norm, ws, size, None)
    x = M(4, 8)
    assert call([x], n=-1) == INVALID
    assert call([x], n=(1 << 20) + 1) == INVALID
    assert call([x], norm=None) == INVALID
    assert call([x], most=-1.0) == INVALID
    assert call([x], most=float("nan")) == INVALID
    assert call([x], eps=-1.0) == INVALID
    assert call([x, x]) == INVALID                                   # scaled twice
    assert call([x, M(4, 8, base=0x8000)], [M(4, 8), M(4, 8)]) == INVALID
    assert call([x], [M(4, 9)]) == INVALID
    assert call([M(4, 8, rs=0)]) == INVALID                          # rows on one address
    assert call([M(4, 8, base=0)]) == INVALID
    assert call([M(4, 8, rs=-8)]) == INVALID
    assert call([M(1 << 40, 1 << 40)], alone=True) == INVALID
    assert call([x], ws=None) == WORKSPACE
    assert call([x], size=8) == WORKSPACE
    assert call([x], ws=0x10004) == WORKSPACE                        # not a multiple of 8
    assert call([x], ws=None, alone=True) == WORKSPACE


def test_clip_refuses_overlaps():
    """Outputs over each other or over other tensors: what is scaled would be scaled twice, or
    read when it is."""
    def call(g, o=None):
        a = (mt.MatF32 * len(g))(*g)
        b = (mt.MatF32 * len(o))(*o) if o is not None else None
        # (no workspace: what is not refused goes no further)
        return mt.lib().mt_clip_grad_norm_f32(a, b, len(g), 1.0, 1e-6, 0x9000, None, 0, None)
    at = lambda e, n=32, **k: M(1, n, base=0x10000 + 4 * e, **k)
    fine = WORKSPACE
    assert call([at(0), at(32), at(100)]) == fine
    assert call([at(0), at(31)]) == INVALID
    assert call([at(100, 8), at(0, 200)]) == INVALID                 # one within another
    assert call([at(0, 200), at(50, 0), at(200)]) == fine
    assert call([at(0), at(32)], [at(100), at(131)]) == INVALID
    assert call([at(0), at(32)], [at(32), at(100)]) == INVALID       # over the next one's input
    assert call([at(0), at(32)], [at(32), at(0)]) == INVALID
    assert call([at(0)], [at(4)]) == INVALID
    assert call([at(0), at(0)], [at(100), at(200)]) == fine          # one input, two outputs
    assert call([at(0), at(0)], [at(0), at(200)]) == INVALID
    assert call([at(0), at(32)], [at(0), at(100)]) == fine
    # two views that lie between each other's elements; one over a dense tensor
    odd = [M(4, 8, rs=32, cs=2, base=0x10000 + 4 * e) for e in (0, 1)]
    assert call(odd) == fine
    assert call([odd[0], at(0, 100)]) == INVALID
    # a matrix over itself, transposed
    assert call([M(8, 8, base=0x10000)], [M(8, 8, rs=1, cs=8, base=0x10000)]) == INVALID
    assert call([M(8, 8, rs=1, cs=8, base=0x10000)], [M(8, 8, rs=1, cs=8, base=0x10000)]) == fine


def test_queries():
    lib = mt.lib()
    f = lib.mt_gated_linear_workspace_f32
    assert f(R(M(0, 8)), R(M(8, 8))) == 0 and f(R(M(8, 8)), R(M(0, 8))) == 0
    assert f(R(M(8, 8)), R(M(8, 9))) == 0 and f(None, R(M(8, 8))) == 0
    # neither way contiguous: the projections go to the workspace
    assert f(R(M(100, 64, rs=256, cs=2)), R(M(512, 64))) >= 100 * 512 * 4
    assert f(R(M(8, 64)), R(M(512, 64))) == 0
    for f in (lib.mt_linear_q8_workspace, lib.mt_gated_linear_q8_workspace):
        assert f(R(Q(0, 8)), R(Q(8, 8))) == 0 and f(R(Q(8, 8)), R(Q(0, 8))) == 0
        assert f(R(Q(8, 8)), R(Q(8, 9))) == 0 and f(None, R(Q(8, 8))) == 0
        # rows that lie as the tiles take them need none, others a copy
        assert f(R(Q(3000, 64)), R(Q(2960, 64))) == 0
        assert 3000 * 64 <= f(R(Q(3000, 63)), R(Q(2960, 63, rs=64))) < 3000 * 128 + 32
        assert 5960 * 64 <= f(R(Q(3000, 64, q=0x1008)), R(Q(2960, 64, rs=72))) < 5960 * 128 + 32
        assert 2960 * 64 <= f(R(Q(3000, 64)), R(Q(2960, 64, rs=1 << 24))) < 2960 * 128 + 32
        assert f(R(Q(64, 63)), R(Q(96, 63))) == 0
    assert lib.mt_grad_norm_workspace_f32(-1) == 0
    assert 0 < lib.mt_grad_norm_workspace_f32(1) <= lib.mt_grad_norm_workspace_f32(1000)
    p = Q8Plan()
    assert lib.mt_linear_q8_plan(4, 8, 8, None) == INVALID
    assert lib.mt_linear_q8_plan(0, 8, 8, R(p)) == INVALID


@pytest.mark.parametrize("gated", [False, True])
def test_q8_plans(gated):
    """Few rows on their kernel, up to the inputs that its sums hold; a split never holds more
    terms than 32 bits do; workspaces of whole tiles."""
    assert plan_q8(1, 4096, 4096, gated)[0] == (0, 0)
    assert plan_q8(2048, 4096, 8192, gated)[0] == (256, 256)
    for m in (1, 70, 300):
        for k in (1, 131071, 200000, 1 << 20, 1 << 27):
            tile, splits = plan_q8(m, k, 100, gated)
            assert tile == (0, 0) and (k < 1 << 19 or k > 1 << 24) or splits * ((1 << 17) - 128) >= k
            f = mt.lib().mt_gated_linear_q8_workspace if gated else mt.lib().mt_linear_q8_workspace
            ws = f(R(Q(m, k, rs=(k + 15) // 16 * 16)), R(Q(200 if gated else 100, k, rs=(k + 15) // 16 * 16)))
            assert (ws > 0) == (splits > 1)
            if splits > 1:
                assert ws >= 4 * splits * m * 100 * (1 + gated)
