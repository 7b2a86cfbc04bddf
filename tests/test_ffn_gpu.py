"""The operators of include/mtffn.h, and mt_linear_q8, against 64 bits, at the sizes,
strides, alignments and values where they can go wrong.  The bounds (tests/ffn_reference.py)
count roundings."""
import math

import numpy as np
import pytest
import torch

import ffn_reference as ref
import minitensor_amd as mt

pytestmark = pytest.mark.gpu

H = ref.H


def rng(*key):
    return np.random.default_rng([int(k) for k in key])


def gpu(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def cpu(t):
    return t.detach().cpu().numpy()


def normal(g, *shape):
    return g.standard_normal(shape).astype(np.float32)


def strided(a, dev, how):
    t = gpu(a, dev)
    if how == "dense":
        return t
    if how == "transposed":
        return t.t().contiguous().t()
    wide = torch.full((a.shape[0], 2 * a.shape[1] + 7), 7.0, device=dev)
    v = wide[:, 1:1 + 2 * a.shape[1]:2] if how == "gaps" else wide[:, 3:3 + a.shape[1]]
    v.copy_(t)
    return v


STRIDES = ["dense", "transposed", "gaps", "offset"]


def check(got, want, bound, what=""):
    got = np.asarray(cpu(got), np.float64)
    # (a value past fp32's range, 2^128 - 2^103 and more, rounds to an infinity)
    past = (np.abs(want) >= 2.0 ** 128 - 2.0 ** 103) & (got == np.copysign(np.inf, want))
    over = np.where(past, -1.0, np.abs(np.where(past, 0.0, got) - want) - bound)
    worst = np.unravel_index(np.argmax(over), over.shape) if over.size else None
    assert not over.size or over[worst] <= 0, (
        f"{what}: off by {abs(got - want)[worst]:.3e} at {worst}, bound {bound[worst]:.3e}, "
        f"got {got[worst]:.9e}, want {want[worst]:.9e}")


def rows8(g, r, k, dev, how="dense"):
    """Random codes, -128 among them, and scales; (q, s) and the tensors."""
    q = g.integers(-128, 128, (r, k)).astype(np.int8)
    s = (g.random(r) + 0.1).astype(np.float32) / 64
    if how == "dense":
        return q, s, mt.Q8Rows(gpu(q, dev), gpu(s, dev))
    pad = {"odd": 5, "by 16": 16 - k % 16 + 16, "offset": 24}[how]
    wide = torch.full((r, k + pad), 99, dtype=torch.int8, device=dev)
    v = wide[:, 3:3 + k] if how == "offset" else wide[:, :k]
    v.copy_(gpu(q, dev))
    return q, s, mt.Q8Rows(v, gpu(s, dev))


# ---- 8-bit Linear --------------------------------------------------------------
# rows around the kernels' choices (few rows, tiles of 64, 128 and 256), columns and inputs
# around their blocks
Q8_SIZES = [(1, 1, 1), (1, 64, 16), (2, 17, 33), (1, 100, 256), (3, 255, 257), (16, 1000, 2048),
            (17, 48, 63), (31, 129, 500), (32, 32, 4096), (33, 65, 127), (33, 1, 1000), (40, 200, 64),
            (64, 128, 128), (65, 129, 129), (17, 16400, 100), (32, 8200, 65),
            (64, 8200, 64), (70, 8200, 96), (100, 257, 300), (128, 256, 512), (257, 511, 255),
            (255, 40, 8192), (300, 1000, 1024), (513, 769, 640), (1027, 520, 2047), (1000, 1500, 257),
            (2100, 1030, 333), (150, 700, 9001), (300, 520, 12001), (1100, 1500, 64), (700, 900, 5008)]


@pytest.mark.parametrize("m,n,k", Q8_SIZES)
def test_linear_q8(dev, m, n, k):
    g = rng(1, m, n, k)
    b = normal(g, n)
    for how in ("dense", "odd", "by 16", "offset"):
        q, s, x = rows8(g, m, k, dev, how)
        w, ws, wt = rows8(g, n, k, dev, how)
        want, bound = ref.linear_q8(q, s, w, ws)
        check(mt.linear_q8(x, wt), want, bound, how)
        want, bound = ref.linear_q8(q, s, w, ws, b)
        y = torch.full((m, 2 * n + 1), -5.0, device=dev)
        mt.linear_q8(x, wt, gpu(np.repeat(b, 2), dev)[::2], out=y[:, 1::2])
        check(y[:, 1::2], want, bound, how + " strided out")
        assert bool((y[:, ::2] == -5).all())


# ... and outputs large enough for the larger tiles
Q8_LARGE = [(1000, 4000, 1100), (1900, 4000, 200), (2000, 8190, 300), (2048, 8192, 256),
            (1000, 4000, 1104), (2000, 8190, 336)]


def test_linear_q8_kernels():
    """Which sizes take which kernel, so that the tests here reach all of them."""
    from test_ffn_capi import plan_q8
    plans = [plan_q8(m, k, n) for m, n, k in Q8_SIZES + Q8_LARGE]
    tiles = {(0, 0), (64, 128), (128, 128), (128, 256), (256, 256)}
    assert {p[0] for p in plans} == tiles, plans
    assert any(p[1] > 1 for p in plans)


@pytest.mark.parametrize("m,n,k", Q8_LARGE)
def test_linear_q8_large_tiles(dev, m, n, k):
    g = rng(2, m, n, k)
    for how in ("dense", "offset"):
        q, s, x = rows8(g, m, k, dev, how)
        w, ws, wt = rows8(g, n, k, dev, how)
        check(mt.linear_q8(x, wt), *ref.linear_q8(q, s, w, ws), how)
        gu, e = ref.linear_q8(q, s / 16, w, ws)
        x = mt.Q8Rows(x.q, gpu(s / 16, dev))
        if n % 2 == 0:
            check(mt.gated_linear(x, wt, act="silu").h, *ref.gate("silu", gu, e), how)


@pytest.mark.parametrize("m,n,k", [(70, 200, 33), (100, 300, 16), (513, 769, 650), (1000, 2000, 255), (2000, 8190, 300)])
def test_linear_q8_one_operand_in_place(dev, m, n, k):
    """Rows that the tiles read in place beside rows that are copied first, to the inputs that
    there are, and both copied, to whole chunks."""
    g = rng(18, m, n, k)
    for a, b in (("by 16", "odd"), ("offset", "by 16"), ("odd", "offset"), ("by 16", "by 16")):
        q, s, x = rows8(g, m, k, dev, a)
        w, ws, wt = rows8(g, n, k, dev, b)
        check(mt.linear_q8(x, wt), *ref.linear_q8(q, s, w, ws), a + ", " + b)


@pytest.mark.parametrize("m", [1, 20, 40, 70])
@pytest.mark.parametrize("k", [131071, 131073, 300001, 600000])
def test_linear_q8_sums_past_32_bits(dev, m, k):
    """Every product 2^14: sums beyond 2^31 from 131072 inputs on."""
    q = torch.full((m, k), -128, dtype=torch.int8, device=dev)
    w = torch.full((5, k), -128, dtype=torch.int8, device=dev)
    w[1] = 127
    one = torch.ones(m, device=dev)
    y = cpu(mt.linear_q8(mt.Q8Rows(q, one), mt.Q8Rows(w, torch.ones(5, device=dev))))
    want = np.array([k * 16384, k * -128 * 127] + [k * 16384] * 3, np.float64)
    assert np.array_equal(y, np.broadcast_to(want.astype(np.float32), (m, 5)))


def test_most_columns(dev):
    """One row by more columns than a grid of few rows holds: the tiles."""
    n = (1 << 27) + 40
    q = torch.randint(-127, 128, (n,), dtype=torch.int8, device=dev)
    s = torch.rand(n, device=dev)
    x = mt.Q8Rows(torch.tensor([[-3]], dtype=torch.int8, device=dev), torch.tensor([0.5], device=dev))
    w = mt.Q8Rows(q[:, None], s)
    # (0.5·s and the sum are exact: one rounding)
    want = (-3.0 * q.double() * (0.5 * s.double())).float()
    assert torch.equal(mt.linear_q8(x, w)[0], want)
    del want, w, q, s
    f = (1 << 25) + 9
    w = torch.randn(2 * f, 1, device=dev)
    r = mt.gated_linear(torch.tensor([[2.0]], device=dev), w, act="relu", keep=True)
    assert torch.equal(r.gu[0], 2 * w[:, 0])
    assert torch.equal(r.h[0], (2 * w[:f, 0]).clamp(min=0) * (2 * w[f:, 0]))


def test_linear_q8_long_rows(dev):
    """Rows of 2^24 inputs and more, and rows that far apart: neither goes to the tiles as it is."""
    k = (1 << 24) + 77
    q = torch.full((70, k), -128, dtype=torch.int8, device=dev)
    w = torch.full((3, k), 127, dtype=torch.int8, device=dev)
    q[33, -1] = 5
    y = cpu(mt.linear_q8(mt.Q8Rows(q, torch.ones(70, device=dev)), mt.Q8Rows(w, torch.ones(3, device=dev))))
    want = np.full((70, 3), -128.0 * 127 * k)
    want[33] += 127 * 133
    assert np.array_equal(y, want.astype(np.float32))
    g = rng(31)
    codes, s = g.integers(-128, 128, (70, 100)).astype(np.int8), g.random(70).astype(np.float32)
    far = q.flatten()[:70 * (1 << 24)].view(70, 1 << 24)[:, :100]
    far.copy_(gpu(codes, dev))
    wq, ws, wt = rows8(g, 64, 100, dev)
    check(mt.linear_q8(mt.Q8Rows(far, gpu(s, dev)), wt), *ref.linear_q8(codes, s, wq, ws))
    gu, e = ref.linear_q8(codes, s / 256, wq, ws)
    check(mt.gated_linear(mt.Q8Rows(far, gpu(s / 256, dev)), wt).h, *ref.gate("silu", gu, e))


def test_linear_q8_same_for_any_tile(dev):
    """A row's result does not depend on the rows beside it (nor so on tiles and splits)."""
    g = rng(3)
    _, _, x = rows8(g, 700, 1111, dev)
    _, _, w = rows8(g, 333, 1111, dev)
    b = gpu(normal(g, 333), dev)
    all_ = mt.linear_q8(x, w, b)
    for n in (1, 5, 32, 33, 64, 65, 130, 400):
        part = mt.linear_q8(mt.Q8Rows(x.q[:n], x.scale[:n]), w, b)
        assert torch.equal(part, all_[:n]), n


def test_linear_q8_scales_that_are_no_numbers(dev):
    g = rng(4)
    x = normal(g, 40, 100)
    x[3, 7] = np.inf
    x[4, 2] = np.nan
    w = normal(g, 30, 100)
    w[9, 5] = np.nan
    y = cpu(mt.linear_q8(mt.quantize_q8(gpu(x, dev)), mt.quantize_q8(gpu(w, dev))))
    bad = np.zeros_like(y, bool)
    bad[3:5] = True
    bad[:, 9] = True
    assert np.array_equal(np.isnan(y) | np.isinf(y), bad)
    assert np.isnan(y[4]).all() and np.isnan(y[:, 9]).all()


def test_linear_q8_empty(dev):
    e = mt.Q8Rows(torch.empty(0, 8, dtype=torch.int8, device=dev), torch.empty(0, device=dev))
    w = mt.quantize_q8(torch.ones(5, 8, device=dev))
    assert mt.linear_q8(e, w).shape == (0, 5)
    assert mt.linear_q8(w, e).shape == (5, 0)
    none = mt.quantize_q8(torch.empty(3, 0, device=dev))
    wn = mt.quantize_q8(torch.empty(40, 0, device=dev))
    b = torch.arange(40.0, device=dev)
    assert torch.equal(mt.linear_q8(none, wn, b), b.expand(3, 40))
    big = mt.quantize_q8(torch.empty(70, 0, device=dev))
    assert bool((mt.linear_q8(big, wn) == 0).all())


# ---- gate and its gradient ------------------------------------------------------
def hard_gates(g, r, f):
    """Projections with values where an activation can go wrong."""
    gu = normal(g, r, 2 * f) * 3
    flat = gu[:, :f].reshape(-1)
    hard = np.array([0, -0.0, 1e-30, -1e-30, 1e-3, -1e-3, 5, -5, 9, -9, 20, -20, 60, -60, 88, -88, 90,
                     -90, 103, -103, 120, -120, 1e4, -1e4, 1e18, -1e18, 3e38, -3e38], np.float32)
    flat[:len(hard)] = hard[:len(flat)]
    gu[:, :f] = flat.reshape(r, f)
    return gu


@pytest.mark.parametrize("act", ref.ACTS)
@pytest.mark.parametrize("how", STRIDES)
def test_gate_and_backward(dev, act, how):
    for r, f in ((1, 1), (3, 5), (7, 64), (37, 130), (64, 1023)):
        g = rng(5, r, f)
        gu, dh = hard_gates(g, r, f), normal(g, r, f)
        t, d = strided(gu, dev, how), strided(dh, dev, how)
        check(mt.gate(t, act), *ref.gate(act, gu), f"{act} {r}x{f}")
        out = strided(np.full((r, 2 * f), 3, np.float32), dev, how)
        got = mt.gate_backward(d, t, act, out=out)
        assert got is out
        want, bound = ref.gate_backward(act, dh, gu)
        check(got, want, bound, f"{act} {r}x{f} backward")
        check(mt.gate_backward(d, t, act, out=t), want, bound, "in place")


def test_gate_backward_is_the_derivative():
    """The 64-bit formulas against differences."""
    a = np.linspace(-6, 6, 241) + 1e-3
    for act in ref.ACTS:
        e = 1e-5
        diff = (ref.act(act, a + e)[0] - ref.act(act, a - e)[0]) / (2 * e)
        # third derivatives below 4: e^2/6 of them, and 64-bit rounding over e
        assert np.abs(diff - ref.act(act, a)[1]).max() < 4 * e * e + 2e-16 * 8 / e


def test_gate_infinities(dev):
    inf, nan = float("inf"), float("nan")
    gu = torch.tensor([[inf, nan, 1.0, 1.0, 0.0, 2.0, 3.0, inf]], device=dev)
    for act in ("silu", "gelu", "gelu_tanh", "relu"):
        h = mt.gate(gu, act)
        assert math.isnan(h[0, 1]) and h[0, 3] == inf
    d = mt.gate_backward(torch.ones(1, 4, device=dev), gu, "silu")
    assert not torch.isnan(d[0, 2]) and torch.isnan(d[0, 1])


# ---- gated Linear ----------------------------------------------------------------
GATE_SIZES = [(1, 1, 1), (1, 64, 16), (2, 33, 17), (4, 100, 256), (5, 31, 257), (8, 512, 1024),
              (3, 9, 513), (9, 65, 100), (16, 256, 2048), (17, 40, 63), (32, 100, 515), (33, 64, 130),
              (6, 40, 90), (8, 1030, 2061), (7, 1100, 70), (13, 70, 515), (16, 33, 1029), (10, 129, 200),
              (16, 1040, 300), (48, 77, 64), (49, 64, 130), (64, 128, 512), (100, 257, 300),
              (130, 96, 1000), (257, 200, 64), (300, 515, 333), (509, 320, 1285),
              (70, 41, 4003), (131, 97, 3001), (513, 301, 1501), (600, 70, 130), (470, 470, 70), (97, 700, 1100)]


@pytest.mark.parametrize("m,f,k", GATE_SIZES)
def test_gated_linear(dev, m, f, k):
    g = rng(6, m, f, k)
    x, w, b = normal(g, m, k), normal(g, 2 * f, k) / np.float32(k ** 0.5), normal(g, 2 * f)
    for how_x, how_w, act, bias in (("dense", "dense", "silu", None), ("offset", "offset", "gelu", b),
                                    ("transposed", "dense", "gelu_tanh", b),
                                    ("dense", "transposed", "silu", b), ("gaps", "gaps", "relu", None),
                                    ("transposed", "transposed", "sigmoid", b)):
        t = (strided(x, dev, how_x), strided(w, dev, how_w), gpu(b, dev) if bias is not None else None)
        gu, e = ref.linear(x, w, bias)
        want, bound = ref.gate(act, gu, e)
        what = f"{how_x} {how_w} {act}"
        r = mt.gated_linear(*t, act=act)
        assert r.gu is None
        check(r.h, want, bound, what)
        kept = mt.gated_linear(*t, act=act, keep=True)
        check(kept.h, want, bound, what + " kept")
        check(kept.gu, gu, e, what + " projections")
        # h is that of the kept projections, to the activation's last rounding
        check(kept.h, *ref.gate(act, cpu(kept.gu)), what + " of its projections")
        out = strided(np.full((m, f), 5, np.float32), dev, how_x)
        assert mt.gated_linear(*t, act=act, out=out).h is out
        assert torch.equal(out, r.h), what


GATE_LARGE = [(2048, 640, 100), (1024, 2048, 128), (700, 3001, 200), (2048, 2000, 250), (1024, 4096, 130),
              (500, 2570, 700)]


def test_gated_linear_kernels():
    """Which sizes take which kernel, so that the tests here reach all of them."""
    from test_ffn_capi import M, plan_gate
    plans = [plan_gate(M(m, k), M(2 * f, k)) for m, f, k in GATE_SIZES + GATE_LARGE]
    assert {p[0] for p in plans} == {0, 1}
    assert {p[1] for p in plans} == {(0, 0), (16, 0), (32, 0), (48, 0), (64, 128), (128, 128), (128, 256)}, plans
    assert any(p[2] > 1 for p in plans)


@pytest.mark.parametrize("m,f,k", GATE_LARGE)
def test_gated_linear_large_tiles(dev, m, f, k):
    g = rng(7, m, f, k)
    x, w, b = normal(g, m, k), normal(g, 2 * f, k) / np.float32(k ** 0.5), normal(g, 2 * f)
    gu, e = ref.linear(x, w, b)
    r = mt.gated_linear(gpu(x, dev), gpu(w, dev), gpu(b, dev), keep=True)
    check(r.gu, gu, e)
    check(r.h, *ref.gate("silu", gu, e))


@pytest.mark.parametrize("m,n,k", Q8_SIZES)
def test_gated_linear_q8(dev, m, n, k):
    g = rng(8, m, n, k)
    b = normal(g, 2 * n)
    for how, act, bias in (("dense", "silu", None), ("odd", "gelu", b), ("by 16", "relu", b),
                           ("offset", "gelu_tanh", None)):
        q, s, x = rows8(g, m, k, dev, how)
        w, ws, wt = rows8(g, 2 * n, k, dev, how)
        s, ws = s / np.float32(k ** 0.5), ws / np.float32(16)
        x, wt = mt.Q8Rows(x.q, gpu(s, dev)), mt.Q8Rows(wt.q, gpu(ws, dev))
        gu, e = ref.linear_q8(q, s, w, ws, bias)
        want, bound = ref.gate(act, gu, e)
        tb = gpu(b, dev) if bias is not None else None
        r = mt.gated_linear(x, wt, tb, act=act, keep=True)
        check(r.gu, gu, e, how)
        check(r.h, want, bound, how)
        out = torch.full((m, 2 * n), -5.0, device=dev)
        mt.gated_linear(x, wt, tb, act=act, out=out[:, ::2])
        assert torch.equal(out[:, ::2], r.h) and bool((out[:, 1::2] == -5).all())


def test_gated_linear_infinities(dev):
    """An infinity among fp32 operands gives what the formula gives, in its row and columns alone."""
    g = rng(9)
    for m in (3, 70, 200):
        x, w = normal(g, m, 96), normal(g, 140, 96) / 10
        x[2, 5], w[7, 11], w[80, 3] = np.inf, np.inf, np.nan
        r = mt.gated_linear(gpu(x, dev), gpu(w, dev), act="relu", keep=True)
        bad = np.zeros((m, 140), bool)
        bad[2], bad[:, 7], bad[:, 80] = True, True, True
        gu = cpu(r.gu)
        assert np.array_equal(~np.isfinite(gu), bad)
        assert np.isnan(gu[:, 80]).all()
        fine = ~(bad[:, :70] | bad[:, 70:])
        assert np.isfinite(cpu(r.h)[fine]).all()


@pytest.mark.parametrize("q8", [False, True])
def test_gated_linear_empty(dev, q8):
    rows = mt.quantize_q8 if q8 else (lambda t: t)
    e = rows(torch.empty(0, 8, device=dev))
    assert mt.gated_linear(e, rows(torch.ones(6, 8, device=dev))).h.shape == (0, 3)
    assert mt.gated_linear(rows(torch.ones(6, 8, device=dev)), e, keep=True).h.shape == (6, 0)
    b = torch.arange(80.0, device=dev) - 20
    for m in (3, 70):
        none, wn = rows(torch.empty(m, 0, device=dev)), rows(torch.empty(80, 0, device=dev))
        r = mt.gated_linear(none, wn, b, act="relu", keep=True)
        assert torch.equal(r.gu, b.expand(m, 80))
        assert torch.equal(r.h, (b[:40].clamp_min(0) * b[40:]).expand(m, 40))
        assert bool((mt.gated_linear(none, wn).h == 0).all())


# ---- gradients --------------------------------------------------------------------
@pytest.mark.parametrize("m,f,k", [(1, 1, 1), (3, 33, 17), (64, 128, 96), (130, 67, 257), (509, 320, 300),
                                   (601, 899, 40)])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gated_linear_backward(dev, m, f, k, act):
    g = rng(10, m, f, k)
    x, w, b = normal(g, m, k), normal(g, 2 * f, k) / np.float32(k ** 0.5), normal(g, 2 * f)
    dh = normal(g, m, f)
    X, W, B, D = (gpu(t, dev) for t in (x, w, b, dh))
    r = mt.gated_linear(X, W, B, act=act, keep=True)
    dx, dw, db = mt.gated_linear_backward(D, r.gu, X, W, act=act)
    # the gradients of the kept projections, and the products of those
    d, e = ref.gate_backward(act, dh, cpu(r.gu))
    a = np.abs(d) + e
    sums = lambda n: (6 * -(-n // 16) + 600) * 2.0 ** -23                 # (as ref.linear, up to 512 splits)
    check(dx, d @ w, e @ np.abs(w) + sums(2 * f) * (a @ np.abs(w)), "dx")
    check(dw, d.T @ x, e.T @ np.abs(x) + sums(m) * (a.T @ np.abs(x)), "dw")
    check(db, d.sum(0), e.sum(0) + (m + 600) * 2.0 ** -23 * a.sum(0), "db")
    # added to gradients that are there, over the projections
    dw0, db0 = gpu(normal(g, 2 * f, k), dev), gpu(normal(g, 2 * f), dev)
    dw1, db1 = dw0.clone(), db0.clone()
    dx2, dw2, db2 = mt.gated_linear_backward(D, r.gu, X, W, act=act, dgu=r.gu, dw=dw1, db=db1,
                                             beta_w=0.5, beta_b=2.0)
    assert dw2 is dw1 and db2 is db1 and torch.equal(dx2, dx)
    check(dw2, 0.5 * cpu(dw0) + cpu(dw).astype(np.float64), 4 * H * (np.abs(cpu(dw)) + np.abs(cpu(dw0))) +
          2 * sums(m) * (a.T @ np.abs(x)))
    check(db2, 2.0 * cpu(db0) + cpu(db).astype(np.float64), 4 * H * (np.abs(cpu(db)) + 2 * np.abs(cpu(db0))) +
          2 * (m + 600) * 2.0 ** -23 * a.sum(0))
    check(r.gu, d, e, "over the projections")
    again = mt.gated_linear(X, W, B, act=act, keep=True)
    n, dw3, n2 = mt.gated_linear_backward(D, again.gu, X, act=act, need_db=False)
    assert n is None and n2 is None
    check(dw3, d.T @ x, e.T @ np.abs(x) + sums(m) * (a.T @ np.abs(x)), "dw alone")


@pytest.mark.parametrize("m,f", [(1, 1), (3, 33), (16, 300), (17, 256), (40, 257), (1000, 70), (2048, 1030), (5, 70001)])
def test_gate_backward_with_sums(dev, m, f):
    """The gradients of gate_backward, and their sums over the rows, over and beside what is there."""
    import ctypes
    g = rng(19, m, f)
    R = lambda t: ctypes.byref(mt.mat(t))
    ws = torch.empty(mt.lib().mt_gate_backward_bias_workspace_f32(m, f), dtype=torch.uint8, device=dev)
    for how, act in zip(STRIDES, (0, 1, 2, 4)):
        dh, gu = strided(normal(g, m, f), dev, how), strided(normal(g, m, 2 * f), dev, how)
        want = mt.gate_backward(dh, gu, ref.ACTS[act])
        for beta in (0.0, 0.5):
            was = normal(g, 4 * f)
            if beta == 0:
                was[:] = np.nan
            db = gpu(was, dev)[::2]
            dgu = torch.empty(m, 2 * f, device=dev) if beta == 0 else gu
            rc = mt.lib().mt_gate_backward_bias_f32(R(dh), R(gu), act, R(dgu), db.data_ptr(), db.stride(0), beta,
                                                    ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
            assert rc == mt.MT_OK and torch.equal(dgu, want)
            d = cpu(want).astype(np.float64)
            old = beta * was[::2].astype(np.float64) if beta else 0.0
            # fewer than m + 8 additions, a rounding each of a part of sum|d|, and the last one's
            check(db, old + d.sum(0), ((m + 8) * np.abs(d).sum(0) + np.abs(old + d.sum(0))) * 2.0 ** -24, how)


def test_gate_backward_sums_of_no_rows(dev):
    import ctypes
    R = lambda t: ctypes.byref(mt.mat(t))
    dh, gu, db = torch.empty(0, 3, device=dev), torch.empty(0, 6, device=dev), torch.full((6,), 2.0, device=dev)
    for beta, want in ((0.25, 0.5), (0.0, 0.0)):
        assert mt.lib().mt_gate_backward_bias_f32(R(dh), R(gu), 0, R(gu), db.data_ptr(), 1, beta, None, 0,
                                                  torch.cuda.current_stream().cuda_stream) == mt.MT_OK
        assert bool((db == want).all())


@pytest.mark.parametrize("m,f,k", [(20, 30, 40), (601, 899, 40)])
def test_backward_by_either_way(dev, m, f, k, monkeypatch):
    """The native call, and the Python one that takes what is not plain: the same."""
    import minitensor_amd.ffn as ffn
    g = rng(20, m, f, k)
    dh, gu, x, w = (gpu(normal(g, *s), dev) for s in ((m, f), (m, 2 * f), (m, k), (2 * f, k)))
    calls = [lambda: mt.gated_linear_backward(dh, gu, x, w),
             lambda: mt.gated_linear_backward(dh, gu, x, need_dw=False),
             lambda: mt.gated_linear_backward(dh, gu, x, w, need_db=False, dgu=torch.empty_like(gu)),
             lambda: mt.gated_linear_backward(dh, gu.clone(), x, w, dw=w.clone(), beta_w=0.5,
                                              db=torch.ones(2 * f, device=dev), beta_b=2.0),
             lambda: mt.gated_linear_backward(dh, gu, mt.quantize_q8(x), w)]
    want = [call() for call in calls]

    class Native:
        def __getattr__(self, name):
            return (lambda *a: None) if name == "gated_linear_backward" else getattr(mt.native(), name)
    monkeypatch.setattr(ffn, "native", lambda: Native())
    for i, (call, a) in enumerate(zip(calls, want)):
        for p, q in zip(call(), a):
            assert (p is None and q is None) or torch.equal(p, q), i


def test_gated_linear_backward_q8_rows(dev):
    g = rng(11)
    x, w, dh = normal(g, 100, 96), normal(g, 140, 96) / 10, normal(g, 100, 70)
    X, W, D = (gpu(t, dev) for t in (x, w, dh))
    r = mt.gated_linear(X, W, keep=True)
    xq = mt.quantize_q8(X)
    dx, dw, db = mt.gated_linear_backward(D, r.gu, xq, W)
    dgu = mt.gate_backward(D, r.gu)
    for a, b in zip((dx, dw, db), mt.linear_backward_q8(dgu, xq, W)):
        assert torch.equal(a, b)


def test_gated_linear_backward_against_differences(dev):
    """A directional derivative of L = sum(h·c) by central differences of the forward pass."""
    g = rng(12)
    m, f, k = 40, 48, 64
    t = [normal(g, m, k), normal(g, 2 * f, k) / 8, normal(g, 2 * f)]
    c = normal(g, m, f)
    step = [normal(g, *a.shape) for a in t]
    e = 2.0 ** -9

    def loss(sign):
        T = [gpu(a + np.float32(sign * e) * s, dev) for a, s in zip(t, step)]
        return float(np.sum(cpu(mt.gated_linear(*T).h).astype(np.float64) * c))
    T = [gpu(a, dev) for a in t]
    r = mt.gated_linear(*T, keep=True)
    grads = mt.gated_linear_backward(gpu(c, dev), r.gu, T[0], T[1])
    want = sum(float(np.sum(cpu(a).astype(np.float64) * s)) for a, s in zip(grads, step))
    got = (loss(1) - loss(-1)) / (2 * e)
    # third derivatives of the sum's 1920 terms: products of four of the steps' projections
    # (each of order 10), so e^2/6 · 1920 · 1e3 with signs that half cancel; rounding of h
    # 1e-6 a term over 2e
    assert abs(got - want) < e * e / 6 * 1e3 * 1920 ** 0.5 * 10 + 1e-6 * 1920 / (2 * e)


# ---- norm and clipping --------------------------------------------------------------
def shapes_of(kind):
    return {"one": [(5,)], "odd": [(1,), (3,), (255,), (1023, 7), (8191,), (8192,), (8193,)],
            "large": [(2000, 3000), (17,), (1 << 20,)], "many": [(i % 97 + 1, i % 13 + 1) for i in range(700)],
            "empty ones": [(0,), (4, 0), (100,), (0, 3)], "axes": [(4, 3, 5, 7), (2, 2, 2, 2, 2), ()]}[kind]


@pytest.mark.parametrize("kind", ["one", "odd", "large", "many", "empty ones", "axes"])
@pytest.mark.parametrize("most", [0.5, 1e9])
def test_clip_grad_norm(dev, kind, most):
    g = rng(13, len(kind))
    data = [np.asarray(normal(g, *s) * np.float32(g.random() + 0.5)) for s in shapes_of(kind)]
    exact = math.sqrt(math.fsum(float(np.sum(d.astype(np.float64) ** 2)) for d in data))
    c = min(1.0, most / (exact + 1e-6))
    ts = [gpu(d, dev).reshape(d.shape) for d in data]
    n = mt.grad_norm(ts)
    assert n.shape == () and n.dtype == torch.float32
    assert abs(float(n) - exact) <= 1.01 * H * exact
    flat = torch.full((sum(d.size for d in data) + 3,), 9.0, device=dev)
    outs, at = [], 1                                    # (on odd addresses, one after the other)
    for d in data:
        outs.append(flat[at:at + d.size].view(d.shape))
        at += d.size
    assert torch.equal(mt.clip_grad_norm(ts, most, out=outs), n)
    for d, t, o in zip(data, ts, outs):
        assert np.array_equal(cpu(t), d)
        check(o, d.astype(np.float64) * c, 2.01 * H * np.abs(d) * c)
        if c == 1.0:
            assert torch.equal(o, t)
    assert float(flat[0]) == 9 and bool((flat[at:] == 9).all())
    assert torch.equal(mt.clip_grad_norm(ts, most), n)
    assert all(torch.equal(t, o) for t, o in zip(ts, outs))
    # twice the same
    again = [gpu(d, dev).reshape(d.shape) for d in data]
    assert torch.equal(mt.clip_grad_norm(again, most), n)
    assert all(torch.equal(t, o) for t, o in zip(again, outs))


def test_clip_views(dev):
    """Strided tensors beside dense ones: transposed, every second column, channels last, an
    output of other strides."""
    g = rng(14)
    base = [gpu(normal(g, 60, 50), dev), gpu(normal(g, 40, 31), dev), gpu(normal(g, 4, 6, 5, 3), dev),
            gpu(normal(g, 7, 9, 11), dev)]
    views = [base[0].t(), base[1][:, ::2], base[2].to(memory_format=torch.channels_last), base[3][:, 1:8, 2:9]]
    data = [cpu(v).copy() for v in views]
    rest = cpu(base[1][:, 1::2]).copy()
    exact = math.sqrt(math.fsum(float(np.sum(d.astype(np.float64) ** 2)) for d in data))
    assert abs(float(mt.grad_norm(views)) - exact) <= 1.01 * H * exact
    outs = [torch.empty(d.shape, device=dev) for d in data]
    mt.clip_grad_norm(views, 1.0, out=outs)
    n = mt.clip_grad_norm(views, 1.0)
    assert abs(float(n) - exact) <= 1.01 * H * exact
    for d, v, o in zip(data, views, outs):
        check(v, d.astype(np.float64) / (exact + 1e-6), 2.01 * H * np.abs(d) / exact)
        assert torch.equal(v, o)
    assert np.array_equal(cpu(base[1][:, 1::2]), rest)
    # a view with elements in common may be measured, not scaled
    e = torch.full((1, 4), 2.0, device=dev).expand(9, 4)
    assert float(mt.grad_norm([e])) == 12.0
    with pytest.raises(ValueError):
        mt.clip_grad_norm([e], 1.0)


def test_clip_magnitudes(dev):
    """Squares past fp32's range either way, infinities and NaN."""
    big = torch.full((1000,), 1e30, device=dev)
    small = torch.full((1000,), 1e-30, device=dev)
    assert float(mt.grad_norm([big])) == float(np.float32(math.sqrt(1000 * float(np.float32(1e30)) ** 2)))
    assert float(mt.grad_norm([small])) == float(np.float32(math.sqrt(1000 * float(np.float32(1e-30)) ** 2)))
    mt.clip_grad_norm([big], 1.0)
    assert abs(float(mt.grad_norm([big])) - 1.0) < 1e-6
    t = torch.tensor([1.0, float("inf")], device=dev)
    assert math.isinf(float(mt.clip_grad_norm([t], 1.0)))
    assert float(t[0]) == 0 and math.isnan(t[1])
    t = torch.tensor([1.0, float("nan")], device=dev)
    o = torch.ones(5, device=dev)
    assert math.isnan(float(mt.clip_grad_norm([t, o], 1.0)))
    assert bool(torch.isnan(t).all()) and bool(torch.isnan(o).all())
    z = torch.zeros(8, device=dev)
    assert float(mt.clip_grad_norm([z], 1.0)) == 0 and bool((z == 0).all())
    assert float(mt.clip_grad_norm([torch.empty(0, device=dev)], 1.0)) == 0
    z = torch.ones(4, device=dev)
    mt.clip_grad_norm([z], 0.0)
    assert bool((z == 0).all())


@pytest.mark.parametrize("sizes", [[1024] * 64, [1024] * 65, [65536], [65537], [1023, 1025, 1], [4099] * 12 + [3] * 4,
                                   [4099] * 12 + [3] * 5, [1] * 64, [1] * 65])
def test_clip_few_elements(dev, sizes):
    """Up to 64 chunks of 1024 go to one workgroup, more to the two launches."""
    g = rng(23, len(sizes), sizes[0])
    data = [normal(g, n) * np.float32(g.random() + 0.5) for n in sizes]
    exact = math.sqrt(math.fsum(float(np.sum(d.astype(np.float64) ** 2)) for d in data))
    c = 0.5 * exact / (exact + 1e-6)
    flat = torch.full((sum(sizes) + 6,), 9.0, device=dev)
    ts = [t.copy_(gpu(d, dev)) for t, d in zip(flat[3:-3].split(sizes), data)]
    outs = [torch.empty_like(t) for t in ts]
    assert abs(float(mt.grad_norm(ts)) - exact) <= 1.01 * H * exact
    n = mt.clip_grad_norm(ts, 0.5 * exact, out=outs)
    assert abs(float(n) - exact) <= 1.01 * H * exact
    for d, t, o in zip(data, ts, outs):
        assert np.array_equal(cpu(t), d)
        # (0.5·exact is rounded to fp32, c, and the product)
        check(o, d.astype(np.float64) * c, 3.02 * H * np.abs(d) * c)
    same = [torch.empty_like(t) for t in ts]
    assert torch.equal(mt.clip_grad_norm(ts, 2 * exact, out=same), n) and all(map(torch.equal, same, ts))
    assert torch.equal(mt.clip_grad_norm(ts, 2 * exact), n) and all(map(torch.equal, same, ts))
    assert torch.equal(mt.clip_grad_norm(ts, 0.5 * exact), n) and all(map(torch.equal, outs, ts))
    assert bool((flat[:3] == 9).all()) and bool((flat[-3:] == 9).all())


def test_clip_magnitudes_of_many(dev):
    """As test_clip_magnitudes, of more than one workgroup takes, and of strided tensors."""
    for rest in (torch.zeros(70000, device=dev), torch.zeros(9, 8, device=dev)[:, ::2]):
        big, small = torch.full((1000,), 1e30, device=dev), torch.full((1000,), 1e-30, device=dev)
        for t in (big, small):
            assert float(mt.grad_norm([t, rest])) == float(np.float32(math.sqrt(1000 * float(t[0]) ** 2)))
        mt.clip_grad_norm([big, rest], 1.0)
        assert abs(float(mt.grad_norm([big, rest])) - 1.0) < 1e-6
        t = torch.tensor([1.0, float("-inf")], device=dev)
        assert math.isinf(float(mt.clip_grad_norm([t, rest], 1.0)))
        assert float(t[0]) == 0 and math.isnan(t[1])
        t, o = torch.tensor([1.0, float("nan")], device=dev), torch.ones(5, device=dev)
        assert math.isnan(float(mt.clip_grad_norm([o, rest, t], 1.0)))
        assert all(bool(torch.isnan(a).all()) for a in (o, rest, t))
        rest.zero_()
        assert float(mt.clip_grad_norm([rest], 1.0)) == 0 and bool((rest == 0).all())
        z = torch.ones(4, device=dev)
        mt.clip_grad_norm([z, rest], 0.0)
        assert bool((z == 0).all())


# ---- use together -----------------------------------------------------------------
def block(x, w, b, wd):
    """A feed-forward block's training step: (output, clipped gradients, norm, served output)."""
    one = torch.ones(x.shape[1], device=x.device)
    n = mt.rms_norm(x, one, q8=True)
    r = mt.gated_linear(n.y, w, b, keep=True)
    y = mt.linear(r.h, wd)
    dh, dwd, _ = mt.linear_backward(y, r.h, wd, need_db=False)
    dx, dw, db = mt.gated_linear_backward(dh, r.gu, n.q8, w)
    dn, dg = mt.rms_norm_backward(dx, n.h, one, n.rstd)
    grads = [dg, dw, db, dwd]
    norm = mt.clip_grad_norm(grads, 1.0)
    served = mt.linear_q8(mt.quantize_q8(mt.gated_linear(n.q8, mt.quantize_q8(w), b).h), mt.quantize_q8(wd))
    return [y, dn, *grads, norm, served]


def block_inputs(dev, m=130, k=256, f=200):
    g = rng(15)
    return (gpu(normal(g, m, k), dev), gpu(normal(g, 2 * f, k) / 16, dev), gpu(normal(g, 2 * f), dev),
            gpu(normal(g, k, f) / 14, dev))


def test_block_trains_and_serves(dev):
    x, w, b, wd = block_inputs(dev)
    out = block(x, w, b, wd)
    X, W, B, D = (cpu(t).astype(np.float64) for t in (x, w, b, wd))
    h = X / np.sqrt((X * X).mean(1, keepdims=True) + 1e-6)
    gu = h @ W.T + B
    y = ref.gate("silu", gu)[0] @ D.T
    assert np.abs(cpu(out[0]) - y).max() <= 1e-4 * np.abs(y).max()
    assert abs(float(mt.grad_norm(out[2:6])) - 1.0) < 1e-5
    # three roundings to 8 bits on the way (rows, weights, h), each off by at most half a step
    # of the row's largest: a few hundredths of the rows' size together
    assert np.abs(cpu(out[7]) - y).max() <= 0.1 * np.abs(y).max()


def test_graph_of_the_block_replays(dev):
    x, w, b, wd = block_inputs(dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        block(x, w, b, wd)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(x, w, b, wd)
    with torch.cuda.graph(second):
        out2 = block(x, w, b, wd)
    for _ in range(3):
        x.mul_(0.75).add_(0.125)
        torch.cuda.synchronize()
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in out]
        eager = block(x, w, b, wd)
        torch.cuda.synchronize()
        for i, (a, c, d) in enumerate(zip(replayed, eager, out2)):
            assert torch.equal(a, c) and torch.equal(d, c), i


def test_block_on_another_stream(dev):
    x, w, b, wd = block_inputs(dev)
    want = block(x, w, b, wd)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x2 = x * 1
    n = mt.rms_norm(x2, q8=True, stream=s)
    r = mt.gated_linear(n.y, w, b, keep=True, stream=s)
    y = mt.linear(r.h, wd, stream=s)
    dh, dwd, _ = mt.linear_backward(y, r.h, wd, need_db=False, stream=s)
    dx, dw, db = mt.gated_linear_backward(dh, r.gu, n.q8, w, stream=s)
    grads = [dw, db, dwd]
    norm = mt.grad_norm(grads, stream=s)
    served = mt.linear_q8(mt.quantize_q8(mt.gated_linear(n.q8, mt.quantize_q8(w, stream=s), b, stream=s).h, stream=s),
                          mt.quantize_q8(wd, stream=s), stream=s)
    h = mt.gate(r.gu, stream=s)
    s.synchronize()
    assert torch.equal(y, want[0]) and torch.equal(served, want[7])
    assert float(norm) > 1
    check(h, *ref.gate("silu", cpu(r.gu)))


def test_gate_of_a_4_bit_product(dev):
    x, w, b, _ = block_inputs(dev)
    gu = mt.linear_q4(x, mt.quantize_q4(w), b)
    check(mt.gate(gu), *ref.gate("silu", cpu(gu)))


def test_refusals(dev):
    x, w = torch.ones(4, 64, device=dev), torch.ones(8, 64, device=dev)
    xq, wq = mt.quantize_q8(x), mt.quantize_q8(w)
    one = torch.ones(64, device=dev)
    gu, dh = torch.ones(4, 8, device=dev), torch.ones(4, 4, device=dev)
    bad = [
        lambda: mt.linear_q8(mt.Q8Rows(xq.q[:, :32], xq.scale), wq),
        lambda: mt.linear_q8(xq, wq, one),
        lambda: mt.linear_q8(mt.Q8Rows(x, xq.scale), wq),
        lambda: mt.linear_q8(mt.Q8Rows(xq.q, xq.scale[:3]), wq),
        lambda: mt.linear_q8(xq, mt.Q8Rows(wq.q.t(), one)),
        lambda: mt.linear_q8(xq, wq, out=torch.empty(4, 9, device=dev)),
        lambda: mt.linear_q8(xq, wq, out=torch.empty(4, 1, device=dev).expand(4, 8)),
        lambda: mt.linear_q8(mt.Q8Rows(xq.q.cpu(), xq.scale), wq),
        lambda: mt.gated_linear(x, w[:7]),
        lambda: mt.gated_linear(x, w, one),
        lambda: mt.gated_linear(x, w, act="tanh"),
        lambda: mt.gated_linear(x, wq),
        lambda: mt.gated_linear(xq, w),
        lambda: mt.gated_linear(x[:, :60], w),
        lambda: mt.gated_linear(x.half(), w),
        lambda: mt.gated_linear(x, w, out=torch.empty(4, 8, device=dev)),
        lambda: mt.gated_linear(x, w, out=torch.empty(1, 4, device=dev).expand(4, 4)),
        lambda: mt.gate(gu[:, :7]),
        lambda: mt.gate(gu[0]),
        lambda: mt.gate(gu, out=torch.empty(4, 8, device=dev)),
        lambda: mt.gate_backward(dh, gu[:3]),
        lambda: mt.gate_backward(dh.cpu(), gu),
        lambda: mt.gated_linear_backward(dh, gu, x[:3], w),
        lambda: mt.gated_linear_backward(dh, gu, x, w[:, :3]),
        lambda: mt.gated_linear_backward(dh, gu, x, dx=x),
        lambda: mt.gated_linear_backward(dh, gu, x, w, beta_w=1.0),
        lambda: mt.gated_linear_backward(dh, gu, x, w, dgu=gu[:, :4], dw=w),
        lambda: mt.gated_linear_backward(dh, gu, x, w, dw=x, dgu=gu),
        lambda: mt.clip_grad_norm([], 1.0),
        lambda: mt.clip_grad_norm([x, x], 1.0),
        lambda: mt.clip_grad_norm([x], -1.0),
        lambda: mt.clip_grad_norm([x], float("nan")),
        lambda: mt.clip_grad_norm([x], 1.0, out=[w]),
        lambda: mt.clip_grad_norm([x, w], 1.0, out=[x]),
        lambda: mt.clip_grad_norm([x.double()], 1.0),
        lambda: mt.clip_grad_norm([x.cpu()], 1.0),
        lambda: mt.grad_norm([None]),
        lambda: mt.clip_grad_norm([torch.ones(3, 4, 5, 6, device=dev)[::2, ::2, ::2, ::2]], 1.0),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"refusal {i} was taken")
    # nothing was written on the way
    assert all(bool((t == 1).all()) for t in (x, w, gu, dh))
    small = torch.empty(4, dtype=torch.uint8, device=dev)
    for f in (lambda: mt.clip_grad_norm([x], 0.5, ws=small),
              lambda: mt.linear_q8(mt.quantize_q8(torch.ones(150, 9001, device=dev)),
                                   mt.quantize_q8(torch.ones(700, 9001, device=dev)), ws=small)):
        with pytest.raises(RuntimeError):
            f()
    torch.cuda.synchronize()
    assert bool((x == 1).all())


def test_backward_refuses_before_it_writes(dev):
    """What is wrong with the second product's operands shows before the projections are
    written over."""
    g = rng(17)
    x, w, gu, dh = (gpu(normal(g, *s), dev) for s in ((200, 96), (400, 96), (200, 400), (200, 200)))
    was = gu.clone()
    row = torch.zeros(1, 96, device=dev)
    for q in (x, mt.quantize_q8(x)):
        small = torch.empty(16, dtype=torch.uint8, device=dev)
        need = (mt.lib().mt_linear_workspace_f32 if q is x else mt.lib().mt_linear_backward_q8_workspace_f32)(200, 96, 400)
        for error, f in (
                (ValueError, lambda: mt.gated_linear_backward(dh, gu, q, w, dgu=gu, dw=row.expand(400, 96))),
                (ValueError, lambda: mt.gated_linear_backward(dh, gu, q, w, dgu=gu, dx=row.expand(200, 96))),
                (ValueError, lambda: mt.gated_linear_backward(dh, gu, q, w, dgu=gu, db=row[0, :1].expand(400))),
                (ValueError, lambda: mt.gated_linear_backward(dh, gu, q, w, dgu=gu, ws=torch.empty(1 << 24))),
                (ValueError, lambda: mt.gated_linear_backward(dh, gu, q, w, dgu=gu, ws=small[:1].expand(1 << 24)))):
            with pytest.raises(error):
                f()
        if need > 16:
            with pytest.raises(RuntimeError):
                mt.gated_linear_backward(dh, gu, q, w, dgu=gu, ws=small)
        assert torch.equal(gu, was)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
        a, b = mt.gated_linear_backward(dh, gu, q, w, ws=ws), mt.gated_linear_backward(dh, gu, q, w)
        assert all(torch.equal(c, d) for c, d in zip(a, b))


def test_two_threads(dev):
    """Two threads, a stream each, one operator of another kind in flight beside each."""
    import threading
    inputs = [block_inputs(dev), block_inputs(dev, 67, 130, 300)]
    want = [block(*i) for i in inputs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for n in range(10):
                got = block(*inputs[i])
                s.synchronize()
                wrong.extend((i, n, j) for j, (a, b) in enumerate(zip(got, want[i])) if not torch.equal(a, b))
    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_views_past_32_bits(dev):
    """More than 2^31 elements, or bytes between a product's rows: the first and last rows."""
    m, f, k = 70000, 16000, 32
    g = rng(21)
    x, w = normal(g, m, k), normal(g, 2 * f, k) / np.float32(k ** 0.5)
    X, W = gpu(x, dev), gpu(w, dev)
    ends = [0, 1, m - 2, m - 1]
    r = mt.gated_linear(X, W, keep=True)
    gu, e = ref.linear(x[ends], w)
    check(r.gu[ends], gu, e)
    check(r.h[ends], *ref.gate("silu", gu, e))
    dh = r.h                                                              # (any gradient does)
    kept = r.gu[ends].clone()
    want, err = ref.gate_backward("silu", cpu(dh[ends]), cpu(kept))
    dx, dw, db = mt.gated_linear_backward(dh, r.gu, X, W, dgu=r.gu)
    check(r.gu[ends], want, err)
    # (in 64 bits on the GPU, rows at a time; bounds as in test_gated_linear_backward)
    s, a = torch.zeros(2 * f, dtype=torch.float64, device=dev), torch.zeros(2 * f, dtype=torch.float64, device=dev)
    for i in range(0, m, 5000):
        d = r.gu[i:i + 5000].double()
        s += d.sum(0)
        a += d.abs().sum(0)
        del d
    check(db, cpu(s), (m + 600) * 2.0 ** -23 * cpu(a), "db")
    out = torch.empty_like(r.gu)
    n = mt.clip_grad_norm([r.gu], 1.0, out=[out])
    total = math.sqrt(sum(float((r.gu[i:i + 5000].double() ** 2).sum()) for i in range(0, m, 5000)))
    assert abs(float(n) - total) <= 2.0 ** -23 * total
    c = min(1.0, 1.0 / (float(n) + 1e-6))
    check(out[ends], c * cpu(r.gu[ends]).astype(np.float64), 2.0 ** -21 * c * np.abs(cpu(r.gu[ends])))
    del r, dh, out, dx, dw, db
    q, sc, xq = rows8(g, m, k, dev)
    wq, ws, wt = rows8(g, 32768, k, dev)
    y = mt.linear_q8(xq, wt)
    check(y[ends], *ref.linear_q8(q[ends], sc[ends], wq, ws))


@pytest.mark.parametrize("n,f,k", [(0, 5, 6), (7, 0, 6), (7, 5, 0)])
def test_backward_of_nothing(dev, n, f, k):
    """No rows, no features, no inputs: gradients of zeros, or of no elements."""
    dh, gu = torch.ones(n, f, device=dev), torch.ones(n, 2 * f, device=dev)
    x, w = torch.ones(n, k, device=dev), torch.ones(2 * f, k, device=dev)
    for rows in (x, mt.quantize_q8(x)):
        dx, dw, db = mt.gated_linear_backward(dh, gu, rows, w)
        assert dx.shape == (n, k) and dw.shape == (2 * f, k) and db.shape == (2 * f,)
        assert bool((dx == 0).all()) and bool((dw == 0).all())
        if n == 0:
            assert bool((db == 0).all())
        elif f:
            check(db, n * ref.gate_backward("silu", np.ones((1, f), np.float32), np.ones((1, 2 * f), np.float32))[0][0],
                  np.full(2 * f, 1e-5))


def test_graph_of_a_backward_with_sums(dev):
    g = rng(22)
    m, f, k = 700, 800, 64
    x, w, dh = gpu(normal(g, m, k), dev), gpu(normal(g, 2 * f, k) / 8, dev), gpu(normal(g, m, f), dev)

    def step():
        r = mt.gated_linear(x, w, keep=True)
        return mt.gated_linear_backward(dh, r.gu, x, w)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        dh.mul_(0.5).add_(0.25)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
        torch.cuda.synchronize()
