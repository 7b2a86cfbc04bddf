"""The operators of include/mtlowbit.h against 64 bits, at the sizes, strides,
alignments and values where they can go wrong.

Tolerances follow from the number of roundings (tests/lowbit_reference.py): codes and
scales are checked bit for bit where they are defined step by step in fp32, sums
against a bound of (roundings)·2^-23 of the sum of the magnitudes."""
import numpy as np
import pytest
import torch

import lowbit_reference as ref
import minitensor_amd as mt

pytestmark = pytest.mark.gpu

ROWS_C = [1, 3, 4, 63, 64, 65, 127, 255, 256, 1023, 1024, 1025, 1285, 4096, 4097, 16384, 16385, 20001]


def rng(*key):
    return np.random.default_rng([int(k) for k in key])


def gpu(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def cpu(t):
    return t.detach().cpu().numpy()


def strided(a, dev, how):
    """`a` on the GPU under other strides: dense, transposed, every second element of
    wider rows, rows of a wider tensor from an odd element on."""
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


# ---- rows in 8 bits ------------------------------------------------------------
@pytest.mark.parametrize("c", ROWS_C)
@pytest.mark.parametrize("r", [1, 5])
def test_quantize_q8_bit_for_bit(dev, r, c):
    x = rng(1, r, c).standard_normal((r, c)).astype(np.float32) * 3
    q, s = ref.quantize_q8(x)
    got = mt.quantize_q8(gpu(x, dev))
    assert np.array_equal(cpu(got.scale), s)
    assert np.array_equal(cpu(got.q), q)
    back = cpu(mt.dequantize_q8(got))
    assert np.array_equal(back, q.astype(np.float32) * s[:, None])


@pytest.mark.parametrize("how", STRIDES)
@pytest.mark.parametrize("c", [5, 256, 1285])
def test_quantize_q8_strides(dev, how, c):
    x = rng(2, c).standard_normal((9, c)).astype(np.float32)
    q, s = ref.quantize_q8(x)
    wide = torch.full((9, c + 5), 99, dtype=torch.int8, device=dev)
    out = mt.Q8Rows(wide[:, 1:1 + c], torch.empty(9, device=dev))
    mt.quantize_q8(strided(x, dev, how), out=out)
    assert np.array_equal(cpu(out.q), q) and np.array_equal(cpu(out.scale), s)
    assert bool((wide[:, 0] == 99).all()) and bool((wide[:, 1 + c:] == 99).all())
    dst = strided(np.zeros_like(x), dev, how)
    mt.dequantize_q8(out, out=dst)
    assert np.array_equal(cpu(dst), q.astype(np.float32) * s[:, None])


@pytest.mark.parametrize("c", [64, 1285, 16385])
def test_quantize_q8_rows_of_special_values(dev, c):
    x = rng(3, c).standard_normal((9, c)).astype(np.float32)
    x[0] = 0
    x[1] = 1e-40                      # subnormal
    x[2, :] = np.finfo(np.float32).min
    x[3, c // 2] = np.inf
    x[4, c - 1] = -np.inf
    x[5, 0] = np.nan
    x[6] = 2.0 ** -149
    x[7] *= 1e-38
    q, s = ref.quantize_q8(x)
    got = mt.quantize_q8(gpu(x, dev))
    assert np.array_equal(cpu(got.q), q) and np.array_equal(cpu(got.scale), s, equal_nan=True)
    back = cpu(mt.dequantize_q8(got))
    for r in (3, 4, 5):
        assert np.isnan(back[r]).all()
    for r in (0, 1, 2, 6, 7, 8):
        assert np.all(np.abs(back[r].astype(np.float64) - x[r]) <= 0.5001 * s[r].astype(np.float64))


# ---- RMS norm ------------------------------------------------------------------
def check_rms(got, h, w, eps, c, q8=True, y=True):
    want, rstd = ref.rms_norm(h, w, eps)
    # the sum's chains (a thread's 16 values or its share of a long row, the wave's and
    # the workgroup's trees), the square root, the division, two products
    e = (16 + c / 1024 + 6 + 16 + 8) * ref.EPS32
    assert np.all(np.abs(cpu(got.rstd) - rstd) <= e * rstd)
    if y:
        assert np.all(np.abs(cpu(got.y) - want) <= e * np.abs(want) + 1e-44)
    if q8:
        top = np.abs(want).max(axis=1)
        s = cpu(got.q8.scale).astype(np.float64)
        assert np.all(np.abs(s - np.maximum(top / 127, 2.0 ** -126)) <= (e + 2 * ref.EPS32) * s)
        assert np.all(np.abs(cpu(got.q8.q) * s[:, None] - want) <=
                      0.5001 * s[:, None] + e * np.abs(want))


@pytest.mark.parametrize("c", ROWS_C)
@pytest.mark.parametrize("r", [1, 6])
def test_rms_norm(dev, r, c):
    g = rng(4, r, c)
    x, res = (g.standard_normal((r, c)).astype(np.float32) for _ in range(2))
    w = (1 + 0.1 * g.standard_normal(c)).astype(np.float32)
    got = mt.rms_norm(gpu(x, dev), gpu(w, dev), residual=gpu(res, dev), q8=True)
    h = x + res
    assert np.array_equal(cpu(got.h), h)
    check_rms(got, h, w, 1e-6, c)


@pytest.mark.parametrize("how", STRIDES)
@pytest.mark.parametrize("c", [4, 130, 1285])
def test_rms_norm_strides(dev, how, c):
    g = rng(5, c)
    x, res = (g.standard_normal((7, c)).astype(np.float32) for _ in range(2))
    w2 = g.standard_normal((c, 2)).astype(np.float32)
    w = gpu(w2, dev)[:, 1] if how == "gaps" else gpu(w2[:, 1], dev)
    h = strided(np.zeros_like(x), dev, how)
    got = mt.rms_norm(strided(x, dev, how), w, residual=strided(res, dev, "offset"), q8=True, h=h)
    assert got.h is h and np.array_equal(cpu(h), x + res)
    check_rms(got, x + res, w2[:, 1], 1e-6, c)


@pytest.mark.parametrize("c", [64, 1285, 20001])
@pytest.mark.parametrize("over", ["x", "residual"])
def test_rms_norm_stream_updated_in_place(dev, c, over):
    g = rng(6, c)
    x, res = (g.standard_normal((3, c)).astype(np.float32) for _ in range(2))
    tx, tr = gpu(x, dev), gpu(res, dev)
    got = mt.rms_norm(tx, None, residual=tr, eps=0.5, y=False, q8=True, h=tx if over == "x" else tr)
    assert np.array_equal(cpu(tx if over == "x" else tr), x + res)
    assert got.y is None
    check_rms(got, x + res, np.ones(c), 0.5, c, y=False)


def test_rms_norm_without_residual_and_broadcast_residual(dev):
    g = rng(7)
    x, row = g.standard_normal((5, 96)).astype(np.float32), g.standard_normal(96).astype(np.float32)
    w = g.standard_normal(96).astype(np.float32)
    tx = gpu(x, dev)
    got = mt.rms_norm(tx, gpu(w, dev))
    assert got.h is tx and got.q8 is None
    check_rms(got, x, w, 1e-6, 96, q8=False)
    got = mt.rms_norm(tx, gpu(w, dev), residual=gpu(row, dev).expand(5, 96))
    assert np.array_equal(cpu(got.h), x + row)
    check_rms(got, x + row, w, 1e-6, 96, q8=False)


@pytest.mark.parametrize("c", [64, 1285, 16385])
def test_rms_norm_special_rows(dev, c):
    """A zero row stays zero; one that holds an infinity or a NaN is NaN in y there
    (infinite: zero elsewhere) and reads back as NaN in 8 bits; its neighbours are
    untouched."""
    g = rng(8, c)
    x = g.standard_normal((6, c)).astype(np.float32)
    x[1] = 0
    x[2, c // 3] = np.inf
    x[3, 0] = np.nan
    x[4] = np.finfo(np.float32).min          # squares overflow: y = 0
    got = mt.rms_norm(gpu(x, dev), None, q8=True)
    y, back = cpu(got.y), cpu(mt.dequantize_q8(got.q8))
    assert np.all(y[1] == 0) and np.all(back[1] == 0)
    assert np.isnan(y[2, c // 3]) and np.all(np.delete(y[2], c // 3) == 0)
    assert np.isnan(y[3]).all() and np.isnan(back[2]).all() and np.isnan(back[3]).all()
    assert np.all(y[4] == 0) and np.all(back[4] == 0)
    keep = mt.RmsNorm(got.y[[0, 5]], got.h[[0, 5]], got.rstd[[0, 5]],
                      mt.Q8Rows(got.q8.q[[0, 5]], got.q8.scale[[0, 5]]))
    check_rms(keep, x[[0, 5]], np.ones(c), 1e-6, c)


@pytest.mark.parametrize("r,c", [(1, 1), (1, 4096), (2, 3), (9, 65), (300, 1285), (37, 4097),
                                 (5000, 64), (3, 16384), (5, 20001), (2100, 200)])
@pytest.mark.parametrize("stream_grad", [False, True])
def test_rms_norm_backward(dev, r, c, stream_grad):
    g = rng(9, r, c)
    h, dy, dh0 = (g.standard_normal((r, c)).astype(np.float32) for _ in range(3))
    w, dw0 = (g.standard_normal(c).astype(np.float32) for _ in range(2))
    rstd = ref.rms_norm(h, w, 1e-6)[1].astype(np.float32)
    t = [gpu(a, dev) for a in (dy, h, w, rstd)]
    beta = 0.5 if stream_grad else 0.0
    dh, dw = mt.rms_norm_backward(*t, dh=gpu(dh0, dev) if stream_grad else None,
                                  dw=gpu(dw0, dev) if stream_grad else None, beta=beta)
    want_h, want_w, size, wsum = ref.rms_norm_backward(dy, h, w, rstd, dh0 if stream_grad else None)
    e = 2 * (16 + c / 1024 + 6 + 16 + 8) * ref.EPS32
    assert np.all(np.abs(cpu(dh) - want_h) <= e * size)
    if stream_grad:
        want_w = want_w + beta * dw0
        wsum = wsum + np.abs(beta * dw0)
    # a group's rows, then the groups: 64 and 16 in a row at most 2048 of them
    assert np.all(np.abs(cpu(dw) - want_w) <= (r / 512 + 2048 / 16 + 16 + 8) * ref.EPS32 * 2 * wsum)


@pytest.mark.parametrize("how", STRIDES)
def test_rms_norm_backward_strides_and_in_place(dev, how):
    g = rng(10)
    r, c = 13, 77
    h, dy, dh0 = (g.standard_normal((r, c)).astype(np.float32) for _ in range(3))
    w = g.standard_normal(c).astype(np.float32)
    rstd = ref.rms_norm(h, w, 1e-6)[1].astype(np.float32)
    acc = strided(dh0, dev, how)
    dws = torch.zeros(c, 3, device=dev)
    dh, dw = mt.rms_norm_backward(strided(dy, dev, "offset"), strided(h, dev, how), gpu(w, dev),
                                  gpu(rstd, dev), dh=acc, out=acc, dw=dws[:, 1])
    want_h, want_w, size, wsum = ref.rms_norm_backward(dy, h, w, rstd, dh0)
    assert dh is acc
    assert np.all(np.abs(cpu(acc) - want_h) <= 100 * ref.EPS32 * size)
    assert np.all(np.abs(cpu(dws[:, 1]) - want_w) <= 100 * ref.EPS32 * wsum)
    assert bool((dws[:, 0] == 0).all()) and bool((dws[:, 2] == 0).all())


def test_rms_norm_gradient_against_differences(dev):
    """The kernel's gradients of L = sum(dy·y) against central differences of the
    64-bit forward (step 1e-4: their own error is below 1e-7 of the gradient's size)."""
    g = rng(11)
    r, c = 4, 37
    h, dy = (g.standard_normal((r, c)).astype(np.float32) for _ in range(2))
    w = g.standard_normal(c).astype(np.float32)
    fwd = mt.rms_norm(gpu(h, dev), gpu(w, dev))
    dh, dw = mt.rms_norm_backward(gpu(dy, dev), fwd.h, gpu(w, dev), fwd.rstd)
    loss = lambda hh, ww: np.sum(dy.astype(np.float64) * ref.rms_norm(hh, ww, 1e-6)[0])  # noqa: E731
    step = 1e-4
    for i, j in [(0, 0), (1, 36), (2, 17), (3, 5)]:
        d = np.zeros((r, c))
        d[i, j] = step
        num = (loss(h + d, w) - loss(h - d, w)) / (2 * step)
        assert abs(num - cpu(dh)[i, j]) <= 2e-5 * np.abs(cpu(dh)).max()
        d = np.zeros(c)
        d[j] = step
        num = (loss(h, w + d) - loss(h, w - d)) / (2 * step)
        assert abs(num - cpu(dw)[j]) <= 2e-5 * np.abs(cpu(dw)).max()


# ---- 4-bit weights -------------------------------------------------------------
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 31), (5, 32), (2, 33), (7, 127), (4, 128), (3, 129),
                                 (9, 1000)])
def test_quantize_q4_bit_for_bit(dev, group, n, k):
    w = rng(12, n, k).standard_normal((n, k)).astype(np.float32)
    w[0, 0] = 0
    code, scale = ref.quantize_q4(w, group)
    for how in ("dense", "transposed", "offset"):
        got = mt.quantize_q4(strided(w, dev, how), group)
        assert np.array_equal(cpu(got.packed), ref.pack_q4(code)), how
        assert np.array_equal(cpu(got.scale), scale), how
    want = code.astype(np.float32) * np.repeat(scale, group, axis=1)[:, :k]
    assert np.array_equal(cpu(mt.dequantize_q4(got)), want)


def test_quantize_q4_special_groups(dev):
    w = rng(13).standard_normal((4, 96)).astype(np.float32)
    w[0, :32] = 0
    w[1, 40] = np.inf
    w[2, 95] = np.nan
    w[3, 32:64] = 1e-40
    got = mt.quantize_q4(gpu(w, dev), 32)
    code, scale = ref.quantize_q4(w, 32)
    assert np.array_equal(cpu(got.packed), ref.pack_q4(code))
    assert np.array_equal(cpu(got.scale), scale, equal_nan=True)
    back = cpu(mt.dequantize_q4(got))
    assert np.isnan(back[1, 32:64]).all() and np.isnan(back[2, 64:]).all()
    assert np.isfinite(back[[0, 3]]).all() and np.all(back[0, :32] == 0)


def q4_case(dev, key, m, n, k, group, q8, low=-8):
    """Operands with every code from -8, random bytes past K, and their 64-bit product."""
    g = rng(14, key, m, n, k, group)
    code = g.integers(low, 8, (n, k)).astype(np.int8)
    scale = (g.random((n, -(-k // group))) + 0.5).astype(np.float32) / 8
    wq = mt.Q4Weight(gpu(ref.pack_q4(code, filler=int(g.integers(-8, 8))), dev), gpu(scale, dev), k,
                     group)
    w = ref.weight_q4(code, scale, group)
    if q8:
        q = g.integers(-128, 128, (m, k)).astype(np.int8)
        s = (g.random(m) + 0.5).astype(np.float32)
        return mt.Q8Rows(gpu(q, dev), gpu(s, dev)), q.astype(np.float64) * s[:, None], wq, w
    x = g.standard_normal((m, k)).astype(np.float32)
    return gpu(x, dev), x.astype(np.float64), wq, w


def check_q4(y, x, w, group, q8, bias=None):
    want, size = x @ w.T, np.abs(x) @ np.abs(w).T
    if bias is not None:
        want, size = want + bias, size + np.abs(bias)
    bound = ref.linear_bound(x.shape[1], group, 1 if q8 else 3) * size + 1e-44
    err = np.abs(cpu(y) - want)
    assert np.all(err <= bound), (float((err / np.maximum(bound, 1e-300)).max()), y.shape)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 16, 128), (1, 17, 31), (2, 15, 33), (3, 100, 160), (5, 33, 1000), (6, 16, 256),
    (8, 129, 127), (10, 48, 129), (11, 64, 512), (16, 31, 2047), (17, 130, 384), (21, 20, 96),
    (32, 257, 640), (48, 64, 300), (49, 65, 4096), (64, 128, 128), (65, 129, 1025), (128, 128, 256),
    (130, 260, 200), (200, 1000, 2048), (1, 4096, 4096), (1, 64, 16500)])
def test_linear_q4(dev, group, q8, m, n, k):
    x, xd, wq, w = q4_case(dev, 0, m, n, k, group, q8)
    b = rng(15, n).standard_normal(n).astype(np.float32)
    check_q4(mt.linear_q4(x, wq, gpu(b, dev)), xd, w, group, q8, b)
    y = mt.linear_q4(x, wq)
    check_q4(y, xd, w, group, q8)
    assert torch.equal(y, mt.linear_q4(x, wq))          # the same bits every time


@pytest.mark.parametrize("m,n,k", [(1, 40, 200), (7, 33, 130), (40, 70, 260), (150, 140, 400)])
@pytest.mark.parametrize("how", STRIDES)
def test_linear_q4_strides(dev, how, m, n, k):
    x, xd, wq, w = q4_case(dev, 1, m, n, k, 64, False)
    b2 = gpu(rng(16, n).standard_normal((n, 3)).astype(np.float32), dev)
    out = strided(np.zeros((m, n), np.float32), dev, how)
    y = mt.linear_q4(strided(cpu(x), dev, how), wq, b2[:, 2], out=out)
    assert y is out
    check_q4(out, xd, w, 64, False, cpu(b2[:, 2]))
    # a run of the weight's rows, and 8-bit rows of a wider tensor at an odd byte
    part = mt.Q4Weight(wq.packed[3:], wq.scale[3:], k, 64)
    check_q4(mt.linear_q4(x, part), xd, w[3:], 64, False)
    xq, xqd, wq, w = q4_case(dev, 2, m, n, k, 64, True)
    wide = torch.zeros(m, k + 9, dtype=torch.int8, device=dev)
    wide[:, 5:5 + k] = xq.q
    check_q4(mt.linear_q4(mt.Q8Rows(wide[:, 5:5 + k], xq.scale), wq), xqd, w, 64, True)


@pytest.mark.parametrize("m", [3, 70, 200])
def test_linear_q4_infinities_and_nan(dev, m):
    """As 64-bit sums of the products give them: an infinity times a code, NaN from inf - inf
    and from inf·0, and only in the rows and columns that hold them."""
    n, k, group = 40, 300, 32
    x, xd, wq, w = q4_case(dev, 3, m, n, k, group, False)
    x[0, 7] = float("inf")
    x[1, 290] = float("-inf")
    x[2, 5] = float("nan")
    wq.scale[11, 2] = float("nan")
    wq.scale[12, 3] = float("inf")
    xd, w = cpu(x).astype(np.float64), np.array(w)
    code = w / np.repeat(cpu(q4_case(dev, 3, m, n, k, group, False)[2].scale), group, 1)[:, :k]
    with np.errstate(all="ignore"):
        w = np.rint(code) * np.repeat(cpu(wq.scale).astype(np.float64), group, 1)[:, :k]
        want = xd @ w.T
    y = cpu(mt.linear_q4(x, wq)).astype(np.float64)
    fine = np.isfinite(want)
    # a group times an infinite scale is one product of its sum, where 64 bits take each
    # code's: the column is not a finite number either way
    others = np.arange(n) != 12
    assert np.array_equal(np.isfinite(y), fine)
    assert np.array_equal(np.isnan(y[:, others]), np.isnan(want[:, others]))
    inf = np.isinf(want) & others
    assert np.array_equal(y[inf], want[inf])
    near = np.where(fine, y, 0) - np.where(fine, want, 0)
    assert np.all(np.abs(near)[fine] <= (ref.linear_bound(k, group, 3) *
                                             (np.abs(np.where(np.isfinite(xd), xd, 0)) @
                                              np.abs(np.where(np.isfinite(w), w, 0)).T))[fine])


@pytest.mark.parametrize("m", [2, 80])
def test_linear_q4_small_and_large_magnitudes(dev, m):
    """Inputs from 1e-30 to 1e30: all 24 bits of each count."""
    x, xd, wq, w = q4_case(dev, 4, m, 48, 256, 128, False)
    for p in (-30, -10, 10, 30):
        xs = x * 10.0 ** p
        check_q4(mt.linear_q4(xs, wq), cpu(xs).astype(np.float64), w, 128, False)


def test_linear_q4_rows_of_another_scale_do_not_mix(dev):
    """Zero rows, rows of scale zero and NaN rows beside ordinary 8-bit ones."""
    x, xd, wq, w = q4_case(dev, 5, 6, 50, 200, 64, True)
    x.scale[1] = 0
    x.scale[3] = float("nan")
    x.q[4] = 0
    y = mt.linear_q4(x, wq)
    assert bool((y[1] == 0).all()) and bool((y[4] == 0).all()) and bool(y[3].isnan().all())
    keep = [0, 2, 5]
    check_q4(y[keep], xd[keep], w, 64, True)


# ---- gradients from rows kept in 8 bits ---------------------------------------
def back_case(dev, r, fin, fout):
    g = rng(17, r, fin, fout)
    q = g.integers(-128, 128, (r, fin)).astype(np.int8)
    s = (g.random(r) + 0.5).astype(np.float32) / 64
    dy = g.standard_normal((r, fout)).astype(np.float32)
    w = g.standard_normal((fout, fin)).astype(np.float32)
    return dy, q, s, w


def check_back(got, dy, q, s, w, dw0=None, db0=None, beta=0.0):
    dx, dw, db = got
    dy, x = dy.astype(np.float64), q.astype(np.float64) * s[:, None]
    r = len(s)
    if dw is not None:
        want, size = dy.T @ x, np.abs(dy).T @ np.abs(x)
        if dw0 is not None:
            want, size = want + beta * dw0, size + np.abs(beta * dw0)
        assert np.all(np.abs(cpu(dw) - want) <= ref.linear_bound(r, 128, 3) * size + 1e-44)
    if db is not None:
        want, size = dy.sum(0), np.abs(dy).sum(0)
        if db0 is not None:
            want, size = want + beta * db0, size + np.abs(beta * db0)
        assert np.all(np.abs(cpu(db) - want) <= (r + 8) * ref.EPS32 * size)
    if dx is not None:
        # the framework's own product of two fp32 operands
        bound = mt.tolerance(dy.shape[1], np.abs(dy).max(), np.abs(w).max())
        assert np.abs(cpu(dx) - dy @ w.astype(np.float64)).max() <= bound


@pytest.mark.parametrize("r,fin,fout", [
    (1, 1, 1), (1, 64, 64), (3, 5, 7), (31, 64, 33), (32, 63, 65), (33, 130, 64), (127, 64, 129),
    (128, 128, 128), (129, 257, 100), (256, 2048, 1000), (1000, 70, 10), (1027, 771, 1285),
    (4096, 64, 64), (5000, 100, 36), (600, 2100, 2050)])
def test_linear_backward_q8(dev, r, fin, fout):
    dy, q, s, w = back_case(dev, r, fin, fout)
    xq = mt.Q8Rows(gpu(q, dev), gpu(s, dev))
    got = mt.linear_backward_q8(gpu(dy, dev), xq, gpu(w, dev))
    check_back(got, dy, q, s, w)
    g = rng(18, r)
    dw0, db0 = g.standard_normal((fout, fin)).astype(np.float32), g.standard_normal(fout).astype(np.float32)
    dw, db = gpu(dw0, dev), gpu(db0, dev)
    got2 = mt.linear_backward_q8(gpu(dy, dev), xq, dw=dw, db=db, beta_w=0.5, beta_b=0.5)
    assert got2[0] is None and got2[1] is dw and got2[2] is db
    check_back(got2, dy, q, s, w, dw0, db0, 0.5)
    again = mt.linear_backward_q8(gpu(dy, dev), xq, gpu(w, dev))
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("how", STRIDES)
def test_linear_backward_q8_strides(dev, how):
    r, fin, fout = 150, 70, 90
    dy, q, s, w = back_case(dev, r, fin, fout)
    wide = torch.zeros(r, fin + 9, dtype=torch.int8, device=dev)
    wide[:, 3:3 + fin] = gpu(q, dev)
    dw = strided(np.zeros((fout, fin), np.float32), dev, how)
    dbs = torch.zeros(fout, 2, device=dev)
    got = mt.linear_backward_q8(strided(dy, dev, how), mt.Q8Rows(wide[:, 3:3 + fin], gpu(s, dev)),
                                strided(w, dev, how), dw=dw, db=dbs[:, 1])
    check_back(got, dy, q, s, w)
    assert bool((dbs[:, 0] == 0).all())
    # one row's gradient for all (a mean's backward pass): dY of stride 0
    row = gpu(dy[:1], dev).expand(r, fout)
    check_back(mt.linear_backward_q8(row, mt.Q8Rows(gpu(q, dev), gpu(s, dev))),
               np.repeat(dy[:1], r, 0), q, s, w)


def test_linear_backward_q8_special_values(dev):
    """An infinity in dY reaches its output's row of dW only; a NaN row of x every one."""
    r, fin, fout = 200, 64, 70
    dy, q, s, w = back_case(dev, r, fin, fout)
    q[5, 3] = 0                                  # inf·0 is NaN
    q[5, 4] = 9
    dy[5, 11] = np.inf
    dy[:, 12] = 0
    _, dw, db = mt.linear_backward_q8(gpu(dy, dev), mt.Q8Rows(gpu(q, dev), gpu(s, dev)))
    dw = cpu(dw)
    assert np.isnan(dw[11, 3]) and np.isposinf(dw[11, 4]) and np.isposinf(cpu(db)[11])
    assert np.isfinite(np.delete(dw, 11, 0)).all() and np.all(dw[12] == 0)
    s[7] = np.nan
    _, dw, _ = mt.linear_backward_q8(gpu(dy, dev), mt.Q8Rows(gpu(q, dev), gpu(s, dev)))
    assert bool(dw.isnan().all())


def test_linear_gradients_against_differences(dev):
    """L = sum(dY·(x·wᵀ)) is linear in w and in x: a difference of any step is the
    gradient, up to 64-bit rounding and the kernel's own bound."""
    r, fin, fout = 40, 50, 30
    dy, q, s, w = back_case(dev, r, fin, fout)
    x = q.astype(np.float64) * s[:, None]
    dx, dw, _ = mt.linear_backward_q8(gpu(dy, dev), mt.Q8Rows(gpu(q, dev), gpu(s, dev)), gpu(w, dev))
    loss = lambda xx, ww: np.sum(dy.astype(np.float64) * (xx @ ww.T))  # noqa: E731
    w64 = w.astype(np.float64)
    for i, j in [(0, 0), (29, 49), (13, 7)]:
        d = np.zeros_like(w64)
        d[i, j] = 1
        assert abs(loss(x, w64 + d) - loss(x, w64) - cpu(dw)[i, j]) <= 1e-5 * np.abs(cpu(dw)).max()
        d = np.zeros_like(x)
        d[i, j] = 1
        assert abs(loss(x + d, w64) - loss(x, w64) - cpu(dx)[i, j]) <= 1e-5 * np.abs(cpu(dx)).max()


# ---- empty, far, other streams, graphs ----------------------------------------
def test_empty_and_zero_length(dev):
    e = torch.empty(0, 8, device=dev)
    assert mt.quantize_q8(e).q.shape == (0, 8)
    assert mt.dequantize_q8(mt.quantize_q8(e)).shape == (0, 8)
    n = mt.rms_norm(e, torch.ones(8, device=dev), q8=True)
    assert n.y.shape == (0, 8) and n.rstd.shape == (0,)
    dh, dw = mt.rms_norm_backward(e, e, None, n.rstd)
    assert dh.shape == (0, 8) and bool((dw == 0).all())
    w = mt.quantize_q4(torch.ones(5, 8, device=dev))
    assert mt.linear_q4(e, w).shape == (0, 5)
    b = torch.arange(5.0, device=dev)
    none = mt.quantize_q4(torch.empty(5, 0, device=dev))
    y = mt.linear_q4(torch.empty(3, 0, device=dev), none, b)
    assert torch.equal(y, b.expand(3, 5))
    assert bool((mt.linear_q4(torch.empty(3, 0, device=dev), none) == 0).all())
    dw0, db0 = torch.ones(4, 8, device=dev), torch.ones(4, device=dev)
    dx, dw, db = mt.linear_backward_q8(torch.empty(0, 4, device=dev), mt.quantize_q8(e),
                                       torch.ones(4, 8, device=dev), dw=dw0, db=db0, beta_w=0.5,
                                       beta_b=0.25)
    assert dx.shape == (0, 8) and bool((dw == 0.5).all()) and bool((db == 0.25).all())
    torch.cuda.synchronize()


def test_offsets_past_32_bits(dev):
    """Rows 1.2e9 elements apart: element offsets beyond 2^31 (fp32 rows, 8-bit rows)."""
    step, c = 1_200_000_000, 96
    big = torch.empty(2 * step + c, device=dev)
    x = big.as_strided((3, c), (step, 1))
    src = gpu(rng(19).standard_normal((3, c)).astype(np.float32), dev)
    x.copy_(src)
    got, want = mt.quantize_q8(x), mt.quantize_q8(src)
    assert torch.equal(got.q, want.q) and torch.equal(got.scale, want.scale)
    w = torch.ones(c, device=dev)
    assert torch.equal(mt.rms_norm(x, w).y, mt.rms_norm(src, w).y)
    wq = mt.quantize_q4(gpu(rng(20).standard_normal((40, c)).astype(np.float32), dev))
    assert torch.equal(mt.linear_q4(x, wq), mt.linear_q4(src, wq))
    n = mt.rms_norm(src, w)
    for a, b in zip(mt.rms_norm_backward(x, n.h, w, n.rstd), mt.rms_norm_backward(src, n.h, w, n.rstd)):
        assert torch.equal(a, b)
    for a, b in zip(mt.linear_backward_q8(x, want), mt.linear_backward_q8(src, want)):
        if a is not None:
            assert torch.equal(a, b)
    bytes_ = big.view(torch.int8)
    far = bytes_.as_strided((3, c), (3 * step, 1))
    far.copy_(want.q)
    rows = mt.Q8Rows(far, want.scale)
    assert torch.equal(mt.dequantize_q8(rows), mt.dequantize_q8(want))
    assert torch.equal(mt.linear_q4(rows, wq), mt.linear_q4(want, wq))
    dy = src[:, :30].contiguous()
    assert torch.equal(mt.linear_backward_q8(dy, rows)[1], mt.linear_backward_q8(dy, want)[1])


def test_on_another_stream(dev):
    """Inputs filled on a stream, operators on the same one through `stream`."""
    g = rng(21)
    x, res = (gpu(g.standard_normal((64, 512)).astype(np.float32), dev) for _ in range(2))
    w = gpu(g.standard_normal((96, 512)).astype(np.float32), dev)
    one = torch.ones(512, device=dev)
    n = mt.rms_norm(x, one, residual=res, q8=True)
    wq = mt.quantize_q4(w)
    y = mt.linear_q4(n.q8, wq)
    back = mt.linear_backward_q8(y, n.q8, w)
    hb = mt.rms_norm_backward(back[0], n.h, one, n.rstd)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x2, res2 = x * 1, res * 1
    n2 = mt.rms_norm(x2, one, residual=res2, q8=True, stream=s)
    y2 = mt.linear_q4(n2.q8, mt.quantize_q4(w, stream=s), stream=s)
    back2 = mt.linear_backward_q8(y2, n2.q8, w, stream=s)
    hb2 = mt.rms_norm_backward(back2[0], n2.h, one, n2.rstd, stream=s)
    s.synchronize()
    assert torch.equal(n.q8.q, n2.q8.q) and torch.equal(y, y2)
    assert all(torch.equal(a, b) for a, b in zip(back + hb, back2 + hb2))


def test_graph_of_the_chain_replays(dev):
    """norm -> 8-bit rows -> 4-bit layer -> gradients, captured, three replays with
    new inputs against the eager calls."""
    g = rng(22)
    x, res = (gpu(g.standard_normal((130, 512)).astype(np.float32), dev) for _ in range(2))
    w = gpu(g.standard_normal((200, 512)).astype(np.float32), dev)
    wq, one = mt.quantize_q4(w), torch.ones(512, device=dev)

    def chain():
        n = mt.rms_norm(x, one, residual=res, q8=True)
        y = mt.linear_q4(n.q8, wq)
        dx, dw, db = mt.linear_backward_q8(y, n.q8, w)
        return [n.h, n.q8.q, y, dx, dw, db, *mt.rms_norm_backward(dx, n.h, one, n.rstd),
                mt.dequantize_q8(n.q8)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        chain()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain()
    for _ in range(3):
        x.mul_(0.5).add_(0.125)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in out]
        eager = chain()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(replayed, eager))


def test_refusals(dev):
    x, w = torch.ones(4, 64, device=dev), torch.ones(8, 64, device=dev)
    wq, xq = mt.quantize_q4(w), mt.quantize_q8(x)
    one = torch.ones(64, device=dev)
    bad = [
        lambda: mt.quantize_q8(x[0]),
        lambda: mt.quantize_q8(x.double()),
        lambda: mt.quantize_q8(x.cpu()),
        lambda: mt.dequantize_q8(mt.Q8Rows(xq.q, xq.scale[:3])),
        lambda: mt.dequantize_q8(mt.Q8Rows(xq.q.float(), xq.scale)),
        lambda: mt.dequantize_q8(mt.Q8Rows(xq.q.t(), one)),
        lambda: mt.rms_norm(x, one[:63]),
        lambda: mt.rms_norm(x, one, residual=x[:3]),
        lambda: mt.rms_norm(x, one, h=x[:, :60]),
        lambda: mt.rms_norm(x, one, eps=-1.0),
        lambda: mt.rms_norm(x.half(), one),
        lambda: mt.rms_norm_backward(x, x, one, one[:3]),
        lambda: mt.rms_norm_backward(x, x, one, one[:4], beta=1.0),
        lambda: mt.quantize_q4(w, 48),
        lambda: mt.linear_q4(x[:, :32], wq),
        lambda: mt.linear_q4(x, wq, one),
        lambda: mt.linear_q4(x, mt.Q4Weight(wq.packed, wq.scale, 64, 16)),
        lambda: mt.linear_q4(x, mt.Q4Weight(wq.packed, wq.scale, 60, 32)),
        lambda: mt.linear_q4(x, mt.Q4Weight(wq.packed.flatten()[8:-8].reshape(-1, 16), wq.scale, 32, 32)),
        lambda: mt.linear_q4(x.cpu(), wq),
        lambda: mt.linear_q4(x, wq, out=torch.empty(4, 9, device=dev)),
        lambda: mt.linear_q4(x, wq, out=torch.empty(4, 1, device=dev).expand(4, 8)),
        lambda: mt.linear_backward_q8(torch.ones(3, 8, device=dev), xq),
        lambda: mt.linear_backward_q8(torch.ones(4, 8, device=dev), xq, w[:7]),
        lambda: mt.linear_backward_q8(torch.ones(4, 8, device=dev), xq, beta_w=1.0),
        lambda: mt.linear_backward_q8(torch.ones(4, 8, device=dev), xq, dw=one),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"refusal {i} was taken")
    # a workspace that is too small is refused before anything is launched
    dy, big = torch.ones(4096, 64, device=dev), mt.quantize_q8(torch.ones(4096, 64, device=dev))
    dw = torch.full((64, 64), 5.0, device=dev)
    with pytest.raises(RuntimeError):
        mt.linear_backward_q8(dy, big, dw=dw, ws=torch.empty(4, dtype=torch.uint8, device=dev))
    torch.cuda.synchronize()
    assert bool((dw == 5).all())
