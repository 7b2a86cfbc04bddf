"""Calls of the operators of include/mtffn.h and mt_linear_q8 at the ends of what they take:
views that no kernel reads, gradients past fp32's range, sums over very many rows, products of
no inputs."""
import ctypes

import numpy as np
import pytest
import torch

import ffn_reference as ref
import minitensor_amd as mt

pytestmark = pytest.mark.gpu

H = ref.H


def negated(*shape, dev):
    """A float32 view whose elements are kept with the other sign (its negative bit is set)."""
    v = torch.complex(torch.ones(shape, device=dev), torch.ones(shape, device=dev)).conj().imag
    assert v.is_neg() and v.dtype == torch.float32
    return v


def test_negated_views_are_refused(dev):
    """Kernels read memory as it lies: a lazily negated view would be taken with the wrong sign."""
    x, w, gu, dh = (torch.ones(*s, device=dev) for s in ((4, 64), (8, 64), (4, 8), (4, 4)))
    b, vec = torch.ones(8, device=dev), torch.ones(64, device=dev)
    img, ker, dimg = (torch.ones(*s, device=dev) for s in ((1, 2, 5, 5), (3, 2, 1, 1), (1, 3, 5, 5)))
    xq, wq = mt.quantize_q8(x), mt.quantize_q8(w)
    n = lambda *s: negated(*s, dev=dev)
    q = mt.Q8Rows(xq.q, n(4))
    h, rstd = x, torch.ones(4, device=dev)
    calls = [
        lambda: mt.gated_linear(n(4, 64), w), lambda: mt.gated_linear(x, n(8, 64)),
        lambda: mt.gated_linear(x, w, n(8)), lambda: mt.gated_linear(x, w, out=n(4, 4)),
        lambda: mt.gated_linear(q, wq), lambda: mt.gated_linear(xq, wq, n(8)),
        lambda: mt.gate(n(4, 8)), lambda: mt.gate(gu, out=n(4, 4)),
        lambda: mt.gate_backward(n(4, 4), gu), lambda: mt.gate_backward(dh, n(4, 8)),
        lambda: mt.gate_backward(dh, gu, out=n(4, 8)),
        lambda: mt.gated_linear_backward(n(4, 4), gu, x, w), lambda: mt.gated_linear_backward(dh, n(4, 8), x, w),
        lambda: mt.gated_linear_backward(dh, gu, n(4, 64), w), lambda: mt.gated_linear_backward(dh, gu, x, n(8, 64)),
        lambda: mt.gated_linear_backward(dh, gu, q, w), lambda: mt.gated_linear_backward(dh, gu, x, w, dgu=n(4, 8)),
        lambda: mt.gated_linear_backward(dh, gu, x, w, dx=n(4, 64)),
        lambda: mt.gated_linear_backward(dh, gu, x, w, dw=n(8, 64)),
        lambda: mt.gated_linear_backward(dh, gu, x, w, db=n(8)),
        lambda: mt.linear_q8(q, wq), lambda: mt.linear_q8(xq, mt.Q8Rows(wq.q, n(8))),
        lambda: mt.linear_q8(xq, wq, n(8)), lambda: mt.linear_q8(xq, wq, out=n(4, 8)),
        lambda: mt.grad_norm([x, n(3, 3)]), lambda: mt.clip_grad_norm([n(3, 3)], 1.0),
        lambda: mt.clip_grad_norm([x], 1.0, out=[n(4, 64)]),
        # ... and the operators beside them, which take their operands the same way
        lambda: mt.gemm(n(4, 64), w.t()), lambda: mt.gemm(x, w.t(), out=n(4, 8)),
        lambda: mt.linear(n(4, 64), w), lambda: mt.linear(x, w, n(8)),
        lambda: mt.linear_backward(n(4, 8), x, w), lambda: mt.linear_backward(gu, x, w, db=n(8)),
        lambda: mt.colsum(n(4, 8)), lambda: mt.axpby(n(4, 8), gu), lambda: mt.axpby(gu, n(4, 8)),
        lambda: mt.conv2d(n(1, 2, 5, 5), ker), lambda: mt.conv2d(img, ker, n(3)),
        lambda: mt.conv2d_backward(img, n(3, 2, 1, 1), dimg),
        lambda: mt.conv2d_backward(img, ker, dimg, dw=n(3, 2, 1, 1)),
        lambda: mt.rms_norm(n(4, 64)), lambda: mt.rms_norm(x, n(64)),
        lambda: mt.rms_norm_backward(n(4, 64), h, vec, rstd), lambda: mt.rms_norm_backward(x, h, vec, n(4)),
        lambda: mt.quantize_q8(n(4, 64)), lambda: mt.quantize_q4(n(8, 64)),
        lambda: mt.dequantize_q8(q), lambda: mt.linear_backward_q8(gu, q, w),
        lambda: mt.linear_q4(n(4, 64), mt.quantize_q4(w)), lambda: mt.linear_q4(x, mt.quantize_q4(w), n(8)),
    ]
    taken = []
    for i, call in enumerate(calls):
        try:
            call()
            taken.append(i)
        except ValueError:
            pass
    assert not taken
    assert all(bool((t == 1).all()) for t in (x, w, gu, dh, b, vec))


def test_rows_over_each_other_are_refused_before_the_projections_are_written_over(dev):
    """Rows that the second product does not take: those in 8 bits that share memory, and longer
    ones than its extents hold."""
    dh, gu, w = torch.ones(6, 5, device=dev), torch.full((6, 10), 2.0, device=dev), torch.ones(10, 32, device=dev)
    one = torch.ones(6, device=dev)
    q = torch.ones(1, 96, dtype=torch.int8, device=dev)
    for rows in (q[:, :32].expand(6, 32), q[0].as_strided((6, 32), (8, 1))):
        with pytest.raises(ValueError):
            mt.gated_linear_backward(dh, gu, mt.Q8Rows(rows, one), w, dgu=gu)
        assert bool((gu == 2).all())
    with pytest.raises(ValueError):
        mt.gated_linear_backward(dh, gu, one[:, None].expand(6, 1 << 31), need_dw=False, dgu=gu)
    assert bool((gu == 2).all())


@pytest.mark.parametrize("m,n", [(300, 4096), (3, 40), (70, 200)])
def test_no_inputs_far_apart(dev, m, n):
    """Rows of no inputs, whatever lies between them: the bias."""
    x = torch.empty(1, dtype=torch.int8, device=dev).as_strided((m, 0), (1 << 24, 1))
    x = mt.Q8Rows(x, torch.ones(m, device=dev))
    b = torch.arange(2.0 * n, device=dev) - n / 2
    w = lambda r: mt.Q8Rows(torch.empty(r, 0, dtype=torch.int8, device=dev), torch.ones(r, device=dev))
    assert torch.equal(mt.linear_q8(x, w(n), b[:n]), b[:n].expand(m, n))
    r = mt.gated_linear(x, w(2 * n), b, act="relu", keep=True)
    assert torch.equal(r.gu, b.expand(m, 2 * n))
    assert torch.equal(r.h, (b[:n].clamp_min(0) * b[n:]).expand(m, n))


@pytest.mark.parametrize("kind", ["few", "many", "strided"])
@pytest.mark.parametrize("value,most", [(3e38, 1.0), (3e38, 1e-3), (1e36, 1e-5), (1e8, 1e-30), (1e-38, 1e-44)])
def test_clip_factors_below_the_normal_range(dev, kind, value, most):
    """A factor below 2^-126 times gradients that lift the product above it again: one rounding
    of the product, not of the factor."""
    n = {"few": 1000, "many": 100000, "strided": 5000}[kind]
    t = torch.full((n // 10, 20), value, device=dev)
    t = t[:, ::2] if kind == "strided" else t[:, :10].contiguous()
    v, m = float(t[0, 0]), float(np.float32(most))
    norm = v * (t.numel() ** 0.5)
    want = v * min(1.0, m / (norm + float(np.float32(0.0))))
    # the product once, of a factor that is right to a few roundings in 64 bits
    bound = 1.01 * H * want + 2.0 ** -149
    out = torch.empty(t.shape, device=dev)
    mt.clip_grad_norm([t], most, out=[out], eps=0.0)
    assert abs(out.double() - want).max().item() <= bound
    mt.clip_grad_norm([t], most, eps=0.0)
    assert torch.equal(t, out)


@pytest.mark.parametrize("dense", [True, False])
def test_bias_gradient_of_very_many_rows(dev, dense):
    """Sums of values of one sign, whose rounding errors add up: the bound does not grow with
    the number of rows."""
    m, f = (1 << 18, 4096) if dense else (70000, 2048)
    d = float(np.float32(1.1))
    if dense:
        gu, dh = torch.full((m, 2 * f), 1.0, device=dev), torch.full((m, f), d, device=dev)
    else:
        gu = torch.full((m, 4 * f), 1.0, device=dev)[:, ::2]
        dh = torch.full((m, 2 * f), d, device=dev)[:, ::2]
    # relu at 1: both gradients are dh, exactly.  Of one sign, an addition's rounding is at most half
    # a step of the sum so far: seven of them in eight rows, then one each for the sums of a wave,
    # of a run and of all
    want, bound = m * d, 10.1 * H * m * d
    if dense:
        x, w = torch.zeros(m, 8, device=dev), torch.zeros(2 * f, 8, device=dev)
        _, _, db = mt.gated_linear_backward(dh, gu, x, w, act="relu", need_dw=False, dgu=gu)
        assert abs(db.double() - want).max().item() <= bound
        gu.fill_(1.0)
    db = torch.empty(2 * f, device=dev)
    ws = torch.empty(mt.lib().mt_gate_backward_bias_workspace_f32(m, f), dtype=torch.uint8, device=dev)
    R = lambda t: ctypes.byref(mt.mat(t))
    assert mt.lib().mt_gate_backward_bias_f32(R(dh), R(gu), ref.ACTS.index("relu"), R(gu), db.data_ptr(), 1, 0.0,
                                              ws.data_ptr(), ws.numel(),
                                              torch.cuda.current_stream().cuda_stream) == mt.MT_OK
    assert abs(db.double() - want).max().item() <= bound


def test_clip_grad_norm_needs_a_largest_norm(dev):
    x = torch.ones(4, 8, device=dev)
    with pytest.raises(ValueError):
        mt.clip_grad_norm([x], None)
    assert bool((x == 1).all())
    mt.clip_grad_norm([x], 0)
    assert bool((x == 0).all())


def scales_of_all_sizes(n, dev, turn):
    """n finite scales from 1e-40 to 1e37, in turn."""
    s = torch.tensor([1e-40, 2.0 ** -126, 1e-30, 1e-12, 0.75, 1e12, 1e18, 2e19, 1e30, 1e37], device=dev)
    return s[(torch.arange(n, device=dev) * turn) % 10] * (1 + torch.arange(n, device=dev) % 7 / 8)


@pytest.mark.parametrize("m,n,k", [(3, 40, 100), (40, 200, 64), (17, 16400, 100), (70, 8200, 96), (17, 18, 9743),
                                   (1000, 4000, 1104), (1900, 4000, 200), (2000, 4096, 336)])
def test_8_bit_products_of_any_finite_scales(dev, m, n, k):
    """Scales whose product leaves fp32's range where y does not: no digits lost, and zero where
    the sum is zero."""
    g = torch.Generator(device=dev).manual_seed(m)
    codes = lambda r: torch.randint(-128, 128, (r, k), dtype=torch.int8, device=dev, generator=g)
    x, w = mt.Q8Rows(codes(m), scales_of_all_sizes(m, dev, 1)), mt.Q8Rows(codes(n), scales_of_all_sizes(n, dev, 3))
    x.q[1], w.q[n - 2] = 0, 0
    assert bool(x.scale.isfinite().all()) and bool(w.scale.isfinite().all())
    want = torch.mm(x.q.double(), w.q.double().t().contiguous()) * torch.outer(x.scale.double(), w.scale.double())
    for y in (mt.linear_q8(x, w), mt.gated_linear(x, w, act="relu", keep=True).gu,
              mt.linear_q8(mt.Q8Rows(x.q[:2], x.scale[:2]), w)):
        t = want[:y.shape[0]]
        over = t.abs() >= 2.0 ** 128 - 2.0 ** 103
        assert bool((y[over] == torch.where(t > 0, float("inf"), float("-inf")).float()[over]).all())
        # the sum to fp32, the product with one scale, and with the other (of small y half a step)
        off = (y.double() - t).abs() - (3.01 * H * t.abs() + 2.0 ** -149)
        assert off[~over].max().item() <= 0
        assert bool((y[1] == 0).all()) and bool((y[:, n - 2] == 0).all())


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu", "sigmoid"])
def test_gradients_whose_factors_overflow_in_part(dev, act):
    """dH·U·act'(G) where dH·U is past fp32's range and the whole is not."""
    g = [-1.0, -3.0, -9.0, -12.0, -20.0, -40.0, -60.0, -80.0, 0.0, -1e4, -3e38]
    pairs = [(1e25, 1e25), (-3e20, 2e19), (2e38, -7.0), (3.0, 2e38), (1e12, 3e38), (3e38, 3e38), (1e-3, 1e-3)]
    gates = np.array(g * len(pairs), np.float32)
    dh, up = (np.repeat(np.array([p[i] for p in pairs], np.float32), len(g)) for i in (0, 1))
    gu = np.concatenate([gates, up])[None]
    want, bound = ref.gate_backward(act, dh[None], gu)
    fits = np.abs(want) < 2.0 ** 128 - 2.0 ** 103
    t, d = torch.from_numpy(gu).to(dev), torch.from_numpy(dh[None]).to(dev)
    got = mt.gate_backward(d, t, act).cpu().numpy().astype(np.float64)
    assert (np.abs(got - want)[fits] <= bound[fits]).all()
    assert (got[~fits] == np.copysign(np.inf, want[~fits])).all()
    strided = torch.stack([t, t], 2)[:, :, 0]
    assert np.array_equal(mt.gate_backward(d, strided, act).cpu().numpy().astype(np.float64), got)
