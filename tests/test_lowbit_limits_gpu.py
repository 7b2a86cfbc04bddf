"""The operators of include/mtlowbit.h at the ends of their ranges: rows of no columns,
finite values whose parts or factors leave fp32's range, very wide rows, arguments that are
refused.  Bounds: tests/lowbit_reference.py."""
import numpy as np
import pytest
import torch

import lowbit_reference as ref
import lowbit_variants as var
import minitensor_amd as mt

pytestmark = pytest.mark.gpu

FLT_MAX = np.finfo(np.float32).max


def rng(*key):
    return np.random.default_rng([int(k) for k in key])


def gpu(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def cpu(t):
    return t.detach().cpu().numpy()


def near(y, x, w, group, parts):
    """y against x·wᵀ in 64 bits, all of them finite."""
    want, size = x @ w.T, np.abs(x) @ np.abs(w).T
    y = cpu(y).astype(np.float64)
    assert np.isfinite(y).all()
    assert np.all(np.abs(y - want) <= ref.linear_bound(x.shape[1], group, parts) * size + 1e-44)


@pytest.mark.parametrize("r", [1, 5, 300])
def test_rows_of_no_columns(dev, r):
    """[R, 0]: the scale of an empty row is the smallest one, its mean square zero."""
    junk = [torch.full((r,), 7.0, device=dev) for _ in range(8)]
    del junk                          # (what the outputs below would hold if left unwritten)
    x = torch.empty(r, 0, device=dev)
    assert bool((mt.quantize_q8(x).scale == 2.0 ** -126).all())
    out = mt.Q8Rows(torch.empty(r, 0, dtype=torch.int8, device=dev), torch.full((r,), 7.0, device=dev))
    mt.quantize_q8(x, out=out)
    assert bool((out.scale == 2.0 ** -126).all())
    assert mt.dequantize_q8(out).shape == (r, 0)
    for q8 in (False, True):
        junk = [torch.full((r,), 7.0, device=dev) for _ in range(8)]
        del junk
        n = mt.rms_norm(x, torch.empty(0, device=dev), residual=x, eps=0.25, q8=q8)
        assert bool((n.rstd == 2.0).all()) and n.y.shape == n.h.shape == (r, 0)
        assert not q8 or bool((n.q8.scale == 2.0 ** -126).all())


@pytest.mark.parametrize("m,n,k,group", [(2, 40, 300, 64), (16, 33, 260, 128), (80, 70, 300, 32),
                                         (130, 140, 257, 128)])
def test_linear_q4_of_the_largest_inputs(dev, m, n, k, group):
    """One input per row past the largest bf16 value, some of its codes zero: finite
    products of finite values."""
    g = rng(1, m, n, k, group)
    code = g.integers(-8, 8, (n, k)).astype(np.int8)
    scale = (1e-3 * (g.random((n, -(-k // group))) + 0.5)).astype(np.float32)
    x = g.standard_normal((m, k)).astype(np.float32)
    for i in range(m):
        x[i, (7 * i + 3) % k] = (FLT_MAX, -FLT_MAX, 3.397e38, -3.4e38, 3.39e38)[i % 5]
    code[:, 3], code[0, 3] = 7, 0
    wq = mt.Q4Weight(gpu(ref.pack_q4(code), dev), gpu(scale, dev), k, group)
    near(mt.linear_q4(gpu(x, dev), wq), x.astype(np.float64), ref.weight_q4(code, scale, group), group, 3)


@pytest.mark.parametrize("r,fin,fout", [(50, 64, 40), (300, 130, 70)])
def test_linear_backward_q8_of_the_largest_gradients(dev, r, fin, fout):
    g = rng(2, r)
    q = g.integers(-1, 2, (r, fin)).astype(np.int8)
    s = np.ones(r, np.float32)
    dy = g.standard_normal((r, fout)).astype(np.float32)
    dy[5, 3], dy[6, 4], dy[r - 1, 39], dy[7, 0] = FLT_MAX, -FLT_MAX, 3.397e38, 3.39e38
    _, dw, _ = mt.linear_backward_q8(gpu(dy, dev), mt.Q8Rows(gpu(q, dev), gpu(s, dev)))
    near(dw, dy.T.astype(np.float64), q.T.astype(np.float64), 128, 3)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 3, 16, 80, 200])
def test_linear_q4_of_the_largest_weights(dev, m, group):
    """A group near 3e38 and its scale: finite products of finite values, and zero where
    the group's codes are."""
    g = rng(3, m, group)
    n, k = 50, 200
    w = g.standard_normal((n, k)).astype(np.float32)
    w[3, :128] *= 1e38
    w[3, 5], w[20, 131] = 3e38, -3.3e38
    x = (1e-4 * g.standard_normal((m, k))).astype(np.float32)
    wq = mt.quantize_q4(gpu(w, dev), group)
    wd = cpu(mt.dequantize_q4(wq)).astype(np.float64)
    assert np.isfinite(wd).all()
    near(mt.linear_q4(gpu(x, dev), wq), x.astype(np.float64), wd, group, 3)
    # any finite scale; rows in 8 bits too, one input of each sign in a group
    code = np.zeros((n, k), np.int8)
    code[:, 5], code[:, 150] = 1, -1
    scale = np.full((n, -(-k // group)), 1.5e38, np.float32)
    code[7] = 0
    wq = mt.Q4Weight(gpu(ref.pack_q4(code), dev), gpu(scale, dev), k, group)
    wd = ref.weight_q4(code, scale, group)
    near(mt.linear_q4(gpu(x, dev), wq), x.astype(np.float64), wd, group, 3)
    q = g.integers(-1, 2, (m, k)).astype(np.int8)
    y = mt.linear_q4(mt.Q8Rows(gpu(q, dev), torch.full((m,), 0.5, device=dev)), wq)
    near(y, 0.5 * q, wd, group, 1)


@pytest.mark.parametrize("c", [(1 << 24) + 5, (1 << 26) + 37])
def test_rms_norm_backward_of_very_wide_rows(dev, c):
    """The weight gradient's sum takes its columns in several rounds from 2^24 of them on (a
    grid's threads are a 32-bit number)."""
    g = torch.Generator(device=dev).manual_seed(c)
    dy, h = (torch.randn(2, c, device=dev, generator=g) for _ in range(2))
    rstd = torch.tensor([0.5, 2.0], device=dev)
    dw0 = torch.randn(c, device=dev, generator=g)
    dw = dw0.clone()
    mt.rms_norm_backward(dy, h, None, rstd, need_dh=False, dw=dw, beta=0.5)
    # a product, its row's 1/rms, the two rows' sum, the old gradient's share
    for a in range(0, c, 1 << 24):
        s = slice(a, a + (1 << 24))
        terms = dy[:, s].double() * h[:, s].double() * rstd.double()[:, None]
        want = terms.sum(0) + 0.5 * dw0[s].double()
        size = terms.abs().sum(0) + 0.5 * dw0[s].double().abs()
        assert bool(((dw[s].double() - want).abs() <= 6 * ref.EPS32 * size).all())


def test_a_place_for_dx_needs_the_weight(dev):
    """linear_backward_q8 gives dX from the weight alone: a dx to write to without one is
    refused, not left as it was."""
    dy, xq = torch.ones(4, 8, device=dev), mt.quantize_q8(torch.ones(4, 16, device=dev))
    dx = torch.full((4, 16), 5.0, device=dev)
    with pytest.raises(ValueError):
        mt.linear_backward_q8(dy, xq, dx=dx)


@pytest.mark.parametrize("r,fin,fout", [(20000, 4096, 2048), (20000, 70, 100)])
def test_linear_backward_q8_bias_gradient_of_many_rows(dev, r, fin, fout):
    """Rows of one sign and one value an output, whose additions all round the same way: a sum of
    eight rows (3 roundings), a compensated one over those (2, and 1 at its end), four groups
    (2), the splits (at most 32 of them) and what the compensation itself rounds (1)."""
    a = torch.linspace(1, 2, fout, device=dev)
    dy = a.expand(r, fout).contiguous()
    xq = mt.Q8Rows(torch.zeros(r, fin, dtype=torch.int8, device=dev), torch.ones(r, device=dev))
    _, dw, db = mt.linear_backward_q8(dy, xq)
    assert bool((dw == 0).all())
    want = r * a.double()
    split = mt.lib().mt_linear_backward_q8_workspace_f32(r, fin, fout) > 0 and fin < 4096
    assert bool(((db.double() - want).abs() <= (9 + 32 * split) * ref.EPS32 * want).all())


def smallest(dev, key, n, k):
    """[n, k], in each row one value from 2^-149 to 2^-100 with all its bits; it, its column."""
    g = torch.Generator(device=dev).manual_seed(key)
    e = torch.arange(n, device=dev) % 50 - 149
    v = ((1 + torch.rand(n, device=dev, generator=g)).double() * 2.0 ** e.double()).float()
    at = (torch.arange(n, device=dev) * 37 + 11) % k
    x = torch.zeros(n, k, device=dev)
    x[torch.arange(n, device=dev), at] = v
    return x, v.double(), at


@pytest.mark.parametrize("scale", [1.0, 2.0 ** 60])
@pytest.mark.parametrize("m,n,k,group", [(16, 64, 300, 64), (100, 130, 300, 128), (100, 130, 300, 32),
                                         (2047, 2050, 300, 128)])
def test_linear_q4_of_the_smallest_inputs(dev, m, n, k, group, scale):
    """To the nearest multiple of 2^-133, subnormal ones too; the product's roundings
    (lowbit_variants.SINGLE), and a subnormal sum's (2^-146: half of 2^-145)."""
    x, v, at = smallest(dev, m, m, k)
    code = rng(8, n, k).integers(-8, 8, (n, k)).astype(np.int8)
    s = np.full((n, -(-k // group)), scale, np.float32)
    wq = mt.Q4Weight(gpu(ref.pack_q4(code), dev), gpu(s, dev), k, group)
    w = gpu(ref.weight_q4(code, s, group), dev)[:, at].t()
    want = v[:, None] * w
    err = (mt.linear_q4(x, wq).double() - want).abs()
    assert bool((err <= 2.0 ** -134 * w.abs() + var.SINGLE * want.abs() + 2.0 ** -146).all())


@pytest.mark.parametrize("r,fin,fout", [(300, 130, 70), (300, 2050, 2050)])
def test_linear_backward_q8_of_the_smallest_gradients(dev, r, fin, fout):
    x, v, at = smallest(dev, r + fin, fout, r)
    q = gpu(rng(9, r, fin).integers(-128, 128, (r, fin)).astype(np.int8), dev)
    _, dw, _ = mt.linear_backward_q8(x.t().contiguous(), mt.Q8Rows(q, torch.ones(r, device=dev)))
    want = v[:, None] * q[at].double()
    err = (dw.double() - want).abs()
    assert bool((err <= 2.0 ** -134 * q[at].double().abs() + var.SINGLE * want.abs() + 2.0 ** -149).all())
