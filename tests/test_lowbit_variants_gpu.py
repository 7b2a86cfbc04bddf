"""Every kernel of the low-bit products at sizes with remainders in every direction
(lowbit_variants.py), against 64 bits: random operands, strides, infinities and the largest
values, and products of a single input, in which every bit of an fp32 operand shows."""
import pytest
import torch

import lowbit_reference as ref
import lowbit_variants as var
import minitensor_amd as mt

pytestmark = pytest.mark.gpu

NARROW = [((False, 80, 130, 300), 1), ((False, 200, 1000, 2047), 1), ((True, 80, 130, 300), 1)]


def generator(dev, *key):
    return torch.Generator(device=dev).manual_seed(hash(key) % (1 << 31))


def weight(dev, g, n, k, group, size=0.125):
    """(Q4Weight with every code and anything past K, the weight in 64 bits)."""
    full = torch.randint(-8, 8, (n, (k + 31) // 32 * 32), device=dev, generator=g)
    scale = (torch.rand(n, (k + group - 1) // group, device=dev, generator=g) + 0.5) * size
    packed = ((full[:, 0::2] & 15) | ((full[:, 1::2] & 15) << 4)).to(torch.uint8)
    w = full[:, :k].double() * scale.double().repeat_interleave(group, 1)[:, :k]
    return mt.Q4Weight(packed, scale, k, group), w


def rows_q8(dev, g, m, k):
    q = torch.randint(-128, 128, (m, k), device=dev, generator=g).to(torch.int8)
    s = torch.rand(m, device=dev, generator=g) + 0.5
    return mt.Q8Rows(q, s), q.double() * s.double()[:, None]


def rows(dev, g, q8, m, k):
    if q8:
        return rows_q8(dev, g, m, k)
    x = torch.randn(m, k, device=dev, generator=g)
    return x, x.double()


def check(y, x, w, group, parts, bias=None):
    want, size = x @ w.t(), x.abs() @ w.abs().t()
    err = (y.double() - want) if bias is None else (y.double() - want - bias.double())
    if bias is not None:
        size = size + bias.double().abs()
    assert bool((err.abs() <= ref.linear_bound(x.shape[1], group, parts) * size + 1e-44).all())
    if bias is None and x.shape[1] > 100:
        assert float(err.norm()) <= var.NORM * float(want.norm())


def q4_cases(listed, groups):
    return [(*case, group) for case, _ in listed for group in groups]


ALL_Q4 = (q4_cases(var.FEW, (32, 64, 128)) + q4_cases(var.WIDE, (64, 128))
          + q4_cases(NARROW, (32, 64, 128)))


@pytest.mark.parametrize("q8,m,n,k,group", ALL_Q4)
def test_linear_q4(dev, q8, m, n, k, group):
    g = generator(dev, 1, q8, m, n, k, group)
    wq, w = weight(dev, g, n, k, group)
    x, xd = rows(dev, g, q8, m, k)
    y = mt.linear_q4(x, wq)
    check(y, xd, w, group, 1 if q8 else 3)
    assert torch.equal(y, mt.linear_q4(x, wq))
    b = torch.randn(n, device=dev, generator=g)
    check(mt.linear_q4(x, wq, b), xd, w, group, 1 if q8 else 3, b)


STRIDED = [(False, 10, 16400, 300, 64), (False, 16, 8200, 300, 32), (True, 17, 16400, 300, 64),
           (True, 48, 8200, 300, 32), (False, 2047, 2050, 300, 64), (True, 2047, 2050, 300, 64),
           (False, 1000, 2050, 1030, 128), (True, 1000, 2050, 4101, 64)]


@pytest.mark.parametrize("q8,m,n,k,group", STRIDED)
def test_linear_q4_strides(dev, q8, m, n, k, group):
    """x transposed (8-bit rows: at an odd byte of wider ones), y transposed, every third element
    of a bias, rows of a larger weight."""
    g = generator(dev, 2, q8, m, n, k, group)
    wq, w = weight(dev, g, n + 3, k, group)
    part = mt.Q4Weight(wq.packed[3:], wq.scale[3:], k, group)
    x, xd = rows(dev, g, q8, m, k)
    if q8:
        wide = torch.zeros(m, k + 9, dtype=torch.int8, device=dev)
        wide[:, 5:5 + k] = x.q
        x = mt.Q8Rows(wide[:, 5:5 + k], x.scale)
    else:
        x = x.t().contiguous().t()
    out = torch.full((n + 2, m), 7.0, device=dev)
    b = torch.randn(n, 3, device=dev, generator=g)[:, 1]
    y = mt.linear_q4(x, part, b, out=out[1:1 + n].t())
    check(y, xd, w[3:], group, 1 if q8 else 3, b)
    assert bool((out[0] == 7).all()) and bool((out[-1] == 7).all())


@pytest.mark.parametrize("m,n,k,group", [(5, 1000, 300, 32), (5, 8200, 300, 64), (10, 16400, 300, 128),
                                         (16, 8200, 1030, 64), (80, 130, 300, 32),
                                         (2047, 2050, 300, 64), (1000, 2050, 1030, 128)])
def test_linear_q4_infinities_and_largest_values(dev, m, n, k, group):
    g = generator(dev, 3, m, n, k, group)
    wq, w = weight(dev, g, n, k, group, size=1e-3)
    x = torch.randn(m, k, device=dev, generator=g)
    x[0, 7], x[1, k - 1], x[2, 5] = float("inf"), float("-inf"), float("nan")
    x[3, 40], x[m - 1, k - 2] = torch.finfo(torch.float32).max, -3.397e38
    xd = x.double()
    want = xd @ w.t()
    y = mt.linear_q4(x, wq).double()
    assert torch.equal(y.isnan(), want.isnan())
    inf = want.isinf()
    assert torch.equal(y.isinf(), inf) and torch.equal(y[inf], want[inf])
    fine = [r for r in range(m) if r > 2]
    check(y[fine], xd[fine], w, group, 3)


SINGLES = [(1, 64, 300), (2, 100, 1030), (5, 1000, 300), (10, 1000, 300), (16, 1000, 300),
           (5, 8200, 300), (16, 8200, 300), (5, 16400, 300), (10, 16400, 300), (80, 130, 300),
           (200, 1000, 2047), (2047, 2050, 300), (1000, 2050, 1030)]


def one_value_each(dev, g, n, k):
    """[n, k], in each row one value, with all its bits and of any size; its column."""
    at = (torch.arange(n, device=dev) * 37 + 11) % k
    v = torch.randn(n, device=dev, generator=g) * 2.0 ** torch.randint(-20, 20, (n,), device=dev,
                                                                       generator=g)
    x = torch.zeros(n, k, device=dev)
    x[torch.arange(n, device=dev), at] = v
    return x, v.double(), at


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", SINGLES)
def test_linear_q4_keeps_every_bit(dev, m, n, k, group):
    g = generator(dev, 4, m, n, k, group)
    wq, w = weight(dev, g, n, k, group)
    x, v, at = one_value_each(dev, g, m, k)
    want = v[:, None] * w[:, at].t()
    y = mt.linear_q4(x, wq).double()
    assert bool(((y - want).abs() <= var.SINGLE * want.abs()).all())


def back_operands(dev, g, r, fin, fout):
    xq, x = rows_q8(dev, g, r, fin)
    return torch.randn(r, fout, device=dev, generator=g), xq, x


@pytest.mark.parametrize("r,fin,fout", [c for c, _ in var.BACK_WIDE])
def test_linear_backward_q8(dev, r, fin, fout):
    g = generator(dev, 5, r, fin, fout)
    dy, xq, x = back_operands(dev, g, r, fin, fout)
    _, dw, db = mt.linear_backward_q8(dy, xq)
    check(dw, dy.double().t(), x.t(), 128, 3)
    sums, size = dy.double().sum(0), dy.double().abs().sum(0)
    assert bool(((db.double() - sums).abs() <= (9 + 32) * ref.EPS32 * size).all())
    # added to the old ones, dW at strides, dY transposed, rows at an odd byte
    wide = torch.zeros(r, fin + 9, dtype=torch.int8, device=dev)
    wide[:, 3:3 + fin] = xq.q
    old = torch.randn(fin, fout, device=dev, generator=g)
    olb = torch.randn(fout, 2, device=dev, generator=g)
    dw2, db2 = old.clone().t(), olb.clone()[:, 1]
    mt.linear_backward_q8(dy.t().contiguous().t(), mt.Q8Rows(wide[:, 3:3 + fin], xq.scale), dw=dw2,
                          db=db2, beta_w=0.5, beta_b=-2.0)
    want = dy.double().t() @ x + 0.5 * old.double().t()
    wsize = dy.double().abs().t() @ x.abs() + 0.5 * old.double().abs().t()
    assert bool(((dw2.double() - want).abs() <= ref.linear_bound(r, 128, 3) * wsize).all())
    assert bool(((db2.double() - sums + 2 * olb[:, 1].double()).abs()
                 <= (9 + 32 + 2) * ref.EPS32 * (size + 2 * olb[:, 1].double().abs())).all())
    again = mt.linear_backward_q8(dy, xq)
    assert torch.equal(dw, again[1]) and torch.equal(db, again[2])


@pytest.mark.parametrize("r,fin,fout", [(300, 130, 70), (4096, 64, 64), (300, 2050, 2050),
                                        (8195, 2050, 1020)])
def test_linear_backward_q8_keeps_every_bit(dev, r, fin, fout):
    g = generator(dev, 6, r, fin, fout)
    xq, _ = rows_q8(dev, g, r, fin)
    dyt, v, at = one_value_each(dev, g, fout, r)
    _, dw, db = mt.linear_backward_q8(dyt.t().contiguous(), xq)
    want = (v * xq.scale.double()[at])[:, None] * xq.q[at].double()
    assert bool(((dw.double() - want).abs() <= var.SINGLE * want.abs()).all())
    assert torch.equal(db.double(), v)


def test_linear_backward_q8_infinities_and_largest_gradients_on_wide_tiles(dev):
    r, fin, fout = 300, 2050, 2050
    g = generator(dev, 7)
    q = torch.randint(-1, 2, (r, fin), device=dev, generator=g).to(torch.int8)
    dy = torch.randn(r, fout, device=dev, generator=g)
    dy[5, 3], dy[6, 4], dy[299, 2049] = torch.finfo(torch.float32).max, -3.397e38, 3.39e38
    dy[7, 0], dy[9, 1] = float("inf"), float("nan")
    _, dw, db = mt.linear_backward_q8(dy, mt.Q8Rows(q, torch.ones(r, device=dev)))
    want = dy.double().t() @ q.double()
    assert torch.equal(dw.isnan(), want.isnan())
    assert torch.equal(dw[0][dw[0].isinf()].double(), want[0][want[0].isinf()])
    check(dw[2:], dy[:, 2:].double().t(), q.double().t(), 128, 3)
    assert bool(db[0] == float("inf")) and bool(db[1].isnan()) and bool(db[2:].isfinite().all())
