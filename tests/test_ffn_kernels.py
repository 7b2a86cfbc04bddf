"""Every kernel that gated_linear and linear_q8 may take, by the queries of which one a call
does: sizes that land on each, with rows on multiples of four bytes and at odd ones, operands
contiguous along the inputs and across them, in one piece and in splits."""
import ctypes

import numpy as np
import pytest
import torch

import ffn_reference as ref
import minitensor_amd as mt
from minitensor_amd.ffn import GatePlan
from minitensor_amd.lowbit import Q8Plan

DIRECT, TILES = (0, 0), ((64, 128), (128, 128), (128, 256), (256, 256))

# rows, columns (gated: features), inputs
Q8 = [(1, 18, 17), (16, 300, 2000), (40, 31, 65), (1, 8191, 500), (2, 4392, 18), (16, 8190, 257), (17, 4090, 500),
      (30, 4093, 141), (147, 452, 16), (257, 511, 255), (36, 2863, 17), (513, 769, 640), (551, 470, 18),
      (20, 16380, 600), (95, 4185, 158), (17, 18, 9743), (167, 3303, 19), (403, 4821, 265), (73, 6480, 7239),
      (1444, 4555, 16), (92, 6585, 16486), (1454, 7730, 16), (908, 2740, 13836)]
Q8_GATED = [(1, 18, 17), (16, 300, 2000), (2, 16, 257), (1, 8191, 500), (17, 4090, 500), (189, 373, 16), (628, 104, 17),
            (257, 511, 255), (229, 663, 16), (20, 4373, 166), (31, 4205, 131), (17, 18, 6933), (1067, 229, 17),
            (398, 2523, 270), (82, 2735, 6979), (619, 5091, 17), (77, 2792, 21015), (665, 7502, 26),
            (484, 4166, 8459)]
# rows, features, inputs: in fp32 from operands contiguous along the inputs
F32 = [(1, 18, 18), (2, 17, 300), (3, 17, 257), (4, 33, 1030), (5, 20, 77), (8, 1030, 2061), (10, 18, 36),
       (16, 33, 1029), (12, 18, 19), (48, 77, 64), (257, 200, 65), (124, 2057, 16), (470, 470, 70), (166, 2967, 16),
       (513, 301, 1501)]
F32_TILES = [(347, 2052, 19), (131, 97, 3001), (1292, 2465, 17), (873, 20, 6625), (976, 3504, 113), (208, 2783, 1189)]


def q8_plan(m, n, k, gated):
    """(rows and columns of a tile, whether in splits, blocks of rows and columns without tiles)."""
    p = Q8Plan()
    f = mt.lib().mt_gated_linear_q8_plan if gated else mt.lib().mt_linear_q8_plan
    assert f(m, k, n, ctypes.byref(p)) == mt.MT_OK
    return (p.tile_rows, p.tile_cols), p.splits > 1, (p.row_blocks, p.column_blocks)


def gate_plan(m, f, k, across=(False, False)):
    """(kind, rows and columns of a tile, whether in splits, rows on the vector units)."""
    def d(r, c, t):
        return ctypes.byref(mt.MatF32(0x1000, 0, r, c, 1 if t else c, r if t else 1, 1, 0))
    p = GatePlan()
    assert mt.lib().mt_gated_linear_plan_f32(d(m, k, across[0]), d(2 * f, k, across[1]), ctypes.byref(p)) == mt.MT_OK
    return p.kind, (p.tile_rows, p.tile_cols), p.splits > 1, p.vector_rows


def test_sizes_reach_every_kernel():
    tiles = {(t, s, (0, 0)) for t in TILES for s in (False, True)}
    assert {q8_plan(*s, False) for s in Q8} == tiles | {
        (DIRECT, False, b) for b in ((1, 1), (2, 1), (1, 2), (2, 2), (4, 2), (2, 4))}
    assert {q8_plan(*s, True) for s in Q8_GATED} == tiles | {
        (DIRECT, False, b) for b in ((1, 2), (2, 2), (4, 2), (2, 4))}
    # (rows of 2^24 inputs and more have a kernel of their own)
    assert q8_plan(17, 18, (1 << 24) + 77, True) == (DIRECT, False, (1, 2))
    assert q8_plan(17, 18, (1 << 24) + 77, False) == (DIRECT, False, (1, 1))
    assert {gate_plan(*s) for s in F32} == {(0, (r, 0), False, 0) for r in (16, 32, 48)} | {
        (0, (0, 0), False, r) for r in (1, 2, 4, 8, 16)}
    for a in ((False, False), (True, False), (False, True), (True, True)):
        assert {gate_plan(*s, a) for s in F32_TILES} == {(1, t, s, 0) for t in TILES[:3] for s in (False, True)}, a


def normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def generator(*key):
    return torch.Generator(device="cuda").manual_seed(hash(key) & 0xffffffff)


def product(x, w):
    """x·wᵀ in 64 bits (whole numbers of 8 bits: exact)."""
    return torch.mm(x.double(), w.double().t().contiguous())


def np64(t):
    return t.detach().cpu().numpy().astype(np.float64)


def check(got, want, bound, what=""):
    got = np64(got)
    over = np.abs(got - want) - bound
    at = np.unravel_index(np.argmax(over), over.shape)
    assert over[at] <= 0, f"{what}: off by {abs(got - want)[at]:.3e} at {at}, bound {bound[at]:.3e}"


def rows8(g, r, k, how, scale):
    """Codes, -128 among them, with rows on multiples of 16 bytes, of 4, or at odd addresses."""
    four = (k + 3) // 4 * 4
    row = {"by 16": (k + 15) // 16 * 16, "by 4": four + 4 * (four % 16 == 0), "odd": k + 1 - k % 2}[how]
    wide = torch.full((r * row + 3,), 99, dtype=torch.int8, device="cuda")
    q = wide[3 if how == "odd" else 0:].as_strided((r, k), (row, 1))
    q.copy_(torch.randint(-128, 128, (r, k), dtype=torch.int8, device="cuda", generator=g))
    return mt.Q8Rows(q, (torch.rand(r, device="cuda", generator=g) + 0.1) * scale)


def bound_q8(x, w, b):
    """As ref.linear_q8: (y, bound)."""
    p = np64(product(x.q, w.q)) * np.outer(np64(x.scale), np64(w.scale))
    y = p if b is None else p + np64(b)
    return y, 3.01 * ref.H * np.abs(p) + 1.01 * ref.H * np.abs(y) + 2.0 ** -140


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", Q8)
def test_linear_q8_of_every_kernel(dev, m, n, k):
    g = generator(1, m, n, k)
    b = normal(g, n)
    for how in ("by 16", "by 4", "odd"):
        x, w = rows8(g, m, k, how, 1 / 64), rows8(g, n, k, how, 1 / 64)
        check(mt.linear_q8(x, w, b), *bound_q8(x, w, b), how)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", Q8_GATED)
def test_gated_linear_q8_of_every_kernel(dev, m, n, k):
    g = generator(2, m, n, k)
    b = normal(g, 2 * n)
    for how in ("by 16", "by 4", "odd"):
        # (projections of order one: codes of 74 rms)
        x, w = rows8(g, m, k, how, 1 / 74), rows8(g, 2 * n, k, how, 1 / 74 / k ** 0.5)
        gu, e = bound_q8(x, w, b)
        r = mt.gated_linear(x, w, b, keep=True)
        check(r.gu, gu, e, how)
        check(r.h, *ref.gate("silu", gu, e), how)
        assert torch.equal(mt.gated_linear(x, w, b).h, r.h), how


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["by 16", "odd"])
def test_gated_linear_q8_of_long_rows(dev, how):
    m, n, k = 17, 18, (1 << 24) + 77
    g = generator(3, m)
    x, w = rows8(g, m, k, how, 1 / 74), rows8(g, 2 * n, k, how, 1 / 74 / k ** 0.5)
    gu, e = bound_q8(x, w, None)
    r = mt.gated_linear(x, w, keep=True)
    check(r.gu, gu, e)
    check(r.h, *ref.gate("silu", gu, e))
    check(mt.linear_q8(x, w), gu, e)


ACROSS = [(False, False), (True, False), (False, True), (True, True)]


def laid(t, across):
    return t.t().contiguous().t() if across else t


@pytest.mark.gpu
@pytest.mark.parametrize("m,f,k", F32 + F32_TILES)
def test_gated_linear_of_one_input_a_row(dev, m, f, k):
    """One nonzero input a row, each input in turn: a projection is one product.  It is off by
    the three parts that are left out, 2^-24 of it, and by roundings of 2^-24 of it and less
    (gemm_split.hpp; on the fp32 units by one): a part more lost, 2^-17 of it, would show."""
    g = generator(4, m, f, k)
    at = torch.randperm(k, device=dev, generator=g).repeat(m // k + 1)[:m]
    v, w = normal(g, m), normal(g, 2 * f, k)
    x = torch.zeros(m, k, device=dev)
    x[torch.arange(m, device=dev), at] = v
    want = v.double()[:, None] * w.double().t()[at]
    for a in ACROSS if (m, f, k) in F32_TILES else ACROSS[:1]:
        r = mt.gated_linear(laid(x, a[0]), laid(w, a[1]), keep=True)
        over = ((r.gu.double() - want).abs() - 2.0 ** -22 * want.abs()).max().item()
        assert over <= 0, (a, over)
        assert torch.equal(mt.gated_linear(laid(x, a[0]), laid(w, a[1])).h, r.h)


@pytest.mark.gpu
@pytest.mark.parametrize("m,f,k", F32_TILES)
def test_gated_linear_of_every_tile(dev, m, f, k):
    g = generator(5, m, f, k)
    x, w, b = normal(g, m, k), normal(g, 2 * f, k) / k ** 0.5, normal(g, 2 * f)
    gu = np64(product(x, w)) + np64(b)
    e = (6 * -(-k // 16) + 70) * 2.0 ** -23 * (np64(product(x.abs(), w.abs())) + np.abs(np64(b)))   # (ref.linear)
    h, he = ref.gate("silu", gu, e)
    for a in ACROSS:
        r = mt.gated_linear(laid(x, a[0]), laid(w, a[1]), b, keep=True)
        check(r.gu, gu, e, a)
        check(r.h, h, he, a)


@pytest.mark.gpu
@pytest.mark.parametrize("m,f,k", F32_TILES)
def test_gated_linear_of_infinities_in_every_tile(dev, m, f, k):
    """A tile with an infinity, a NaN or a value past bf16's range among its operands is taken
    again in fp32: what the formula gives, and the rows and columns beside it as they are."""
    g = generator(6, m, f, k)
    x, w = normal(g, m, k), normal(g, 2 * f, k) / k ** 0.5
    x[2, 5], w[7, 11], w[f + 10, 3] = float("inf"), float("-inf"), float("nan")
    x[m - 1, 7], w[:, 7] = torch.finfo(torch.float32).max, 2e-38 * torch.sign(w[:, 7])
    want = product(x, w)
    sizes = product(x.abs().nan_to_num(0, 0, 0), w.abs().nan_to_num(0, 0, 0))
    e = (6 * -(-k // 16) + 70) * 2.0 ** -23 * sizes
    fine = want.isfinite()
    assert int((~fine).sum()) == 2 * f + 2 * (m - 1)
    for a in ACROSS:
        gu = mt.gated_linear(laid(x, a[0]), laid(w, a[1]), act="relu", keep=True).gu
        assert torch.equal(gu.isnan(), want.isnan()) and torch.equal(gu.isinf(), want.isinf()), a
        assert torch.equal(gu.sign()[want.isinf()].double(), want.sign()[want.isinf()]), a
        assert bool(((gu.double() - want).abs()[fine] <= e[fine]).all()), a
