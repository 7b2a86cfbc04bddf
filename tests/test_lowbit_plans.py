"""Which kernel the low-bit products take, without a GPU: the sizes of lowbit_variants.py reach the
ones that they are there for, whatever the planner's prices become; and the bounds that those are
checked with see a part of an fp32 operand that is left out."""
import ctypes

import numpy as np
import pytest

import lowbit_variants as var
import minitensor_amd as mt
from minitensor_amd.lowbit import LowbitPlan


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("case,columns", var.FEW)
def test_few_rows(case, columns, group):
    p = var.q4_plan(*case, group)
    assert (p.tile_rows, p.splits, p.column_blocks) == (0, 1, columns)


@pytest.mark.parametrize("group", [64, 128])
@pytest.mark.parametrize("case,splits", var.WIDE)
def test_wide_tile(case, splits, group):
    p = var.q4_plan(*case, group)
    assert p.tile_rows == 128 and (p.splits > 1) == (splits > 1) and p.column_blocks == 0


@pytest.mark.parametrize("case,splits", var.BACK_WIDE)
def test_wide_tile_of_the_weight_gradient(case, splits):
    p = var.back_plan(*case)
    assert p.tile_rows == 128 and (p.splits > 1) == (splits > 1)


def test_groups_of_32_take_the_narrow_tile():
    for q8 in (False, True):
        assert var.q4_plan(q8, 2047, 2050, 300, 32).tile_rows == 64
        assert var.q4_plan(q8, 80, 130, 300, 64).tile_rows == 64


def test_plan_queries_refuse():
    p, lib = LowbitPlan(), mt.lib()
    for args in ((0, 64, 64, 32, 0), (4, 0, 64, 32, 0), (4, 64, 0, 32, 0), (4, 64, 64, 48, 0),
                 (1 << 31, 64, 64, 32, 0), (4, 64, 1 << 26, 32, 0)):
        assert lib.mt_linear_q4_plan(*args, ctypes.byref(p)) == mt.MT_ERR_INVALID
    assert lib.mt_linear_q4_plan(4, 64, 64, 32, 0, None) == mt.MT_ERR_INVALID
    assert lib.mt_linear_backward_q8_plan(4, 64, 0, ctypes.byref(p)) == mt.MT_ERR_INVALID
    assert lib.mt_linear_backward_q8_plan(4, 64, 4, None) == mt.MT_ERR_INVALID


def test_the_parts_hold_every_bit():
    g = np.random.default_rng(1)
    bits = g.integers(0x0d000000, 0x7f800000, 200000).astype(np.uint32)   # from 2^-102 on
    x = np.concatenate([bits, bits | 0x80000000, [0x7f7fffff, 0x7f7f8000, 0]]).astype(np.uint32).view(np.float32)
    h, m, l = var.parts(x)
    assert np.isfinite(h).all()
    assert np.array_equal(h.astype(np.float64) + m + l, x.astype(np.float64))
    for v in (h, m, l):                                   # each a bf16 value
        assert np.all(v.view(np.uint32) & 0xffff == 0)


def test_the_bounds_see_a_part_left_out():
    g = np.random.default_rng(2)
    x = (g.standard_normal((64, 512)) * 2.0 ** g.integers(-20, 20, (64, 512))).astype(np.float32)
    h, m, _ = var.parts(x)
    two = h.astype(np.float64) + m
    assert np.mean(np.abs(two - x) > var.SINGLE * np.abs(x)) > 0.9
    x = g.standard_normal((64, 512)).astype(np.float32)
    h, m, _ = var.parts(x)
    w = g.integers(-8, 8, (512, 48)).astype(np.float64)
    want, got = x.astype(np.float64) @ w, (h.astype(np.float64) + m) @ w
    assert np.linalg.norm(got - want) > 4 * var.NORM * np.linalg.norm(want)
    # (rounded to nearest, as parts might be cut as well)
    near = lambda v: ((v.view(np.uint32) + 0x7fff + (v.view(np.uint32) >> 16 & 1))   # noqa: E731
                      & np.uint32(0xffff0000)).view(np.float32)
    h = near(x)
    two = h.astype(np.float64) + near(x - h)
    assert np.mean(np.abs(two - x) > var.SINGLE * np.abs(x)) > 0.5
