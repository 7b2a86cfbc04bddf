"""Sizes that reach each kernel of the low-bit products, with remainders in every direction, and
the kernel that each has to reach (checked without a GPU by test_lowbit_plans.py, run by
test_lowbit_variants_gpu.py); bounds that see whether an fp32 operand keeps all its bits."""
import ctypes

import numpy as np

import minitensor_amd as mt
from minitensor_amd.lowbit import LowbitPlan

# (8-bit rows, rows, outputs, inputs), column blocks of a workgroup
FEW = [((q8, m, n, k), nc)
       for q8, rows in ((False, (3, 5, 10, 16)), (True, (7, 16, 17, 32, 33, 48)))
       for m in rows
       for n, k, nc in ((1000, 1030, 1), (8200, 300, 2), (16400, 1030, 4 if m * (1 if q8 else 3) <= 32 else 2))]

# (8-bit rows, rows, outputs, inputs), splits of the 128 x 256 tile
WIDE = [((False, 2047, 2050, 33), 1), ((False, 2047, 2050, 300), 1), ((False, 1999, 4090, 1030), 1),
        ((False, 1000, 2050, 1030), 3), ((False, 129, 4090, 4101), 7), ((False, 2047, 257, 4101), 7),
        ((True, 2047, 2050, 33), 1), ((True, 2047, 2050, 300), 1), ((True, 1999, 4090, 1030), 1),
        ((True, 2047, 1030, 4101), 3), ((True, 1000, 2050, 4101), 3)]

# (rows, inputs, outputs), splits of the 128 x 256 tile of the weight gradient
BACK_WIDE = [((33, 4090, 2050), 1), ((300, 2050, 2050), 1), ((4101, 1030, 1020), 6),
             ((8195, 2050, 1020), 3), ((2050, 257, 4090), 4)]

# A product of one nonzero input and a whole number of eight bits: two matrix instructions whose
# sums take more than 24 bits (2^-23 each, they do not round to nearest), at most two fp32 roundings
# by a scale and in dY·scale (2^-24 each), and the parts' sums where they meet in fp32 (2^-24 each).
SINGLE = 2.0 ** -21

# 2-norm of a random product's error by that of the product: a group's sum passes 24 matrix
# instructions (128 inputs in three parts), each of which loses half an ulp on average of a sum
# that is two thirds of the group's on average: 24·2/3·2^-24 = 2^-20; the fp32 additions of the
# groups and splits, random, a quarter of that at most.
NORM = 1.25 * 2.0 ** -20


def q4_plan(q8, m, n, k, group):
    p = LowbitPlan()
    assert mt.lib().mt_linear_q4_plan(m, k, n, group, q8, ctypes.byref(p)) == mt.MT_OK
    return p


def back_plan(r, fin, fout):
    p = LowbitPlan()
    assert mt.lib().mt_linear_backward_q8_plan(r, fin, fout, ctypes.byref(p)) == mt.MT_OK
    return p


def parts(x):
    """The three bf16 parts of fp32 values, eight bits each, as the kernels take them."""
    x = np.asarray(x, np.float32)
    cut = lambda v: (v.view(np.uint32) & np.uint32(0xffff0000)).view(np.float32)  # noqa: E731
    h = cut(x)
    m = cut(x - h)
    return h, m, x - h - m
