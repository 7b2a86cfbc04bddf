"""Plain 64-bit forms of the operators of include/mtlowbit.h, for their tests."""
from __future__ import annotations

import numpy as np

EPS32 = 2.0 ** -24    # half an ulp of fp32, relative


def quantize_q8(x):
    """Codes and scales, step by step in fp32 as the header defines them."""
    x = np.asarray(x, np.float32)
    a = np.max(np.abs(x), axis=1) if x.shape[1] else np.zeros(x.shape[0], np.float32)
    scale = np.maximum(a * np.float32(1 / np.float32(127)), np.float32(2.0 ** -126))
    with np.errstate(all="ignore"):
        v = np.rint(x * (np.float32(1) / scale)[:, None])
    return np.nan_to_num(v, nan=0.0).astype(np.int8), scale


def quantize_q4(w, group):
    """(codes [N, K], scales [N, ceil(K/group)]), step by step in fp32."""
    w = np.asarray(w, np.float32)
    n, k = w.shape
    g = -(-k // group)
    pad = np.zeros((n, g * group), np.float32)
    pad[:, :k] = w
    pad = pad.reshape(n, g, group)
    scale = np.maximum(np.max(np.abs(pad), axis=2) * np.float32(1 / np.float32(7)),
                       np.float32(2.0 ** -126))
    with np.errstate(all="ignore"):
        v = np.rint(pad * (np.float32(1) / scale)[:, :, None])
    return np.nan_to_num(v, nan=0.0).astype(np.int8).reshape(n, g * group)[:, :k], scale


def pack_q4(code, filler=0):
    """uint8 [N, 16·ceil(K/32)] of codes -8..7; `filler` in the inputs past K."""
    n, k = code.shape
    full = np.full((n, -(-k // 32) * 32), filler, np.int64)
    full[:, :k] = code
    full &= 15
    return (full[:, 0::2] | (full[:, 1::2] << 4)).astype(np.uint8)


def weight_q4(code, scale, group):
    """code·scale [N, K] in 64 bits."""
    s = np.repeat(np.asarray(scale, np.float64), group, axis=1)[:, :code.shape[1]]
    return code.astype(np.float64) * s


def rms_norm(h, weight, eps):
    h = np.asarray(h, np.float64)
    rstd = 1 / np.sqrt(np.mean(h * h, axis=1) + eps)
    return h * rstd[:, None] * np.asarray(weight, np.float64), rstd


def rms_norm_backward(dy, h, weight, rstd, dh0=None):
    """(dh, dweight, bound of |dh| terms, sum |dy·xh|) from the same h and rstd."""
    dy, h, weight, rstd = (np.asarray(t, np.float64) for t in (dy, h, weight, rstd))
    xh = h * rstd[:, None]
    g = dy * weight
    c = np.mean(g * xh, axis=1, keepdims=True)
    dh = rstd[:, None] * (g - xh * c)
    size = np.abs(rstd)[:, None] * (np.abs(g) + np.abs(xh) * np.mean(np.abs(g * xh), axis=1,
                                                                     keepdims=True))
    if dh0 is not None:
        dh = dh + np.asarray(dh0, np.float64)
        size = size + np.abs(dh0)
    return dh, np.sum(dy * xh, axis=0), size, np.sum(np.abs(dy * xh), axis=0)


def linear_bound(k, group, parts):
    """Roundings on the way of a product's sum, each at most 2^-23 of the sum of the
    magnitudes (the matrix unit does not round to nearest): a group's matrix
    instructions (16 k and more each, `parts` products), an addition per group, and at
    most 64 waves or splits, the parts' sums, scale and bias after that."""
    return (parts * -(-min(group, max(k, 1)) // 16) + -(-k // group) + 64 + 8) * 2.0 ** -23
