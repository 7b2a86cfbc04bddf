"""Plain 64-bit forms of the operators of include/mtffn.h and of mt_linear_q8, and what
their fp32 results may be off by."""
from __future__ import annotations

import math

import numpy as np

H = 2.0 ** -24        # half a step of fp32, relative
ACTS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")

_erfc = np.vectorize(math.erfc, otypes=[np.float64])


def act(name, a):
    """(act(a), act'(a), the parts that rounding acts on).  act(a) = a·t(a) (sigmoid: t(a)):
    parts = (|act|, |a|·|d act/d t|·|a·t'(a)| / |a|), see act_bound."""
    a = np.asarray(a, np.float64)
    c = math.sqrt(2 / math.pi)
    with np.errstate(over="ignore", invalid="ignore"):
        if name == "relu":
            return np.maximum(a, 0), (a > 0).astype(np.float64), np.zeros_like(a)
        if name in ("silu", "sigmoid"):
            t = np.where(a < 0, np.exp(np.minimum(a, 0)) / (1 + np.exp(-np.abs(a))),
                         1 / (1 + np.exp(-np.abs(a))))
            p = np.exp(-np.abs(a)) / (1 + np.exp(-np.abs(a))) ** 2
            if name == "sigmoid":
                return t, p, np.zeros_like(a)
            return a * t, t + a * p, np.abs(a * p)
        if name == "gelu":
            t = 0.5 * _erfc(-a / math.sqrt(2))
            p = np.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)
            return a * t, t + a * p, np.abs(a * p)
        z = 2 * c * (a + 0.044715 * a ** 3)
        e = np.exp(-np.abs(z))
        t = np.where(z < 0, e / (1 + e), 1 / (1 + e))
        p = e / (1 + e) ** 2 * 2 * c * (1 + 3 * 0.044715 * a * a)
        return a * t, t + a * p, np.abs(a * p)


def act_bound(name, a):
    """How far an fp32 act(a) and act'(a) may be off for an exact a: 16 half steps of the
    value (exp or erfc 2 ulp, a sum, a reciprocal of 1 ulp, two products), and of t's argument
    8 half steps: a·t'(a) each, times a in act; the slope's second term is a·p(a), whose p
    (a Gaussian, or t(1-t)) changes with the argument's error as much again as |a|^2·p."""
    v, d, ap = act(name, a)
    a = np.abs(np.asarray(a, np.float64))
    tiny = 2.0 ** -125                       # results below fp32's normal range
    if name == "relu":
        return np.zeros_like(a), np.zeros_like(a)
    if name == "sigmoid":
        return 16 * H * np.abs(v) + tiny, 24 * H * np.abs(d) + tiny
    grow = a if name != "gelu_tanh" else 2 * a * (1 + 3 * 0.044715 * a * a)
    return (16 * H * np.abs(v) + 8 * H * a * ap + tiny * (1 + a),
            24 * H * (np.abs(d) + ap) + 8 * H * (ap + ap * a * (1 + grow)) + tiny * (1 + a))


def gate(name, gu, dgu=0.0):
    """(h, bound) of projections that are themselves off by dgu."""
    f = gu.shape[1] // 2
    g, u = np.asarray(gu[:, :f], np.float64), np.asarray(gu[:, f:], np.float64)
    e = np.broadcast_to(np.asarray(dgu, np.float64), gu.shape)
    v, d, _ = act(name, g)
    # |act''| <= 1.2 for all of them: the slope within the error of g
    dv = act_bound(name, g)[0] + (np.abs(d) + 1.2 * e[:, :f]) * e[:, :f]
    if name == "relu":
        dv = e[:, :f]                        # (slope 0 or 1)
    bound = dv * np.abs(u) + np.abs(v) * e[:, f:] + dv * e[:, f:]
    return v * u, bound + 2 * H * np.abs(v * u) + 2.0 ** -148


def gate_backward(name, dh, gu):
    """(dgu, bound) of exact projections."""
    f = gu.shape[1] // 2
    g, u, dh = (np.asarray(t, np.float64) for t in (gu[:, :f], gu[:, f:], dh))
    v, d, _ = act(name, g)
    bv, bd = act_bound(name, g)
    want = np.concatenate([dh * u * d, dh * v], 1)
    bound = np.concatenate([np.abs(dh * u) * bd, np.abs(dh) * bv], 1)
    return want, bound + 4 * H * np.abs(want) + 2.0 ** -140


def linear_q8(q, s, w, ws, b=None):
    """(y, bound): the whole sum once to fp32, the scales' product, their product, the bias."""
    total = q.astype(np.float64) @ w.astype(np.float64).T
    p = total * np.outer(np.asarray(s, np.float64), np.asarray(ws, np.float64))
    y = p if b is None else p + np.asarray(b, np.float64)
    return y, 3.01 * H * np.abs(p) + 1.01 * H * np.abs(y) + 2.0 ** -140


def linear(x, w, b=None):
    """(y, bound) of an fp32 product on the bf16 units: per 16 inputs six instructions, each
    off by at most 2^-23 of the magnitudes' sum (the unit does not round to nearest), the
    products left out (2^-24 of it), up to 64 splits or waves, and the bias."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    size = np.abs(x) @ np.abs(w).T
    y = x @ w.T
    if b is not None:
        y = y + b
        size = size + np.abs(b)
    return y, (6 * -(-x.shape[1] // 16) + 70) * 2.0 ** -23 * size
