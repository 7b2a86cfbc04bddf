"""The operators of a gated feed-forward block, trained in fp32 and served in 8 bits, as
their users call them, and their plain forms.

  q8      a Linear layer on 8-bit rows and 8-bit weights: y = (q·wqᵀ)·s·ws (+ b), with a
          scale for each row (token) and each output channel
  gate    a gated feed-forward block's two projections, their activation and product:
          h = act(x·Wgᵀ + bg) * (x·Wuᵀ + bu), W [2F, K] with the gate's rows first; in
          fp32, for training with the gradients too, or with rows and weights in 8 bits
  clip    the norm of all gradients of a model, and the gradients scaled down to a
          largest norm

Rows in 8 bits: q int8 [R, C], scale [R]: x[r, c] ~ q[r, c]·scale[r]; a weight's rows are
its output channels.
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6


def listed():
    return [
        # one token of a decoding loop through a square layer: the weights' bytes and latency
        dict(name="q8_token", kind="q8", rows=1, fin=4096, fout=4096, bias=False),
        # a batch of samples into a classifier head
        dict(name="q8_batch_head", kind="q8", rows=16, fin=2048, fout=1000, bias=True),
        # a prompt: compute-bound
        dict(name="q8_prompt", kind="q8", rows=2048, fin=4096, fout=8192, bias=False),
        # a ragged prompt
        dict(name="q8_prompt_ragged", kind="q8", rows=1027, fin=2047, fout=4095, bias=True),
        # one token into a block's hidden layer, in fp32: the weights' bytes
        dict(name="gate_token", kind="gate", rows=1, fin=2048, hidden=4096, act="silu", q8=False,
             bias=False, train=False),
        # a ragged training step, forward and backward
        dict(name="gate_train_ragged", kind="gate", rows=509, fin=1285, hidden=2570,
             act="gelu_tanh", q8=False, bias=True, train=True),
        # a large batch's training step, forward and backward: the largest work
        dict(name="gate_train_large", kind="gate", rows=4096, fin=2048, hidden=4096, act="silu",
             q8=False, bias=False, train=True),
        # one token with rows and weights in 8 bits
        dict(name="gate_q8_token", kind="gate", rows=1, fin=4096, hidden=8192, act="silu", q8=True,
             bias=False, train=False),
        # a prompt with rows and weights in 8 bits
        dict(name="gate_q8_prompt", kind="gate", rows=2048, fin=4096, hidden=8192, act="silu",
             q8=True, bias=False, train=False),
        # a small model's gradients: latency
        dict(name="clip_small", kind="clip", blocks=2, width=64, hidden=256, most=1.0),
        # many tensors of middling size, odd ones among them
        dict(name="clip_many", kind="clip", blocks=48, width=255, hidden=1023, most=1.0),
        # a few blocks with large weights: memory
        dict(name="clip_large", kind="clip", blocks=4, width=2048, hidden=5632, most=1.0),
    ]


def _log_int(rng, lo, hi, aligned):
    """An integer spread over [lo, hi] by its logarithm; a multiple of 16
    above 32 when `aligned`."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if aligned and v > 32:
        v = max(lo, v // 16 * 16)
    return min(max(v, lo), hi)


def draw(rng):
    kind = rng.choice(["q8", "q8", "q8", "gate", "gate", "gate", "gate_q8", "gate_q8", "clip", "clip"])
    al = rng.random() < 0.6          # most programs' sizes are multiples of 16
    while True:
        few = rng.random() < 0.5     # decoding, or a prompt
        rows = _log_int(rng, 1, 64, False) if few else _log_int(rng, 65, 4096, al)
        if kind == "q8":
            c = dict(kind="q8", rows=rows, fin=_log_int(rng, 64, 8192, al),
                     fout=_log_int(rng, 10, 16384, al), bias=rng.random() < 0.5)
        elif kind == "gate":
            c = dict(kind="gate", rows=rows, fin=_log_int(rng, 64, 4096, al),
                     hidden=_log_int(rng, 64, 8192, al),
                     act=rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu", "sigmoid"]),
                     q8=False, bias=rng.random() < 0.5, train=rng.random() < 0.5)
        elif kind == "gate_q8":
            c = dict(kind="gate", rows=rows, fin=_log_int(rng, 64, 8192, al),
                     hidden=_log_int(rng, 64, 16384, al),
                     act=rng.choice(["silu", "silu", "gelu", "gelu_tanh"]), q8=True,
                     bias=rng.random() < 0.5, train=False)
        else:
            c = dict(kind="clip", blocks=_log_int(rng, 1, 64, False), width=_log_int(rng, 16, 2048, al),
                     hidden=_log_int(rng, 16, 8192, al), most=rng.choice([1.0, 1.0, 0.25, 1e9]))
        w = work(c)
        if w["flops"] <= 4e11 and w["bytes"] <= 1.1e9:
            return c


def _shapes(case):
    """The parameters of `blocks` residual blocks: norm weight, both projections with their
    bias, and the projection back with its."""
    d, f = case["width"], case["hidden"]
    return [(d,), (2 * f, d), (2 * f,), (d, f), (d,)] * case["blocks"]


def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, device=DEV, generator=g) * std


def _rows_q8(x):
    """Rows in 8 bits: (q int8, scale)."""
    scale = (x.abs().amax(1) / 127).clamp_min(2.0 ** -126)
    return torch.round(x * (1.0 / scale)[:, None]).to(torch.int8), scale


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case=case)
    if case["kind"] == "clip":
        # gradients as they come out of a backward pass: some layers' far larger than others'
        shapes = _shapes(case)
        sizes = [math.prod(shape) for shape in shapes]
        flat = _normal(g, sum(sizes), std=0.01)
        std = torch.exp(_normal(g, len(shapes)))
        s["grads"] = [(t * std[i]).view(shapes[i]) for i, t in enumerate(flat.split(sizes))]
        # where the program has the scaled ones: one after the other in one buffer
        s["flat"] = torch.empty_like(flat)
        s["out"] = [t.view(shape) for t, shape in zip(s["flat"].split(sizes), shapes)]
        return s
    r, k = case["rows"], case["fin"]
    n = case["fout"] if case["kind"] == "q8" else 2 * case["hidden"]
    # rows out of a norm, a few wide channels among them
    wide = 1 + 3 * (torch.rand(k, device=DEV, generator=g) < 0.01)
    x = _normal(g, r, k) * wide
    w = _normal(g, n, k, std=k ** -0.5) * (0.5 + torch.rand(n, 1, device=DEV, generator=g))
    if case["kind"] == "q8" or case["q8"]:
        s["x"], s["x_scale"] = _rows_q8(x)
        s["w"], s["w_scale"] = _rows_q8(w)
    else:
        s["x"], s["w"] = x, w
    s["bias"] = _normal(g, n, std=0.1) if case["bias"] else None
    if case["kind"] == "gate" and case["train"]:
        s["dh"] = _normal(g, r, case["hidden"], std=0.01)
    return s


def _act(name, a):
    """(the activation, its derivative) at a."""
    if name == "silu":
        t = 1 / (1 + torch.exp(-a))
        return a * t, t * (1 + a * (1 - t))
    if name == "sigmoid":
        t = 1 / (1 + torch.exp(-a))
        return t, t * (1 - t)
    if name == "relu":
        return a * (a > 0), (a > 0).to(a.dtype)
    if name == "gelu":
        phi = 0.5 * (1 + torch.erf(a * 0.5 ** 0.5))
        return a * phi, phi + a * torch.exp(-0.5 * a * a) * (2 * math.pi) ** -0.5
    c = (2 / math.pi) ** 0.5
    t = torch.tanh(c * (a + 0.044715 * a * a * a))
    return 0.5 * a * (1 + t), 0.5 * (1 + t) + 0.5 * a * (1 - t * t) * c * (1 + 3 * 0.044715 * a * a)


def _plain_projections(s):
    x, w = s["x"], s["w"]
    if x.dtype == torch.int8:
        x = x.float() * s["x_scale"][:, None]
        w = w.float() * s["w_scale"][:, None]
    y = x @ w.t()
    return y if s["bias"] is None else y + s["bias"]


def _plain_gate(s):
    case = s["case"]
    gu = _plain_projections(s)
    a, u = gu.split(case["hidden"], 1)
    act, slope = _act(case["act"], a)
    h = act * u
    if not case["train"]:
        return h
    dgu = torch.cat([s["dh"] * u * slope, s["dh"] * act], 1)
    return {"h": h, "dx": dgu @ s["w"], "dw": dgu.t() @ s["x"], "db": dgu.sum(0)}


def _plain_clip(s):
    total = sum((t * t).sum(dtype=torch.float64) for t in s["grads"])
    norm = torch.sqrt(total)
    c = torch.clamp(s["case"]["most"] / (norm + EPS), max=1.0).float()
    for t, o in zip(s["grads"], s["out"]):
        torch.mul(t, c, out=o)
    return {"norm": norm.float(), "grads": s["flat"]}


def _own(s):
    import minitensor_amd as mt
    case = s["case"]
    if case["kind"] == "clip":
        norm = mt.clip_grad_norm(s["grads"], case["most"], eps=EPS, out=s["out"])
        return {"norm": norm, "grads": s["flat"]}
    x, w = s["x"], s["w"]
    if x.dtype == torch.int8:
        x, w = mt.Q8Rows(x, s["x_scale"]), mt.Q8Rows(w, s["w_scale"])
    if case["kind"] == "q8":
        return mt.linear_q8(x, w, s["bias"])
    r = mt.gated_linear(x, w, s["bias"], act=case["act"], keep=case["train"])
    if not case["train"]:
        return r.h
    dx, dw, db = mt.gated_linear_backward(s["dh"], r.gu, x, w, act=case["act"])
    return {"h": r.h, "dx": dx, "dw": dw, "db": db}


def run(s):
    if own:
        return _own(s)
    kind = s["case"]["kind"]
    if kind == "clip":
        return _plain_clip(s)
    return _plain_projections(s) if kind == "q8" else _plain_gate(s)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "clip":
        g = torch.cat([t.double().flatten() for t in s["grads"]])
        norm = float(torch.linalg.vector_norm(g))
        if norm + EPS > case["most"]:
            g = g * (case["most"] / (norm + EPS))
        return {"norm": torch.tensor(norm, dtype=torch.float64), "grads": g}
    x, w = s["x"].double(), s["w"].double()
    y = torch.mm(x, w.t().contiguous())
    if s["x"].dtype == torch.int8:               # whole numbers, exact
        y = y * torch.outer(s["x_scale"].double(), s["w_scale"].double())
    if s["bias"] is not None:
        y += s["bias"].double()
    if case["kind"] == "q8":
        return y
    f = case["hidden"]
    a, u = y[:, :f].contiguous(), y[:, f:].contiguous()
    name = case["act"]
    a.requires_grad_(True)
    if name == "silu":
        act = torch.sigmoid(a) * a
    elif name == "sigmoid":
        act = torch.sigmoid(a)
    elif name == "relu":
        act = torch.clamp_min(a, 0)
    elif name == "gelu":
        act = 0.5 * a * torch.erfc(-a / math.sqrt(2))
    else:
        act = a * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3))
    if not case["train"]:
        return (act * u).detach()
    dh = s["dh"].double()
    da, = torch.autograd.grad(act, a, dh * u)
    act = act.detach()
    dgu = torch.cat([da, dh * act], 1)
    return {"h": act * u, "dx": torch.mm(dgu, w), "dw": torch.mm(dgu.t().contiguous(), x),
            "db": dgu.sum(0)}


def work(case):
    if case["kind"] == "clip":
        n = sum(math.prod(shape) for shape in _shapes(case))
        return {"bytes": 8 * n + 4, "flops": 3 * n}
    r, k = case["rows"], case["fin"]
    if case["kind"] == "q8":
        n = case["fout"]
        b = r * k + n * k + 4 * (r + n) + 4 * r * n + (4 * n if case["bias"] else 0)
        return {"bytes": b, "flops": 2 * r * n * k}
    f = case["hidden"]
    b = (r * k + 2 * f * k + 4 * (r + 2 * f)) if case["q8"] else 4 * (r * k + 2 * f * k)
    b += 4 * r * f + (8 * f if case["bias"] else 0)
    n = 4 * r * k * f + 6 * r * f
    if case["train"]:
        # dh read; dx, dw and db written; two more products of the same size
        b += 4 * (r * f + r * k + 2 * f * k + 2 * f)
        n += 8 * r * k * f + 10 * r * f
    return {"bytes": b, "flops": n}
