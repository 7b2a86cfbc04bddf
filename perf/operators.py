"""The operators around a Linear layer whose activations are kept in 8 bits and
whose weights are served in 4, as their users call them, and their plain forms.

  rms     y = rms_norm(x + residual)·weight: the sum, the norm and its rows in
          8 bits with a scale each, and for training the gradients
  q4      a Linear layer over 4-bit weights with a scale per group of inputs, its
          rows in 32 bits or in 8 (from rms or keep)
  keep    rows kept in 8 bits for the backward pass, and read back
  back    a Linear layer's gradients from the rows that were kept

Rows in 8 bits: q int8 [R, C], scale [R]: x[r, c] ~ q[r, c]·scale[r], with
scale = max(max|x[r]|/127, 2^-126) and q = x·(1/scale) rounded to nearest.
4-bit weights: packed uint8 [N, 16·ceil(K/32)]: input 2i in the low four bits of
byte i, 2i + 1 in the high ones, two's complement; scale [N, ceil(K/group)].
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6


def listed():
    return [
        # one token of a decoding loop between two blocks: latency alone
        dict(name="rms_token", kind="rms", rows=1, width=4096, train=False),
        # a prompt on its way into a layer with 8-bit rows
        dict(name="rms_prompt", kind="rms", rows=2048, width=4096, train=False),
        # a training step's norm, forward and backward: ragged, and a large batch
        dict(name="rms_train_ragged", kind="rms", rows=1027, width=1285, train=True),
        dict(name="rms_train_large", kind="rms", rows=8192, width=2048, train=True),
        # one token through a square layer: the weights' bytes, and a call's fixed cost
        dict(name="q4_token", kind="q4", rows=1, fin=4096, fout=4096, group=128, q8=False, bias=False),
        # one token, its row in 8 bits, into a wide hidden layer
        dict(name="q4_token_wide_q8", kind="q4", rows=1, fin=4096, fout=16384, group=128, q8=True,
             bias=False),
        # a batch of samples into a classifier head
        dict(name="q4_batch_head", kind="q4", rows=16, fin=2048, fout=1000, group=64, q8=False,
             bias=True),
        # a prompt: compute-bound, the largest work
        dict(name="q4_prompt", kind="q4", rows=2048, fin=4096, fout=8192, group=128, q8=False,
             bias=False),
        # a ragged prompt with 8-bit rows and small groups
        dict(name="q4_prompt_q8_ragged", kind="q4", rows=1027, fin=2047, fout=4096, group=32,
             q8=True, bias=True),
        # a large layer's input put away and read back
        dict(name="keep_large", kind="keep", rows=8192, width=4096),
        # a classifier head's backward pass, gradients accumulated over two batches
        dict(name="back_head", kind="back", rows=256, fin=2048, fout=1000, dx=True, beta=1.0),
        # a large first layer's backward pass (it needs no dX)
        dict(name="back_large", kind="back", rows=8192, fin=4096, fout=4096, dx=False, beta=0.0),
    ]


def _log_int(rng, lo, hi, aligned):
    """An integer spread over [lo, hi] by its logarithm; a multiple of 16
    above 32 when `aligned`."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if aligned and v > 32:
        v = max(lo, v // 16 * 16)
    return min(max(v, lo), hi)


def draw(rng):
    kind = rng.choice(["rms", "rms", "q4", "q4", "q4", "keep", "back", "back"])
    al = rng.random() < 0.6          # most programs' sizes are multiples of 16
    while True:
        if kind == "rms":
            c = dict(kind="rms", rows=_log_int(rng, 1, 8192, False),
                     width=_log_int(rng, 64, 8192, al), train=rng.random() < 0.5)
        elif kind == "q4":
            few = rng.random() < 0.5     # decoding, or a prompt
            c = dict(kind="q4", rows=_log_int(rng, 1, 64, False) if few else _log_int(rng, 65, 2048, al),
                     fin=_log_int(rng, 128, 8192, al), fout=_log_int(rng, 64, 16384, al),
                     group=rng.choice([32, 64, 128, 128]), q8=rng.random() < 0.4,
                     bias=rng.random() < 0.5)
        elif kind == "keep":
            c = dict(kind="keep", rows=_log_int(rng, 1, 8192, al), width=_log_int(rng, 64, 8192, al))
        else:
            c = dict(kind="back", rows=_log_int(rng, 8, 8192, al), fin=_log_int(rng, 64, 4096, al),
                     fout=_log_int(rng, 10, 4096, al), dx=rng.random() < 0.6,
                     beta=rng.choice([0.0, 1.0]))
        w = work(c)
        if w["flops"] <= 1.4e11 and w["bytes"] <= 4e8:
            return c


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
    if case["kind"] == "rms":
        t, d = case["rows"], case["width"]
        # a block's output and the stream that it is added to, a few wide channels
        wide = 1 + 7 * (torch.rand(d, device=DEV, generator=g) < 0.01)
        s["x"] = _normal(g, t, d, std=0.5)
        s["residual"] = _normal(g, t, d) * wide
        s["weight"] = 1 + _normal(g, d, std=0.1)
        if case["train"]:
            s["dy"] = _normal(g, t, d, std=0.01)
            s["dh"] = _normal(g, t, d, std=0.01)   # arrives along the residual stream
    elif case["kind"] == "q4":
        m, k, n, group = case["rows"], case["fin"], case["fout"], case["group"]
        x = _normal(g, m, k)
        s["q"], s["scale"] = _rows_q8(x) if case["q8"] else (None, None)
        s["x"] = None if case["q8"] else x
        # codes of a normal weight: +-7 at 2.5 standard deviations, and its scales
        kp = (k + 31) // 32 * 32
        code = torch.zeros(n, kp, device=DEV)
        code[:, :k] = _normal(g, n, k, std=2.8).round().clamp(-7, 7)
        code = code.to(torch.int16) & 15
        s["packed"] = (code[:, 0::2] | (code[:, 1::2] << 4)).to(torch.uint8)
        s["wscale"] = (0.5 + torch.rand(n, (k + group - 1) // group, device=DEV, generator=g)) \
            * (0.36 / math.sqrt(k))
        s["bias"] = _normal(g, n, std=0.1) if case["bias"] else None
    elif case["kind"] == "keep":
        s["x"] = torch.relu(_normal(g, case["rows"], case["width"]))
    else:
        r, fi, fo = case["rows"], case["fin"], case["fout"]
        # activations after a ReLU, He weights, a loss gradient's scale
        s["q"], s["scale"] = _rows_q8(torch.relu(_normal(g, r, fi)))
        s["w"] = _normal(g, fo, fi, std=(2.0 / fi) ** 0.5)
        s["dy"] = _normal(g, r, fo, std=0.01)
        # gradients of the batch before, added to (kept apart from the sums, so
        # that every pass gives the same)
        s["dw0"] = _normal(g, fo, fi, std=0.01) if case["beta"] else None
        s["db0"] = _normal(g, fo, std=0.01) if case["beta"] else None
    return s


def _plain_rms(s):
    h = s["x"] + s["residual"]
    rstd = torch.rsqrt((h * h).mean(1) + EPS)
    xhat = h * rstd[:, None]
    y = xhat * s["weight"]
    q, scale = _rows_q8(y)
    out = {"h": h, "codes": q.to(torch.bfloat16), "scale": scale}
    if s["case"]["train"]:
        gy = s["dy"] * s["weight"]
        out["y"] = y
        out["dh"] = s["dh"] + rstd[:, None] * (gy - xhat * (gy * xhat).mean(1, keepdim=True))
        out["dweight"] = (s["dy"] * xhat).sum(0)
    return out


def _plain_q4(s):
    case = s["case"]
    k, group = case["fin"], case["group"]
    low, high = (s["packed"] & 15).int(), (s["packed"] >> 4).int()
    code = torch.stack([low, high], 2).flatten(1)[:, :k]
    w = ((code ^ 8) - 8).float() * s["wscale"].repeat_interleave(group, 1)[:, :k]
    x = s["q"].float() * s["scale"][:, None] if case["q8"] else s["x"]
    y = x @ w.t()
    return y if s["bias"] is None else y + s["bias"]


def _plain_back(s):
    case = s["case"]
    x = s["q"].float() * s["scale"][:, None]
    out = {"dw": s["dy"].t() @ x, "db": s["dy"].sum(0)}
    if case["beta"]:
        out["dw"] = out["dw"] + case["beta"] * s["dw0"]
        out["db"] = out["db"] + case["beta"] * s["db0"]
    if case["dx"]:
        out["dx"] = s["dy"] @ s["w"]
    return out


def _own(s):
    import minitensor_amd as mt
    case = s["case"]
    if case["kind"] == "rms":
        r = mt.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS, y=case["train"],
                        q8=True)
        # (an 8-bit code is exact in bfloat16)
        out = {"h": r.h, "codes": r.q8.q.to(torch.bfloat16), "scale": r.q8.scale}
        if case["train"]:
            out["y"] = r.y
            out["dh"], out["dweight"] = mt.rms_norm_backward(s["dy"], r.h, s["weight"], r.rstd,
                                                             dh=s["dh"])
        return out
    if case["kind"] == "q4":
        x = mt.Q8Rows(s["q"], s["scale"]) if case["q8"] else s["x"]
        w = mt.Q4Weight(s["packed"], s["wscale"], case["fin"], case["group"])
        return mt.linear_q4(x, w, s["bias"])
    if case["kind"] == "keep":
        x = mt.quantize_q8(s["x"])
        return {"x": mt.dequantize_q8(x), "scale": x.scale}
    out = {}
    dw, db = (s["dw0"].clone(), s["db0"].clone()) if case["beta"] else (None, None)
    dx, out["dw"], out["db"] = mt.linear_backward_q8(
        s["dy"], mt.Q8Rows(s["q"], s["scale"]), s["w"] if case["dx"] else None, dw=dw, db=db,
        beta_w=case["beta"], beta_b=case["beta"])
    if case["dx"]:
        out["dx"] = dx
    return out


def run(s):
    if own:
        return _own(s)
    kind = s["case"]["kind"]
    if kind == "rms":
        return _plain_rms(s)
    if kind == "q4":
        return _plain_q4(s)
    if kind == "keep":
        q, scale = _rows_q8(s["x"])
        return {"x": q.float() * scale[:, None], "scale": scale}
    return _plain_back(s)


def work(case):
    if case["kind"] == "rms":
        t, d = case["rows"], case["width"]
        # x, residual and weight read; h, the codes and their scales written
        b, f = 4 * (3 * t * d + d + t) + t * d, 8 * t * d
        if case["train"]:
            # and y, rstd and both gradients written, dy and the incoming dh read
            b += 4 * (4 * t * d + t + d)
            f += 11 * t * d
        return {"bytes": b, "flops": f}
    if case["kind"] == "q4":
        m, k, n, group = case["rows"], case["fin"], case["fout"], case["group"]
        b = n * ((k + 1) // 2) + 4 * n * ((k + group - 1) // group) + 4 * m * n
        b += m * k + 4 * m if case["q8"] else 4 * m * k
        b += 4 * n if case["bias"] else 0
        return {"bytes": b, "flops": 2 * m * n * k}
    if case["kind"] == "keep":
        r, c = case["rows"], case["width"]
        # read, put away in 8 bits, read from there, written in 32
        return {"bytes": 4 * r * c + 2 * (r * c + 4 * r) + 4 * r * c, "flops": 4 * r * c}
    r, fi, fo = case["rows"], case["fin"], case["fout"]
    grads = fo * fi + fo
    b = r * fi + 4 * r + 4 * r * fo + 4 * grads * (2 if case["beta"] else 1)
    f = 2 * r * fi * fo + r * fo
    if case["dx"]:
        b += 4 * (fo * fi + r * fi)
        f += 2 * r * fi * fo
    return {"bytes": b, "flops": f}


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["kind"] == "rms":
        h = d["x"] + d["residual"]
        inv = 1 / torch.sqrt(torch.mean(h ** 2, dim=1, keepdim=True) + EPS)
        y = h * inv * d["weight"]
        scale = y.abs().max(dim=1, keepdim=True).values / 127
        # the codes before they are rounded: both sides are off by the rounding
        out = {"h": h, "codes": y / scale, "scale": scale[:, 0]}
        if case["train"]:
            # d/dh of sum(dy·y): the product rule over h and inv(h)
            dinv = (d["dy"] * d["weight"] * h).sum(1, keepdim=True)
            out["y"] = y
            out["dh"] = d["dh"] + d["dy"] * d["weight"] * inv - dinv * inv ** 3 * h / case["width"]
            out["dweight"] = torch.einsum("td,td,tu->d", d["dy"], h, inv)
        return out
    if case["kind"] == "q4":
        m, k, n, group = case["rows"], case["fin"], case["fout"], case["group"]
        x = d["q"] * d["scale"].unsqueeze(1) if case["q8"] else d["x"]
        bits = s["packed"].to(torch.int64)
        w = torch.empty(n, 2 * bits.shape[1], dtype=torch.float64, device=DEV)
        w[:, 0::2], w[:, 1::2] = bits % 16, bits // 16
        w = torch.where(w > 7, w - 16, w)[:, :k]
        y = torch.zeros(m, n, dtype=torch.float64, device=DEV)
        for j in range(0, k, group):
            y += (x[:, j:j + group] @ w[:, j:j + group].t()) * d["wscale"][:, j // group]
        return y + d["bias"] if case["bias"] else y
    if case["kind"] == "keep":
        top = d["x"].abs().max(dim=1).values
        scale = torch.clamp(top / 127, min=2.0 ** -126)
        return {"x": torch.round(d["x"] / scale.unsqueeze(1)) * scale.unsqueeze(1), "scale": scale}
    x = d["q"] * d["scale"].unsqueeze(1)
    out = {"dw": torch.matmul(d["dy"].t(), x), "db": d["dy"].sum(dim=0)}
    if case["beta"]:
        out["dw"] += case["beta"] * d["dw0"]
        out["db"] += case["beta"] * d["db0"]
    if case["dx"]:
        out["dx"] = torch.matmul(d["dy"], d["w"])
    return out
