"""Residual blocks that train with their activations kept in 8 bits and are then served with
4-bit weights, token by token.

A block is  h = stream + (the block before's output);  out = Linear(rms_norm(h)).  One pass of
rms_norm adds, normalises and keeps the rows in 8 bits; the backward pass takes the weight's
gradient from those (a quarter of the memory that fp32 rows would hold until then), and the
gradient that comes down the residual stream joins inside rms_norm_backward.

    python examples/lowbit_block.py
"""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import minitensor_amd as mt  # noqa: E402


class Block:
    def __init__(self, width, generator):
        self.gain = torch.ones(width, device="cuda")
        self.w = torch.randn(width, width, device="cuda", generator=generator) / (2 * width) ** 0.5
        self.b = torch.zeros(width, device="cuda")

    def forward(self, x, stream):
        """The block's output, and what its backward pass needs; kept.h is the stream now."""
        kept = mt.rms_norm(x, self.gain, residual=stream, q8=True)
        out = mt.linear(kept.y, self.w, self.b)
        return out, kept._replace(y=None)                     # (the fp32 rows are let go)

    def backward(self, dout, dstream, kept):
        """(gradient of h, which is that of the block before's output and of its stream;
        gradients of gain, w and b)."""
        dy, dw, db = mt.linear_backward_q8(dout, kept.q8, self.w)
        dh, dgain = mt.rms_norm_backward(dy, kept.h, self.gain, kept.rstd, dh=dstream)
        return dh, (dgain, dw, db)

    def step(self, grads, rate):
        for p, g in zip((self.gain, self.w, self.b), grads):
            p.sub_(g, alpha=rate)


def train_step(blocks, x, target, rate=0.0):
    """Mean squared error of the blocks' stream against target; (loss, gradients by block)."""
    out, stream, kept = x, torch.zeros_like(x), []
    for block in blocks:
        out, k = block.forward(out, stream)
        stream = k.h
        kept.append(k)
    diff = out + stream - target
    dout = dstream = diff * (2.0 / diff.numel())
    grads = []
    for block, k in zip(reversed(blocks), reversed(kept)):
        dstream, g = block.backward(dout, dstream, k)
        dout = dstream
        grads.append(g)
    grads.reverse()
    if rate:
        for block, g in zip(blocks, grads):
            block.step(g, rate)
    return float(diff.square().mean()), grads


class Served:
    """The blocks with weights in 4 bits."""

    def __init__(self, blocks, group=128):
        self.layers = [(b.gain, mt.quantize_q4(b.w, group), b.b) for b in blocks]

    def token(self, x):
        out, stream = x, torch.zeros_like(x)
        for gain, w, b in self.layers:
            r = mt.rms_norm(out, gain, residual=stream, y=False, q8=True, h=stream)
            out = mt.linear_q4(r.q8, w, b)
        return out + stream


def main(width=1024, rows=512, depth=2, steps=40):
    g = torch.Generator(device="cuda").manual_seed(0)
    blocks = [Block(width, g) for _ in range(depth)]
    x = torch.randn(rows, width, device="cuda", generator=g)
    target = x + 0.5 * torch.tanh(x.roll(1, 1))
    for i in range(steps):
        loss, _ = train_step(blocks, x, target, rate=0.1 * width)
        if i % 10 == 0 or i == steps - 1:
            print("step %2d  loss %.4f" % (i, loss))
    served = Served(blocks)
    y = torch.cat([served.token(x[i:i + 1]) for i in range(8)])
    print("served, 8 tokens: mean squared error %.4f" % (y - target[:8]).square().mean().item())


if __name__ == "__main__":
    main()
