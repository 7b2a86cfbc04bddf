"""Residual feed-forward blocks with a gated hidden layer, trained in fp32 with their gradients
clipped, and served with rows and weights in 8 bits.

A block is  h = stream + (the block before's output);  n = rms_norm(h);
out = Linear(act(n·Wgᵀ + bg) * (n·Wuᵀ + bu)).  Training keeps n and the projections; the
gradient at the projections is written over them.  Serving takes n and the hidden rows in 8
bits, each with a scale, by weights in 8 bits.

    python examples/gated_block.py
"""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import minitensor_amd as mt  # noqa: E402

ACT = "silu"


class Block:
    def __init__(self, width, hidden, generator):
        def normal(*shape):
            return torch.randn(*shape, device="cuda", generator=generator)
        self.gain = torch.ones(width, device="cuda")
        self.w = normal(2 * hidden, width) / width ** 0.5     # gates, then up rows
        self.b = torch.zeros(2 * hidden, device="cuda")
        self.out = normal(width, hidden) * (0.5 / hidden) ** 0.5

    def parameters(self):
        return [self.gain, self.w, self.b, self.out]

    def forward(self, x, stream):
        """The block's output, and what its backward pass needs; kept[0].h is the stream now."""
        n = mt.rms_norm(x, self.gain, residual=stream)
        g = mt.gated_linear(n.y, self.w, self.b, act=ACT, keep=True)
        return mt.linear(g.h, self.out), (n, g)

    def backward(self, dout, dstream, kept):
        """(gradient of h, which is that of the block before's output and of its stream;
        gradients in the order of parameters())."""
        n, g = kept
        dh, dw_out, _ = mt.linear_backward(dout, g.h, self.out, need_db=False)
        dn, dw, db = mt.gated_linear_backward(dh, g.gu, n.y, self.w, act=ACT, dgu=g.gu)
        d, dgain = mt.rms_norm_backward(dn, n.h, self.gain, n.rstd, dh=dstream)
        return d, [dgain, dw, db, dw_out]


def gradients(blocks, x, target):
    """Mean squared error of the blocks' stream against target: (loss, each block's gradients)."""
    out, stream, kept = x, torch.zeros_like(x), []
    for block in blocks:
        out, k = block.forward(out, stream)
        stream = k[0].h
        kept.append(k)
    diff = out + stream - target
    dout = dstream = diff * (2.0 / diff.numel())
    grads = []
    for block, k in zip(reversed(blocks), reversed(kept)):
        dstream, g = block.backward(dout, dstream, k)
        dout = dstream
        grads.append(g)
    grads.reverse()
    return diff.square().mean(), grads


def train_step(blocks, x, target, rate, max_norm):
    """(loss, norm of all gradients before they were clipped), on the GPU."""
    loss, grads = gradients(blocks, x, target)
    flat = [g for block in grads for g in block]
    norm = mt.clip_grad_norm(flat, max_norm)
    for block, gs in zip(blocks, grads):
        for p, g in zip(block.parameters(), gs):
            p.sub_(g, alpha=rate)
    return loss, norm


class Served:
    """The blocks with weights in 8 bits."""

    def __init__(self, blocks):
        self.layers = [(b.gain, mt.quantize_q8(b.w), b.b, mt.quantize_q8(b.out)) for b in blocks]

    def rows(self, x):
        out, stream = x, torch.zeros_like(x)
        for gain, w, b, w_out in self.layers:
            n = mt.rms_norm(out, gain, residual=stream, y=False, q8=True, h=stream)
            h = mt.gated_linear(n.q8, w, b, act=ACT).h
            out = mt.linear_q8(mt.quantize_q8(h), w_out)
        return out + stream


def main(width=512, hidden=1408, rows=512, depth=2, steps=40):
    g = torch.Generator(device="cuda").manual_seed(0)
    blocks = [Block(width, hidden, g) for _ in range(depth)]
    x = torch.randn(rows, width, device="cuda", generator=g)
    target = x + 0.5 * torch.tanh(x.roll(1, 1))
    for i in range(steps):
        loss, norm = train_step(blocks, x, target, rate=4.0, max_norm=0.1)
        if i % 10 == 0 or i == steps - 1:
            print("step %2d  loss %.4f  gradient norm %.3f" % (i, loss.item(), norm.item()))
    served = Served(blocks)
    y = torch.cat([served.rows(x[i:i + 1]) for i in range(8)])
    print("served, 8 tokens: mean squared error %.4f" % (y - target[:8]).square().mean().item())
    print("served, a prompt: mean squared error %.4f" % (served.rows(x) - target).square().mean().item())


if __name__ == "__main__":
    main()
