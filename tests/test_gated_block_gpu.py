"""examples/gated_block.py: the operators of a gated feed-forward block together, as a program
uses them.  One block's gradients against float64 autograd, a step's clipping, and served rows.

Bounds of the gradients: all of a step's products and sums in fp32, each off by 2^-16 of the
sum of its terms' magnitudes at most (sums of up to 512 terms, six matrix instructions for 16
of them at 2^-23 each are 2^-15.4, of which random signs leave far less), carried through at
most four of them: compared in norm, 2^-13 of the gradient's."""
import importlib.util
import os

import pytest
import torch

import minitensor_amd as mt

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ex():
    path = os.path.join(os.path.dirname(__file__), "..", "examples", "gated_block.py")
    spec = importlib.util.spec_from_file_location("gated_block", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def block_of(ex, width, hidden, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    block = ex.Block(width, hidden, g)
    block.gain = 1 + 0.1 * torch.randn(width, device="cuda", generator=g)
    block.b = 0.1 * torch.randn(2 * hidden, device="cuda", generator=g)
    return block, g


def plain(params, x):
    gain, w, b, out = params
    n = x * (x.square().mean(1, keepdim=True) + 1e-6).rsqrt() * gain
    gate, up = (n @ w.t() + b).chunk(2, 1)
    return (gate * torch.sigmoid(gate) * up) @ out.t()


@pytest.mark.parametrize("rows,width,hidden", [(5, 48, 96), (130, 96, 200), (257, 128, 512)])
def test_gradients_of_a_block(ex, rows, width, hidden):
    block, g = block_of(ex, width, hidden, rows)
    x = torch.randn(rows, width, device="cuda", generator=g)
    target = torch.randn(rows, width, device="cuda", generator=g)
    loss, (grads,) = ex.gradients([block], x, target)
    params = [p.cpu().double().requires_grad_(True) for p in block.parameters()]
    X = x.cpu().double()
    want = (plain(params, X) + X - target.cpu().double()).square().mean()
    assert abs(loss.item() - want.item()) <= 2.0 ** -13 * want.item()
    for got, p in zip(grads, torch.autograd.grad(want, params)):
        assert (got.cpu().double() - p).norm() <= 2.0 ** -13 * p.norm()


def test_a_clipped_step(ex):
    block, g = block_of(ex, 64, 96, 1)
    x, target = (torch.randn(40, 64, device="cuda", generator=g) for _ in range(2))
    _, (grads,) = ex.gradients([block], x, target)
    before = [p.clone() for p in block.parameters()]
    norm = sum(t.double().square().sum() for t in grads).sqrt().item()
    most = 0.5 * norm
    _, n = ex.train_step([block], x, target, rate=1.0, max_norm=most)
    assert abs(n.item() - norm) <= 2.0 ** -23 * norm
    moved = sum((p.double() - q.double()).square().sum() for p, q in zip(block.parameters(), before)).sqrt()
    # (each parameter's subtraction rounds by 2^-24 of it)
    slack = 2.0 ** -23 * sum(q.double().square().sum() for q in before).sqrt().item()
    assert abs(moved.item() - most) <= 1e-5 * most + slack


def test_served_rows(ex):
    """A token and a prompt give a row the same, and that is the block's on the rows and weights
    that were put in 8 bits."""
    block, g = block_of(ex, 200, 320, 2)
    x = torch.randn(70, 200, device="cuda", generator=g)
    served = ex.Served([block])
    all_ = served.rows(x)
    for i in (0, 33, 69):
        assert torch.equal(served.rows(x[i:i + 1]), all_[i:i + 1])
    gain, w, b, out = served.layers[0]
    n = mt.dequantize_q8(mt.rms_norm(x, gain, y=False, q8=True).q8).double()
    gate, up = (n @ mt.dequantize_q8(w).double().t() + b.double()).chunk(2, 1)
    h = mt.dequantize_q8(mt.quantize_q8((gate * torch.sigmoid(gate) * up).float())).double()
    want = h @ mt.dequantize_q8(out).double().t() + x.double()
    # a hidden value that lies on the border of two codes may fall on either side: one step
    # of its row for a few of 320 of them; the rest is fp32 rounding
    step = (h.abs().amax(1, keepdim=True) / 127) * mt.dequantize_q8(out).double().abs().amax(1)
    assert ((all_.double() - want).abs() <= 3 * step + 1e-5 * want.abs().amax()).all()


def test_the_example_runs(ex, capsys):
    ex.main(width=64, hidden=96, rows=80, depth=2, steps=2)
    assert "served, a prompt" in capsys.readouterr().out
