"""examples/lowbit_block.py: the low-bit operators together, as a program uses them.  Last
block's gradients and a served token against float64; bounds: half a step of the kept 8-bit
rows (and 2^-16 of one) times what they are multiplied by, and fp32 sums, 2^-18 of the sum of
the terms' magnitudes."""
import importlib.util
import os

import pytest
import torch

import minitensor_amd as mt

pytestmark = pytest.mark.gpu
EPS32 = 2.0 ** -18


@pytest.fixture(scope="module")
def ex():
    path = os.path.join(os.path.dirname(__file__), "..", "examples", "lowbit_block.py")
    spec = importlib.util.spec_from_file_location("lowbit_block", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("rows,width", [(33, 96), (128, 256)])
def test_gradients_of_a_block(ex, rows, width):
    g = torch.Generator(device="cuda").manual_seed(rows)
    block = ex.Block(width, g)
    block.gain = 1 + 0.1 * torch.randn(width, device="cuda", generator=g)
    x = torch.randn(rows, width, device="cuda", generator=g)
    target = torch.randn(rows, width, device="cuda", generator=g)
    _, ((dgain, dw, db),) = ex.train_step([block], x, target)

    h, w, gain = x.double(), block.w.double(), block.gain.double()
    rstd = (h.square().mean(1, keepdim=True) + 1e-6).rsqrt()
    y = h * rstd * gain
    d = (y @ w.t() + h - target.double()) * (2.0 / x.numel())
    step = y.abs().amax(1, keepdim=True) / 127
    # (d itself has fp32's rounding: its terms are |y| |w|, |h| and |target|)
    de = EPS32 * (y.abs() @ w.abs().t() + h.abs() + target.double().abs()) * (2.0 / x.numel())
    bound = d.abs().t() @ ((0.5 + 2.0 ** -16) * step).expand_as(y) + de.t() @ y.abs() \
        + EPS32 * (d.abs().t() @ y.abs())
    assert ((dw.double() - d.t() @ y).abs() <= bound).all()
    assert ((db.double() - d.sum(0)).abs() <= de.sum(0) + EPS32 * d.abs().sum(0)).all()
    dy, dye = d @ w, de @ w.abs() + EPS32 * (d.abs() @ w.abs())
    xhat = h * rstd
    assert ((dgain.double() - (dy * xhat).sum(0)).abs()
            <= (dye * xhat.abs()).sum(0) + EPS32 * (dy * xhat).abs().sum(0)).all()


def test_it_learns(ex):
    g = torch.Generator(device="cuda").manual_seed(1)
    blocks = [ex.Block(64, g) for _ in range(2)]
    x = torch.randn(128, 64, device="cuda", generator=g)
    target = x + 0.5 * torch.tanh(x.roll(1, 1))
    loss = [ex.train_step(blocks, x, target, rate=3.0)[0] for _ in range(30)]
    assert loss[-1] < 0.5 * loss[0]


@pytest.mark.parametrize("group", [32, 128])
def test_a_served_token(ex, group):
    g = torch.Generator(device="cuda").manual_seed(2)
    block = ex.Block(200, g)
    x = torch.randn(1, 200, device="cuda", generator=g)
    served = ex.Served([block], group)
    out = served.token(x).double()
    q = mt.rms_norm(x, block.gain, y=False, q8=True).q8
    rows = q.q.double() * q.scale.double()[:, None]
    w = mt.dequantize_q4(served.layers[0][1]).double()
    # (a code times its scale, as dequantize_q4 gives it, has been rounded once)
    bound = EPS32 * (rows.abs() @ w.abs().t() + block.b.double().abs() + x.double().abs())
    assert ((out - (rows @ w.t() + block.b.double() + x.double())).abs() <= bound).all()
