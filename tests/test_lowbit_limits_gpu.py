"""The operators of include/mtlowbit.h at the ends of their ranges: rows of no columns,
finite values whose parts or factors leave fp32's range, very wide rows, arguments that are
refused.  Bounds: tests/lowbit_reference.py."""
import numpy as np
import pytest
import torch

import lowbit_reference as ref
import minitensor_amd as mt

pytestmark = pytest.mark.gpu

FLT_MAX = np.finfo(np.float32).max


def rng(*key):
    return np.random.default_rng([int(k) for k in key])


def gpu(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def cpu(t):
    return t.detach().cpu().numpy()


def near(y, x, w, group, parts):
    """y against x·wᵀ in 64 bits, all of them finite."""
    want, size = x @ w.T, np.abs(x) @ np.abs(w).T
    y = cpu(y).astype(np.float64)
    assert np.isfinite(y).all()
    assert np.all(np.abs(y - want) <= ref.linear_bound(x.shape[1], group, parts) * size + 1e-44)


@pytest.mark.parametrize("r", [1, 5, 300])
def test_rows_of_no_columns(dev, r):
    """[R, 0]: the scale of an empty row is the smallest one, its mean square zero."""
    junk = [torch.full((r,), 7.0, device=dev) for _ in range(8)]
    del junk                          # (what the outputs below would hold if left unwritten)
    x = torch.empty(r, 0, device=dev)
    assert bool((mt.quantize_q8(x).scale == 2.0 ** -126).all())
    out = mt.Q8Rows(torch.empty(r, 0, dtype=torch.int8, device=dev), torch.full((r,), 7.0, device=dev))
    mt.quantize_q8(x, out=out)
    assert bool((out.scale == 2.0 ** -126).all())
    assert mt.dequantize_q8(out).shape == (r, 0)
    for q8 in (False, True):
        junk = [torch.full((r,), 7.0, device=dev) for _ in range(8)]
        del junk
        n = mt.rms_norm(x, torch.empty(0, device=dev), residual=x, eps=0.25, q8=q8)
        assert bool((n.rstd == 2.0).all()) and n.y.shape == n.h.shape == (r, 0)
        assert not q8 or bool((n.q8.scale == 2.0 ** -126).all())
