"""A caller's workspace has to be memory that the GPU reaches, to its last element: a host
tensor's or an expanded view's address in a kernel would be a write out of range."""
import pytest
import torch

import minitensor_amd as mt

N = 1 << 24


def test_host_memory_and_expanded_views_are_refused():
    with pytest.raises(ValueError):
        mt._require_ws(torch.empty(N, dtype=torch.uint8))
    with pytest.raises(ValueError):
        mt._require_ws(bytearray(16))
    mt._require_ws(None)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["host", "expanded"])
def test_every_call_checks_its_workspace(dev, kind):
    ws = (torch.empty(N, dtype=torch.uint8) if kind == "host"
          else torch.empty(1, dtype=torch.uint8, device=dev).expand(N))
    x, w = torch.ones(200, 4096, device=dev), torch.ones(64, 4096, device=dev)
    dy, dx = torch.ones(200, 64, device=dev), torch.full((200, 4096), 5.0, device=dev)
    img, ker = torch.ones(2, 8, 9, 9, device=dev), torch.ones(4, 8, 3, 3, device=dev)
    wq, xq = mt.quantize_q4(w), mt.quantize_q8(x)
    n = mt.rms_norm(x, None)
    calls = [
        lambda: mt.gemm(x, w.t(), ws=ws),
        lambda: mt.linear(x, w, ws=ws),
        lambda: mt.linear_backward(dy, x, w, dx=dx, ws=ws),
        lambda: mt.conv2d(img, ker, ws=ws),
        lambda: mt.conv2d_backward(img, ker, torch.ones(2, 4, 7, 7, device=dev), ws=ws),
        lambda: mt.linear_q4(x, wq, ws=ws),
        lambda: mt.linear_q4(xq, wq, ws=ws),
        lambda: mt.linear_backward_q8(dy, xq, w, dx=dx, ws=ws),
        lambda: mt.rms_norm_backward(x, n.h, None, n.rstd, out=dx, ws=ws),
    ]
    for i, f in enumerate(calls):
        with pytest.raises(ValueError, match="workspace"):
            f()
            pytest.fail(f"call {i} was taken")
    torch.cuda.synchronize()
    assert bool((dx == 5).all())


@pytest.mark.gpu
def test_a_slice_of_gpu_memory_is_taken(dev):
    big = torch.empty(N + 64, dtype=torch.uint8, device=dev)
    x = torch.randn(200, 4096, device=dev)
    wq = mt.quantize_q4(torch.randn(64, 4096, device=dev))
    assert torch.equal(mt.linear_q4(x, wq, ws=big[64:]), mt.linear_q4(x, wq))


@pytest.mark.gpu
def test_a_workspace_of_floats_counts_in_bytes(dev):
    x, dy = torch.randn(4096, 64, device=dev), torch.randn(4096, 64, device=dev)
    xq = mt.quantize_q8(x)
    need = mt.lib().mt_linear_backward_q8_workspace_f32(4096, 64, 64)
    assert need > 0
    ws = torch.empty((need + 3) // 4, device=dev)
    assert torch.equal(mt.linear_backward_q8(dy, xq, ws=ws)[1], mt.linear_backward_q8(dy, xq)[1])
    a, b = torch.randn(64, 65536, device=dev), torch.randn(65536, 64, device=dev)
    need = mt.lib().mt_gemm_workspace_f32(mt.mat(a), mt.mat(b), mt.mat(torch.empty(64, 64, device=dev)))
    assert need > 0
    assert torch.equal(mt.gemm(a, b, ws=torch.empty((need + 3) // 4, device=dev)), mt.gemm(a, b))
