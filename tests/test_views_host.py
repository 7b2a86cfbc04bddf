"""What the Python paths refuse of a tensor before they hand its memory to a kernel, without a
GPU: a stand-in for a GPU tensor has all that the checks look at."""
import pytest
import torch

import minitensor_amd as mt
from minitensor_amd import lowbit


class View(torch.Tensor):
    """A tensor that says it is on the GPU."""
    device = torch.device("cuda")


def view(t):
    return t.as_subclass(View)


def test_a_negated_view_is_refused():
    z = torch.complex(torch.ones(3, 4), torch.ones(3, 4)).conj()
    mt._require_gpu(None, view(torch.ones(3, 4)))
    assert z.imag.is_neg()
    with pytest.raises(ValueError, match="negated"):
        mt._require_gpu(view(torch.ones(3, 4)), view(z.imag))
    lowbit._bytes_on_gpu(view(torch.ones(3, dtype=torch.int8)), torch.int8, "q")
    with pytest.raises(ValueError, match="negated"):
        lowbit._bytes_on_gpu(view(torch._neg_view(torch.ones(3, dtype=torch.int8))), torch.int8, "q")


def test_clipping_without_a_largest_norm_is_refused():
    """(It used to measure the norm and scale nothing.)"""
    with pytest.raises(ValueError, match="largest norm"):
        mt.clip_grad_norm([torch.ones(3)], None)
