"""The 8-bit saved activations and the layer over them where they can go wrong beside their sizes."""
import pytest
import torch

from sgnn_amd import nn as snn

pytestmark = pytest.mark.gpu


def test_products_of_two_numbers(gpu_device):
    """An fp32 product takes six of the nine products of two numbers' three parts; what it leaves out is at
    most 2^-22 of the whole.  Numbers 1 + 2^-7 - m 2^-23, for which every sum on the way is exact (all are
    multiples of 2^-23 below 2), so that nothing else is off; the result is no further than that."""
    m = torch.tensor([1, 2, 5, 31, 64, 127, 128])
    v = (1 + 2.0 ** -7 - m.double() * 2.0 ** -23).float()
    assert torch.equal(v.double(), 1 + 2.0 ** -7 - m.double() * 2.0 ** -23)
    want = v.double()[:, None] * v.double()[None]
    x, w = v[:, None].to(gpu_device), v[:, None].to(gpu_device)
    y = snn.linear_saved_int8(x, w).double().cpu()
    assert bool(((y - want).abs() <= 2.0 ** -22 * want).all())
    x.requires_grad_()
    eye = torch.zeros(7, 7, device=gpu_device)
    eye[:, 3] = v.to(gpu_device)                     # dx = grad . weight, one product each
    snn.linear_saved_int8(x, w).backward(eye)
    want = v.double() * v.double()[3]
    assert bool(((x.grad[:, 0].double().cpu() - want).abs() <= 2.0 ** -22 * want).all())
