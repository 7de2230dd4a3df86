"""Rows whose mean is far larger than their deviation: the gradients are of the normalised values that the forward pass gave."""
import pytest
import torch

from test_gpu_experts import BF16, FP16, FP32, gen, normal

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def norm():
    from flash_sinkhorn_b200.experts import layer_norm
    return layer_norm


# sums of a thread's columns in registers, by a kernel of their own, rows that registers do not hold; vector loads and single values
@pytest.mark.parametrize("f", [64, 501, 2048, 2049, 4096, 4104, 4097, 16384, 16392, 20001, 40000])
@pytest.mark.parametrize("mean", [0.0, 1000.0, -3e5])
def test_backward_takes_the_forward_s_values(norm, f, mean):
    """With one row, dy = 1 and w = 1 (all products and sums exact), the gradient to w is the normalised row itself."""
    x = (normal(gen(f), 1, f) + mean).requires_grad_()
    w = torch.ones(f, device="cuda", requires_grad=True)
    y = norm(x, w, eps=0.0)
    (dw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert torch.equal(dw, y[0].detach())


@pytest.mark.parametrize("f", [2048, 501, 4104, 16392])
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
def test_gradient_to_rows_with_a_large_mean(norm, f, dtype):
    """dx from the normalised values that the forward pass gave, in 64 bits.

    Sums of a row in fp32: at most 42 additions of a thread's values, five shuffles and the warps', 2^-24 each (rows above 16384: 128), so
    ``deep`` of the sum of magnitudes for either mean, twice that for the products and differences, and the same once more for r.
    """
    g = gen(f + 1)
    x = (normal(g, 7, f) + 1000).to(dtype).requires_grad_()
    dy = normal(g, 7, f).to(dtype)
    (dx,) = torch.autograd.grad(norm(x, eps=0.0), x, dy)
    d = x.detach().double()
    n = norm(x.detach().float(), eps=0.0).double()
    r = 1 / (d - d.mean(1, keepdim=True)).square().mean(1, keepdim=True).sqrt()
    u = dy.double()
    want = r * (u - u.mean(1, keepdim=True) - n * (u * n).mean(1, keepdim=True))
    deep = (42 if f <= 16384 else 128) * 2.0**-24
    bound = 4 * deep * r * (u.abs() + u.abs().mean(1, keepdim=True) + n.abs() * (u * n).abs().mean(1, keepdim=True))
    bound = bound + (torch.finfo(dtype).eps / 2 if dtype != FP32 else 2.0**-24) * want.abs() + (2.0**-24 if dtype == FP16 else 0.0)
    assert ((dx.double() - want).abs() <= bound).all(), ((dx.double() - want).abs() / bound).max().item()
