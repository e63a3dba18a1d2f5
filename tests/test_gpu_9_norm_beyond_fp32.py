"""Clipping where the norm itself leaves the range of fp32 though every gradient is finite: the norm is reported as
infinite, and the factor is that of the norm in 64 bits.  Tolerance: the factor, the product with the gradient and
its share of the momentum are rounded to fp32 once each (2^-24 relative; a factor below the normal numbers is off by
up to 2^-150 instead), 1 - beta2 = 0.01 once more."""
import math

import pytest
import torch

from fast_ops_b200.lion import Lion, grad_norm
from fast_ops_b200.lion.grad_norm import finish_norm

pytestmark = pytest.mark.gpu


def factor(norm, max_norm):
    return min(1.0, max_norm / (norm + 1e-6))


@pytest.mark.parametrize("n", [1000, 300_000])  # one launch, and two
@pytest.mark.parametrize("max_norm", [1.0, 1e30, 1e39, math.inf])
def test_finite_gradients_are_scaled_by_their_norm(n, max_norm, cuda_device):
    value = 3e38
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    p.grad = torch.full_like(p, value)
    p.grad[::3] *= -1
    opt = Lion([p], lr=1e-3, max_grad_norm=max_norm)
    opt.step()
    g = p.grad.double()
    norm = g.square().sum().sqrt().item()
    assert norm > torch.finfo(torch.float32).max and opt.grad_norm.item() == math.inf
    coef = factor(norm, max_norm)
    rel = 4 * 2.0**-24 + 2.0**-150 / coef
    want = g * coef * 0.01
    assert ((opt.state[p]["exp_avg"].double() - want).abs() <= rel * want.abs()).all()
    assert torch.equal(p.detach().sign(), -p.grad.sign())


def test_factor_from_a_sum_of_squares(cuda_device):
    for root, max_norm in ((1e40, 1e30), (1e100, 1e80), (3e38, 1.0), (1e39, 1e39)):
        sumsq = torch.tensor([root * root], device="cuda", dtype=torch.float64)
        norm, coef = finish_norm(sumsq, max_norm)
        assert norm.item() == (math.inf if root > torch.finfo(torch.float32).max else torch.tensor(root).item())
        want = factor(root, max_norm)
        assert abs(coef.item() - want) <= 4 * 2.0**-24 * want + 2.0**-150
    norm, coef = finish_norm(torch.tensor([math.inf], device="cuda", dtype=torch.float64), 1.0)
    assert norm.item() == math.inf and coef.item() == 0.0
    norm, coef = finish_norm(torch.tensor([math.nan], device="cuda", dtype=torch.float64), 1.0)
    assert math.isnan(norm.item()) and math.isnan(coef.item())


def test_infinite_gradients_still_show(cuda_device):
    p = torch.nn.Parameter(torch.zeros(10, device="cuda"))
    p.grad = torch.full_like(p, 3e38)
    p.grad[3] = math.inf
    opt = Lion([p], max_grad_norm=1.0)
    opt.step()
    assert opt.grad_norm.item() == math.inf and grad_norm([p.grad]).item() == math.inf
    assert torch.isnan(opt.state[p]["exp_avg"][3]) and (opt.state[p]["exp_avg"][:3] == 0).all()
