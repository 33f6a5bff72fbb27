"""The operators' forms for CPU tensors where sums are long and operands out of the ordinary."""
import pytest
import torch

from cbm4gnn_b200.norm import group_norm

from operators64 import SUM, U, assert_within, norm64


@pytest.mark.parametrize("n,c,groups,mean,listed", [(300_000, 4, 1, 1000.0, False), (400_000, 6, 2, 100.0, True)])
def test_norm_of_a_long_sample_beside_a_large_mean(n, c, groups, mean, listed):
    """Of a mean far from 0 no more is lost than its one rounding, and that of x - mean."""
    x = mean + torch.randn((n, c), generator=torch.Generator().manual_seed(6))
    ptr = torch.tensor([0, 0, n]) if listed else None
    y = group_norm(x, groups, ptr=ptr)
    v = x.double().view(n, groups, -1)
    m = v.mean((0, 2), keepdim=True)
    r = (v.var((0, 2), keepdim=True, correction=0) + 1e-5).rsqrt()
    xh = (v - m) * r
    assert_within(y.view(n, groups, -1), xh, r * 2 * U * m.abs() + (SUM + 8 * U) * xh.abs(), "y")


def test_norm_gradient_of_a_long_sample():
    """Sums of a gradient whose terms do not cancel."""
    n, c = 1_000_000, 2
    g = torch.Generator().manual_seed(7)
    x, gy = torch.randn((n, c), generator=g), 30.0 + torch.randn((n, c), generator=g)
    x.requires_grad_(True)
    gx, = torch.autograd.grad(group_norm(x, 1), x, gy)
    want, _ = norm64(x, 1, None, None, [0, n], 1e-5, None, gy)
    # r about 1: u is rounded, its mean too, and what is left of them, about 1, by some operations more
    assert_within(gx, want["gx"], 8 * U * 32 + SUM * want["gx"].abs(), "gx")
