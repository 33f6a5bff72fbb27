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


@pytest.mark.parametrize("activation", [None, "relu", "silu"])
def test_norm_rows_of_no_sample_have_no_gradient_whatever_they_hold(activation):
    g = torch.Generator().manual_seed(8)
    x, gy = torch.randn((20, 6), generator=g), torch.randn((20, 6), generator=g)
    w, b = (torch.randn(6, generator=g).requires_grad_(True) for _ in range(2))
    x[0], x[17:] = torch.nan, torch.inf
    x.requires_grad_(True)
    y = group_norm(x, 2, w, b, torch.tensor([1, 9, 9, 17]), activation=activation)
    got = torch.autograd.grad(y, (x, w, b), gy)
    inside = x.detach()[1:17].clone().requires_grad_(True)
    alone = group_norm(inside, 2, w, b, torch.tensor([0, 8, 8, 16]), activation=activation)
    want = torch.autograd.grad(alone, (inside, w, b), gy[1:17])
    for t, u in ((y, alone), (got[0], want[0])):
        assert torch.equal(t[1:17], u) and t[0].eq(0).all() and t[17:].eq(0).all()
    # (sums of other rows may be ordered otherwise)
    assert torch.allclose(got[1], want[1], atol=1e-5) and torch.allclose(got[2], want[2], atol=1e-5)
