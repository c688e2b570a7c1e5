"""The gradients of linear_act8 at inputs up to the ends of bf16, where squares and products overflow and the derivative
does not."""
import pytest
import torch

from dmad_b200 import ops

SIZES = (12.0, 40.0, 1e3, 1e10, 1e19, 2e19, 1e25, 3e38)


def far_gelu(R, N, device):
    """x of one size a block of 32 columns (its codes hold it to 2^-7), both signs; w, g."""
    gen = torch.Generator().manual_seed(R + N)
    x = torch.tensor(SIZES).repeat_interleave(32) * (1 - 2 * torch.randint(0, 2, (R, 32 * len(SIZES)), generator=gen))
    w, g = torch.randn(N, x.shape[1], generator=gen), torch.randn(R, N, generator=gen)
    return [t.to(torch.bfloat16).to(device) for t in (x, w, g)]


def check_far_gelu(x, w, g):
    x = x.requires_grad_(True)
    dx, = torch.autograd.grad(ops.linear_act8(x, w, None, "gelu_tanh"), x, g)
    da = g.double() @ w.double()
    # the derivative is 1 or 0 to 10^-60; fp32 sums, and one rounding to bf16
    bound = 2.0 ** -8 * da.abs() + 2.0 ** -23 * (w.shape[0] + 8) * (g.double().abs() @ w.double().abs())
    assert ((dx.double() - torch.where(x > 0, da, torch.zeros_like(da))).abs() <= bound * (x > 0)).all()


@pytest.mark.parametrize("R,N", [(3, 5), (40, 24)])
def test_gelu(R, N):
    check_far_gelu(*far_gelu(R, N, "cpu"))


def test_gelu_slope_against_differences():
    from dmad_b200.ops.act8 import _gelu_slope
    v = torch.linspace(-12, 12, 481, dtype=torch.float64)
    f = lambda t: 0.5 * t * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (t + 0.044715 * t ** 3)))
    h = 1e-5
    assert (_gelu_slope(v) - (f(v + h) - f(v - h)) / (2 * h)).abs().max() <= 1e-8
    assert _gelu_slope(torch.tensor([float("nan")])).isnan().all()


def far_swiglu(R, N, device):
    """Values up to 3e38 beside gates far below zero (slope 0), and gates up to 3e38 beside small values; gradients of 100."""
    gen = torch.Generator().manual_seed(R + N)
    sign = lambda: 1 - 2 * torch.randint(0, 2, (R, 128), generator=gen)
    v = torch.tensor([3e38, 1e30, 1.0, 0.5]).repeat_interleave(32) * sign()
    u = torch.tensor([-200.0, -3e38, 1e30, 3e38]).repeat_interleave(32) * torch.ones(R, 1)
    w, g = torch.randn(N, 128, generator=gen), 100 * torch.randn(R, N, generator=gen)
    return [t.to(torch.bfloat16).to(device) for t in (torch.cat([v, u], 1), w, g)]


def check_far_swiglu(x, w, g):
    x = x.requires_grad_(True)
    dx, = torch.autograd.grad(ops.linear_act8(x, w, None, "swiglu"), x, g)
    dv, du = dx.double().chunk(2, dim=1)
    v = x.detach().double()[:, :128]
    da = g.double() @ w.double()
    err = 2.0 ** -23 * (w.shape[0] + 8) * (g.double().abs() @ w.double().abs())
    assert not dv[:, :64].any() and not du[:, :64].any()  # silu and its slope are 0 to 10^-80
    # the gate's slope is 1 to 10^-80; v's codes are off by 2^-7 of it, and silu(u) = u is larger than bf16 only with da
    assert ((du - da * v)[:, 64:].abs() <= 2.0 ** -6 * (da * v)[:, 64:].abs() + (err * v.abs())[:, 64:]).all()
    assert not dv.isnan().any()


@pytest.mark.parametrize("R,N", [(3, 5), (40, 24)])
def test_swiglu(R, N):
    check_far_swiglu(*far_swiglu(R, N, "cpu"))
