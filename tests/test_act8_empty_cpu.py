"""linear_act8 on the CPU without rows, and without outputs."""
import pytest
import torch

from dmad_b200 import ops


@pytest.mark.parametrize("act", [None, "gelu_tanh", "swiglu"])
@pytest.mark.parametrize("lead,N", [((5,), 0), ((), 0), ((2, 0), 4), ((0,), 0), ((), 4)])
def test_empty(lead, N, act):
    x = torch.randn(*lead, 80 if act == "swiglu" else 40, requires_grad=True)
    w, b = torch.randn(N, 40, requires_grad=True), torch.randn(N, requires_grad=True)
    y = ops.linear_act8(x, w, b, act)
    assert y.shape == (*lead, N)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert dx.shape == x.shape and dw.shape == w.shape and db.shape == b.shape
    if y.numel() == 0:
        assert not dx.any() and not dw.any() and not db.any()
