"""linear_act8 on the CPU: the forward pass, the gradients against the formulas in fp64 and against differences, refusals."""
import pytest
import torch

from dmad_b200 import ops
from tests import _int8_oracle as oracle

ACTS = (None, "gelu_tanh", "swiglu")


def act64(h, act):
    if act == "gelu_tanh":
        return 0.5 * h * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (h + 0.044715 * h ** 3)))
    if act == "swiglu":
        v, u = h.chunk(2, dim=-1)
        return v * u / (1 + torch.exp(-u))
    return h


def kept64(x, act):
    if act == "swiglu":
        return torch.cat([oracle.values(h, 32) for h in x.chunk(2, dim=-1)], dim=-1)
    return oracle.values(x, 32)


def reference(x, w, b, g, act):
    """y and the gradients in fp64: those at the kept values."""
    y = act64(x.double(), act) @ w.double().t()
    y = y if b is None else y + b.double()
    xk, w64 = kept64(x, act).requires_grad_(True), w.double().requires_grad_(True)
    dx, dw = torch.autograd.grad(act64(xk, act) @ w64.t(), (xk, w64), g.double())
    return y, dx, dw, g.double().sum(0)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("R,N,F", [(1, 1, 1), (5, 7, 33), (40, 24, 64)])
def test_gradients_are_those_at_the_kept_values(act, R, N, F):
    g = torch.Generator().manual_seed(R)
    x = torch.randn(R, F * (2 if act == "swiglu" else 1), generator=g, requires_grad=True)
    w = torch.randn(N, F, generator=g, requires_grad=True)
    b = torch.randn(N, generator=g, requires_grad=True)
    gy = torch.randn(R, N, generator=g)
    y = ops.linear_act8(x, w, b, act)
    got = (y, *torch.autograd.grad(y, (x, w, b), gy))
    for a, r in zip(got, reference(x.detach(), w.detach(), b.detach(), gy, act)):
        assert a.shape == r.shape
        torch.testing.assert_close(a.double(), r, rtol=1e-4, atol=1e-4)  # fp32 sums of up to 64 numbers of size 10


@pytest.mark.parametrize("act", ACTS)
def test_gradients_against_differences(act):
    # inputs that the code holds exactly: whole numbers of a block's step
    g = torch.Generator().manual_seed(3)
    R, N, F = 3, 5, 64
    x = torch.randint(-90, 91, (R, F * (2 if act == "swiglu" else 1)), generator=g).double() / 64
    x[:, ::32] = 100 / 64.0
    assert torch.equal(kept64(x, act), x)
    w, gy = torch.randn(N, F, generator=g).double(), torch.randn(R, N, generator=g).double()
    xf, wf = x.float().requires_grad_(True), w.float().requires_grad_(True)
    y = ops.linear_act8(xf, wf, None, act)
    dx, dw = torch.autograd.grad(y, (xf, wf), gy.float())
    h = 1e-5
    loss = lambda x, w: (act64(x, act) @ w.t() * gy).sum()
    for t, d, at in ((x, dx, 0), (w, dw, 1)):
        for i in range(0, t.numel(), 17):
            e = torch.zeros_like(t).reshape(-1)
            e[i] = h
            e = e.reshape(t.shape)
            diff = (loss(x + e, w) - loss(x - e, w)) if at == 0 else (loss(x, w + e) - loss(x, w - e))
            assert abs(diff / (2 * h) - d.reshape(-1)[i].double()) < 1e-3


def test_shapes_types_and_what_is_kept():
    x = torch.randn(2, 3, 40, dtype=torch.bfloat16, requires_grad=True)
    w, b = torch.randn(8, 40, dtype=torch.bfloat16, requires_grad=True), torch.randn(8, requires_grad=True)
    y = ops.linear_act8(x, w, b, "gelu_tanh")
    assert y.shape == (2, 3, 8) and y.dtype == torch.bfloat16
    y.float().sum().backward()
    assert x.grad.dtype == w.grad.dtype == torch.bfloat16 and b.grad.dtype == torch.float32 and x.grad.shape == x.shape
    with torch.no_grad():
        assert torch.equal(ops.linear_act8(x, w, b, "gelu_tanh"), y)
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
        ops.linear_act8(x, w, b)
    assert all(t is None or t.dtype in (torch.int8, torch.uint8) or t.shape == w.shape for t in saved)
    empty = ops.linear_act8(x[:0], w, b)
    assert empty.shape == (0, 3, 8)
    d = torch.autograd.grad(empty, (w, b), torch.zeros(0, 3, 8, dtype=torch.bfloat16))
    assert not d[0].any() and not d[1].any()


def test_refusals():
    x, w = torch.randn(4, 32), torch.randn(8, 32)
    for bad in (lambda: ops.linear_act8(x, w, None, "relu"), lambda: ops.linear_act8(x.double(), w.double()),
                lambda: ops.linear_act8(x, w.half()), lambda: ops.linear_act8(x, w[0]), lambda: ops.linear_act8(x[:, :31], w),
                lambda: ops.linear_act8(x, w, None, "swiglu"), lambda: ops.linear_act8(x, w, torch.zeros(7)),
                lambda: ops.linear_act8(x, w, torch.zeros(8).double()), lambda: ops.linear_act8(torch.tensor(1.0), w[:, :0])):
        with pytest.raises(ValueError):
            bad()
    with torch.autograd.forward_ad.dual_level():
        d = torch.autograd.forward_ad.make_dual(x, x)
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.linear_act8(d, w)
    x.requires_grad_(True)
    dx, = torch.autograd.grad(ops.linear_act8(x, w).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
