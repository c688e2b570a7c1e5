"""Operators without a derivative refuse what asks for one, in either mode."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from dmad_b200 import ops


def _weight():
    return ops.quantize_fp4(torch.randn(8, 64), "nvfp4")


def _calls(w):
    x, b = torch.randn(4, 64).bfloat16(), torch.randn(8)
    return [(lambda t: ops.quantize_fp4(t).data, x), (lambda t: ops.fp4_linear(t, w), x),
            (lambda t: ops.fp4_linear(x, w, t), b), (lambda t: ops.fp4_linear(ops.quantize_fp4(x), w, t), b)]


@pytest.mark.parametrize("i", range(4))
def test_dual_tensors_are_refused(i):
    f, t = _calls(_weight())[i]
    with fwd.dual_level():
        d = fwd.make_dual(t, torch.ones_like(t))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                f(d)
        f(fwd.unpack_dual(d).primal)  # without its tangent it is an ordinary tensor
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(f, (t,), (torch.ones_like(t),))
    f(t)


def test_norm_carries_tangents_on_the_cpu():
    q, k = torch.randn(3, 2, 16), torch.randn(3, 1, 16)
    d = torch.randn_like(q)
    _, (tq, tk) = torch.func.jvp(lambda x: ops.qk_head_norm_rope(x, k), (q,), (d,))
    h = 2.0 ** -10
    num = (ops.qk_head_norm_rope(q + h * d, k)[0] - ops.qk_head_norm_rope(q - h * d, k)[0]) / (2 * h)
    # a central difference: h^2 times third derivatives of size |d|^3, and fp32 noise over h
    assert (tq - num).abs().max() <= 1e-2 and tk.abs().max() == 0


def _row_scale_calls(dev):
    """Calls with a stored factor that wants a derivative."""
    x, w = torch.randn(4, 64, device=dev).bfloat16(), ops.quantize_fp4(torch.randn(8, 64, device=dev), "nvfp4")
    xq = ops.quantize_fp4(x, "nvfp4")

    def coded(q, rs):
        return ops.Fp4Tensor(q.data, q.scales, rs, q.fmt, q.shape)

    return [(lambda rs: ops.dequantize_fp4(coded(w, rs)), w.row_scale), (lambda rs: ops.fp4_linear(x, coded(w, rs)), w.row_scale),
            (lambda rs: ops.fp4_linear(coded(xq, rs), w), xq.row_scale)]


def check_row_scale_refusals(dev):
    for f, rs in _row_scale_calls(dev):
        leaf = rs.clone().requires_grad_(True)
        with pytest.raises(RuntimeError, match="forward only"):
            f(leaf)
        with torch.no_grad():
            assert torch.equal(f(leaf), f(rs))
        with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            f(fwd.make_dual(rs, torch.ones_like(rs)))


def test_row_factors_have_no_derivative():
    check_row_scale_refusals("cpu")
