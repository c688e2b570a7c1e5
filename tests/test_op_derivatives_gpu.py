"""Kernels without a derivative refuse what asks for one."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from tests.test_head_norm_gpu import _case

pytestmark = pytest.mark.gpu
dev = "cuda"


def test_dual_tensors_are_refused():
    """No forward-mode derivative: an error, and not a result without its tangent."""
    from dmad_b200 import ops
    q, k, w, c, s = _case(3, 2, 1, 64, 32, 3, torch.bfloat16, torch.float32)
    args = [q, k, *w, c, s]
    for i, t in enumerate(args):
        with fwd.dual_level():
            a = list(args)
            a[i] = fwd.make_dual(t, torch.ones_like(t))
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                    ops.qk_head_norm_rope(*a)
    with fwd.dual_level():  # a level without a dual input is no reason
        assert torch.isfinite(ops.qk_head_norm_rope(*args)[0]).all()
    x = torch.randn(4, 64, device=dev).bfloat16()
    wq = ops.quantize_fp4(torch.randn(8, 64, device=dev))
    for f in (lambda t: ops.fp4_linear(t, wq), lambda t: ops.quantize_fp4(t).data):
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.func.jvp(f, (x,), (torch.ones_like(x),))
    assert torch.isfinite(ops.fp4_linear(x, wq)).all()


def test_row_factors_have_no_derivative():
    from tests.test_op_derivatives_cpu import check_row_scale_refusals
    check_row_scale_refusals(dev)
