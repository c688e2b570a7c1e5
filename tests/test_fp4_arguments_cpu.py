"""Arguments that the 4-bit operators refuse by a ValueError, and not by an error from inside."""
import pytest
import torch

from dmad_b200 import ops


def check_arguments(dev):
    w = ops.quantize_fp4(torch.randn(8, 64, device=dev), "nvfp4")
    point = ops.Fp4Tensor(w.data, w.scales, w.row_scale, "nvfp4", ())
    for f in (lambda: ops.fp4_linear(torch.tensor(1.0, device=dev).bfloat16(), w), lambda: ops.dequantize_fp4(point),
              lambda: ops.fp4_linear(point, w), lambda: ops.quantize_fp4(torch.tensor(1.0, device=dev)),
              lambda: ops.fp4_linear(torch.randn(2, 64, device=dev).bfloat16(), point)):
        with pytest.raises(ValueError):
            f()
    # one row without a dimension of its own, and no rows in the middle
    x = torch.randn(64, device=dev).bfloat16()
    assert torch.equal(ops.fp4_linear(x, w), ops.fp4_linear(x[None], w)[0])
    assert torch.equal(ops.fp4_linear(ops.quantize_fp4(x), w), ops.fp4_linear(x, w))
    e = ops.quantize_fp4(torch.randn(2, 0, 64, device=dev))
    assert ops.dequantize_fp4(e).shape == (2, 0, 64) and ops.fp4_linear(e, w).shape == (2, 0, 8)


def test_shapes_without_columns():
    check_arguments("cpu")
