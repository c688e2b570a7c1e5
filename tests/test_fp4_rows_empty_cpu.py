"""forward_rows past the last row is empty, as a slice of a weight is."""
import torch

from dmad_b200.models.layers import SegLinear


def test_rows_past_the_end_are_empty():
    lin = SegLinear(32, [("a", 200)], flat_name="").bfloat16().requires_grad_(False)
    x = torch.randn(3, 32).bfloat16()
    want = [lin.forward_rows(x, *r).shape for r in ((200, 300), (300, 400), (64, 64))]
    lin.quantize_fp4_("mxfp4")
    assert [lin.forward_rows(x, *r).shape for r in ((200, 300), (300, 400), (64, 64))] == want
