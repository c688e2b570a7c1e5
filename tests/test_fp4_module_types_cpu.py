"""The 16-bit type of a quantised layer follows its module."""
import torch

from dmad_b200 import ops
from dmad_b200.models.layers import SegLinear


def test_layer_computes_in_the_modules_type():
    torch.manual_seed(0)
    lin = SegLinear(64, [("a", 48)], flat_name="").to(torch.bfloat16).quantize_fp4_("nvfp4").requires_grad_(False)
    x = torch.randn(3, 64)
    assert lin(x.bfloat16()).dtype == torch.bfloat16
    lin.half()
    y = lin(x.half())
    assert y.dtype == torch.float16 and lin.effective_weight().dtype == torch.float16
    assert torch.equal(y, ops.fp4_linear(x.half(), lin.fp4, lin.bias))
    lin.float()  # no 16-bit type: it goes on in the last one
    assert lin(x).dtype == torch.float16
    lin.to(torch.bfloat16)
    assert lin(x).dtype == torch.bfloat16 and lin.forward_rows(x, 0, 8).dtype == torch.bfloat16
    net = torch.nn.Sequential(lin, torch.nn.Linear(48, 4).bfloat16()).half()
    assert net(x.half()).dtype == torch.float16
