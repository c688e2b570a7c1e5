"""Ranges of rows of a 4-bit weight: no more of the product than was asked for, and the same numbers."""
import copy

import pytest
import torch

from dmad_b200 import ops
from dmad_b200.models.layers import SegLinear


def _layer(fmt, out=(300, 212), device="cpu"):
    torch.manual_seed(0)
    return SegLinear(96, [("a", out[0]), ("b", out[1])], flat_name="ab").to(device, torch.bfloat16).quantize_fp4_(fmt)


def check_rows(fmt, device, monkeypatch):
    lin, x = _layer(fmt, device=device), torch.randn(7, 96, device=device).bfloat16()
    lin.bias.data.normal_()
    lin.requires_grad_(False)
    full = lin(x).double()
    seen = []
    real = ops.fp4_linear
    monkeypatch.setattr(ops, "fp4_linear", lambda x, w, *a, **k: seen.append(w.shape[0]) or real(x, w, *a, **k))
    xv, wv = (ops.dequantize_fp4(q, torch.float32).double().abs() for q in (ops.quantize_fp4(x, fmt), lin.fp4))
    size = xv @ wv.t() + lin.bias.double().abs()
    for start, stop in ((0, 512), (0, 300), (300, 512), (256, 384), (384, 385), (511, 600), (130, 130)):
        y = lin.forward_rows(x, start, stop)
        want = full[:, start:stop]
        assert y.shape == want.shape
        # two results of one product: each off by half a bf16 step and a few fp32 sums
        assert ((y.double() - want).abs() <= 2.0 ** -7 * want.abs() + 220 * 2.0 ** -23 * size[:, start:stop]).all()
        assert seen.pop() - (min(stop, 512) - start) < 128 and not seen


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_forward_rows_of_a_quantised_layer(fmt, monkeypatch):
    check_rows(fmt, "cpu", monkeypatch)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_row_slice_is_the_rows(fmt):
    w = ops.quantize_fp4(torch.randn(400, 40), fmt)
    v = ops.dequantize_fp4(w, torch.float32)
    for a, b in ((0, 400), (128, 400), (128, 256), (256, 257), (384, 384)):
        assert torch.equal(ops.dequantize_fp4(w.row_slice(a, b), torch.float32), v[a:b])
    for a, b in ((1, 400), (0, 401), (256, 128), (-128, 128)):
        with pytest.raises(ValueError, match="row_slice"):
            w.row_slice(a, b)
    with pytest.raises(ValueError, match="row_slice"):
        ops.quantize_fp4(torch.randn(2, 200, 40), fmt).row_slice(0, 1)
    with pytest.raises(RuntimeError, match="4-bit"):
        _layer(fmt).seg_weight("a")


def test_row_chunked_blocks_of_a_quantised_model():
    from dmad_b200.inference.lowmem import chunked_block_forward
    from tests.test_fp4_models_cpu import _h3_inputs, _tiny_h3
    m = _tiny_h3().bfloat16().eval().requires_grad_(False)
    m.quantize_fp4_("nvfp4")
    v, a, pe, kw = _h3_inputs()
    c = copy.deepcopy(m)
    for b in c.transformer_blocks:
        b.forward = chunked_block_forward(b, 50)
    with torch.no_grad():
        for x, y in zip(m(v, a, pe, **kw), c(v, a, pe, **kw)):
            # the separate norm and rotation round q and k to bf16 once more (2^-8 of each), and a number at a border of two
            # 4-bit codes may go to the other one: a sixth of its size at most, of few numbers
            assert (x - y).norm() <= 5e-2 * x.norm()
