"""Block-scaled 4-bit formats on the CPU: the restatement against a search over the representable numbers, the
storage layout, and every refusal."""
import pytest
import torch

from dmad_b200 import ops
from dmad_b200.ops.fp4 import Fp4Tensor, fp4_storage_shapes
from tests import _fp4_oracle as oracle


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("R,K,kind", [(1, 1, "normal"), (3, 33, "normal"), (130, 160, "grid"), (7, 71, "grid"),
                                      (2, 1000, "normal")])
def test_values_are_the_nearest_ones(fmt, dtype, R, K, kind):
    x = oracle.inputs(R, K, dtype, seed=R + K, kind=kind)
    q = ops.quantize_fp4(x, fmt)
    v, codes, row = oracle.values(x, fmt)
    assert torch.equal(ops.dequantize_fp4(q, torch.float32).double(), v)
    if fmt == "nvfp4":
        assert torch.equal(q.row_scale.double(), row)
    # byte of block b of row r as the layout's description says
    for r in (0, R // 2, R - 1):
        for b in range(codes.shape[1]):
            assert int(q.scales[r // 128, b // 4, (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4]) == int(codes[r, b])


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_padding_is_zero(fmt):
    R, K = 5, 37
    q = ops.quantize_fp4(torch.randn(R, K), fmt)
    assert (tuple(q.data.shape), tuple(q.scales.shape)) == fp4_storage_shapes(R, K, fmt)
    assert int(q.data[:, 18].max()) < 16 and int(q.data[:, 19:].max()) == 0
    nb = -(-K // oracle.BLOCK[fmt])
    tile = q.scales.view(1, -1, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(128, -1)
    assert int(tile[R:].max()) == 0 and (tile.shape[1] == nb or int(tile[:, nb:].max()) == 0)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_zeros_extremes_and_non_finite_blocks(fmt):
    blk = oracle.BLOCK[fmt]
    x = torch.zeros(6, 4 * blk)
    x[1, 0] = 1e-40                                  # a subnormal
    x[2, 0], x[2, blk] = 3.0e38, -1.0e-30            # both ends of fp32 in one row
    x[3, 0], x[3, blk], x[3, 2 * blk] = float("inf"), float("nan"), 2.0
    x[4] = -float("inf")
    x[5, 1] = -0.0
    got = ops.dequantize_fp4(ops.quantize_fp4(x, fmt), torch.float32).double()
    want, _, _ = oracle.values(x, fmt)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
    assert torch.isnan(got[3, :2 * blk]).all() and torch.isfinite(got[3, 2 * blk:]).all() and torch.isnan(got[4]).all()


def test_leading_dimensions_and_empty_rows():
    x = torch.randn(2, 3, 48)
    q = ops.quantize_fp4(x, "nvfp4")
    assert ops.dequantize_fp4(q).shape == x.shape and q.rows == 6
    e = ops.quantize_fp4(torch.randn(0, 48), "mxfp4")
    assert ops.dequantize_fp4(e).shape == (0, 48) and e.data.shape == (0, 32)
    w = ops.quantize_fp4(torch.randn(5, 48), "mxfp4")
    assert ops.fp4_linear(torch.randn(0, 48).bfloat16(), w).shape == (0, 5)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_linear_is_the_product_of_the_coded_values(fmt):
    x, w, b = torch.randn(3, 4, 100).bfloat16(), torch.randn(7, 100), torch.randn(7)
    wq = ops.quantize_fp4(w, fmt)
    y = ops.fp4_linear(x, wq, b)
    xv, wv = oracle.values(x.reshape(12, 100), fmt)[0], oracle.values(w, fmt)[0]
    ref = (xv @ wv.t() + b.double()).view(3, 4, 7)
    size = (xv.abs() @ wv.abs().t() + b.double().abs()).view(3, 4, 7)
    # one rounding to bf16 (half a step: 2^-8 of the value) and at most 101 fp32 additions of 2^-24 of their size
    assert ((y.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 110 * 2.0 ** -24 * size).all()
    assert torch.equal(ops.fp4_linear(ops.quantize_fp4(x, fmt), wq, b), y)


def test_refusals():
    x = torch.randn(4, 64).bfloat16()
    w = ops.quantize_fp4(torch.randn(8, 64), "nvfp4")
    bad = [lambda: ops.quantize_fp4(x, "fp4"), lambda: ops.quantize_fp4(x.double(), "mxfp4"),
           lambda: ops.quantize_fp4(x.int(), "mxfp4"), lambda: ops.quantize_fp4(torch.randn(4, 0), "mxfp4"),
           lambda: ops.quantize_fp4(torch.tensor(1.0), "mxfp4"),
           lambda: ops.dequantize_fp4(w, torch.float64), lambda: ops.fp4_linear(x.float(), w),
           lambda: ops.fp4_linear(x[:, :32], w), lambda: ops.fp4_linear(ops.quantize_fp4(x, "mxfp4"), w),
           lambda: ops.fp4_linear(x, w, torch.randn(7)), lambda: ops.fp4_linear(x, w, torch.zeros(8).double()),
           lambda: ops.fp4_linear(x, w, out_dtype=torch.float32),
           lambda: ops.fp4_linear(x, ops.quantize_fp4(torch.randn(2, 4, 64), "nvfp4")),
           lambda: ops.dequantize_fp4(Fp4Tensor(w.data[:, :16], w.scales, w.row_scale, "nvfp4", (8, 64))),
           lambda: ops.dequantize_fp4(Fp4Tensor(w.data, w.scales, w.row_scale, "nvfp4", (8, 80))),
           lambda: ops.dequantize_fp4(Fp4Tensor(w.data, w.scales[:, :0], w.row_scale, "nvfp4", (8, 64))),
           lambda: ops.dequantize_fp4(Fp4Tensor(w.data, w.scales, None, "nvfp4", (8, 64))),
           lambda: ops.dequantize_fp4(Fp4Tensor(w.data, w.scales, w.row_scale.double(), "nvfp4", (8, 64))),
           lambda: ops.dequantize_fp4(Fp4Tensor(w.data.int(), w.scales, w.row_scale, "nvfp4", (8, 64)))]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    g = x.clone().requires_grad_(True)
    for f in (lambda: ops.quantize_fp4(g), lambda: ops.fp4_linear(g, w),
              lambda: ops.fp4_linear(x, w, torch.zeros(8, requires_grad=True))):
        with pytest.raises(RuntimeError, match="forward only"):
            f()
    with torch.no_grad():
        assert ops.fp4_linear(g, w).shape == (4, 8)


def test_native_checks_raise():
    """The extension's own checks end in a Python error, numbers in their messages included."""
    if not ops.native_available():
        pytest.skip("extension not built")
    e = ops.ext()
    x = torch.randn(4, 64)
    q = ops.quantize_fp4(torch.randn(8, 64))
    z = torch.randn(4, 2, 16)
    for f in (lambda: e.fp4_quantize(x, True),
              lambda: e.fp4_dequantize(q.data[:4], q.scales, q.row_scale, 8, 64, True, 0),
              lambda: e.fp4_dequantize(q.data, q.scales[:, :0], q.row_scale, 8, 64, True, 0),
              lambda: e.fp4_dequantize(q.data, q.scales, q.row_scale[:4], 8, 64, True, 0),
              lambda: e.fp4_dequantize(q.data, q.scales, None, 8, 64, True, 0),
              lambda: e.fp4_dequantize(q.data, q.scales, q.row_scale, 8, 64, True, 0),
              lambda: e.fp4_linear(x.bfloat16(), q.data, q.scales, q.row_scale, None, 8, 64, True, -1),
              lambda: e.fp4_matmul(q.data, q.scales, q.row_scale, 8, q.data, q.scales, q.row_scale, None, 8, 64, True, 0),
              lambda: e.head_norm_rope_fwd(x, x, None, None, None, None, None, 1e-6, True),
              lambda: e.head_norm_rope_fwd(z, z[:3], None, None, None, None, None, 1e-6, True),
              lambda: e.head_norm_rope_fwd(z, z, None, None, None, None, None, 1e-6, True)):
        with pytest.raises(ValueError):
            f()
