"""8-bit integer codes and products on the CPU, against their definition in fp64; refusals."""
import pytest
import torch

from dmad_b200 import ops
from dmad_b200.ops.int8 import INT8_MAX_K
from tests import _int8_oracle as oracle

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _matrix(R, K, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, K, generator=g) * torch.exp2(torch.randint(-12, 12, (R, 1), generator=g).float())
    x[:, ::7] *= 16
    if R > 3:
        x[1] = 0
        x[2, K // 2:] = 0
        x[3] = torch.randint(-127, 128, (K,), generator=g).float() / 2  # quotients on halves
        x[3, 0] = 127.0
    return x.to(DT[dtype])


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("R,K", [(1, 1), (1, 31), (5, 32), (4, 33), (7, 100), (9, 512)])
@pytest.mark.parametrize("block", [0, 32])
def test_codes_are_the_definition(R, K, dtype, block):
    x = _matrix(R, K, dtype)
    q = ops.quantize_int8(x, block)
    assert q.data.shape == (R, (K + 31) // 32 * 32) and not q.data[:, K:].any()
    if block:
        c, e = oracle.blocks(x)
        assert torch.equal(q.scale.double(), e)
    else:
        c, s = oracle.rows(x)
        assert torch.equal(q.scale.double(), s)
    assert torch.equal(q.data[:, :K].double(), c)
    v = ops.dequantize_int8(q, torch.float32)
    assert torch.equal(v, oracle.values(x, block).float())


def test_nearly_half_quotients_are_decided_exactly():
    # x = (n + 1/2) s rounded to fp32, and its neighbours: an fp32 quotient is often exactly n + 1/2
    s = torch.tensor(3.3333333 / 127, dtype=torch.float32)
    x = ((torch.arange(-126, 126).double() + 0.5) * s.double()).float()
    x = torch.cat([x, torch.nextafter(x, torch.tensor(9.0)), torch.nextafter(x, torch.tensor(-9.0)), torch.tensor([3.3333333])])
    q = ops.quantize_int8(x[None], 0)
    assert torch.equal(q.data[0, :x.numel()].double(), oracle.rows(x[None])[0][0])


@pytest.mark.parametrize("block", [0, 32])
def test_ends_of_fp32_and_non_finite_values(block):
    big, tiny = torch.finfo(torch.float32).max, 2.0 ** -149
    x = torch.zeros(7, 64)
    x[0, :40] = torch.linspace(-big, big, 40)  # its step overflows: a row with NaN
    x[6, :40] = torch.linspace(-1, 1, 40) * big
    x[1, :40] = torch.linspace(-1, 1, 40) * 2.0 ** -130
    x[2, 3] = tiny
    x[3], x[4] = torch.randn(64), torch.randn(64)
    x[3, 5], x[4, 40] = float("inf"), float("nan")
    q = ops.quantize_int8(x, block)
    v = ops.dequantize_int8(q, torch.float32)
    assert torch.equal(torch.nan_to_num(v, nan=7.0), torch.nan_to_num(oracle.values(x, block).float(), nan=7.0))
    bad = 64 if block == 0 else 32
    assert v[3, :bad].isnan().all() and v[4, 64 - bad:].isnan().all() and not v[[1, 2, 5, 6]].isnan().any()
    assert v[0, :32].isnan().all() and v[6].isfinite().all()


def test_leading_dimensions_and_empty():
    x = torch.randn(2, 3, 40)
    for block in (0, 32):
        q = ops.quantize_int8(x, block)
        assert q.shape == (2, 3, 40) and q.rows == 6 and ops.dequantize_int8(q).shape == (2, 3, 40)
        e = ops.quantize_int8(x[:0], block)
        assert e.rows == 0 and ops.dequantize_int8(e).shape == (0, 3, 40)
    assert ops.dequantize_int8(ops.quantize_int8(torch.randn(40)), torch.float32).shape == (40,)


@pytest.mark.parametrize("bias", [None, "fp32", "bf16"])
def test_linear_is_the_product_of_the_coded_values(bias):
    x, w = _matrix(6, 100, "bf16"), _matrix(11, 100, "fp32", 1)
    b = None if bias is None else torch.randn(11).to(DT[bias])
    qw = ops.quantize_int8(w)
    y = ops.int8_linear(x.view(2, 3, 100), qw, b)
    want = oracle.values(x, 0) @ oracle.values(w, 0).t()
    want = want if b is None else want + b.double()
    assert y.shape == (2, 3, 11) and y.dtype == torch.bfloat16
    assert torch.equal(y.view(6, 11), want.to(torch.bfloat16))
    assert torch.equal(ops.int8_linear(ops.quantize_int8(x), qw, b, torch.float16), want.to(torch.float16))
    assert ops.int8_linear(x[:0], qw, b).shape == (0, 11)
    part = ops.int8_linear(x, qw.row_slice(3, 7), None if b is None else b[3:7])
    assert torch.equal(part, want[:, 3:7].to(torch.bfloat16))


def test_refusals():
    x, w = torch.randn(4, 64), ops.quantize_int8(torch.randn(8, 64))
    xb = x.to(torch.bfloat16)
    for bad in (lambda: ops.quantize_int8(x.double()), lambda: ops.quantize_int8(x, 16), lambda: ops.quantize_int8(torch.tensor(1.0)),
                lambda: ops.quantize_int8(torch.zeros(3, 0)), lambda: ops.dequantize_int8(w, torch.float64),
                lambda: ops.int8_linear(x, w), lambda: ops.int8_linear(xb[:, :32], w),
                lambda: ops.int8_linear(xb, ops.quantize_int8(torch.randn(8, 64), 32)),
                lambda: ops.int8_linear(ops.quantize_int8(xb, 32), w), lambda: ops.int8_linear(xb, w, torch.randn(7)),
                lambda: ops.int8_linear(xb, w, torch.randn(8).double()), lambda: ops.int8_linear(xb, w, None, torch.float32),
                lambda: ops.int8_linear(xb, ops.Int8Tensor(w.data[:, :32], w.scale, 0, (8, 64))),
                lambda: ops.int8_linear(xb, ops.Int8Tensor(w.data, w.scale[:4], 0, (8, 64))),
                lambda: ops.int8_linear(xb, ops.Int8Tensor(w.data, w.scale, 0, (2, 4, 64))),
                lambda: w.row_slice(5, 9), lambda: w.row_slice(3, 2)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ValueError, match="int32 sums"):
        K = INT8_MAX_K + 1
        ops.int8_linear(torch.zeros(1, K, dtype=torch.bfloat16), ops.Int8Tensor(
            torch.zeros(1, -(-K // 32) * 32, dtype=torch.int8), torch.ones(1), 0, (1, K)))
    for t in (x.requires_grad_(True), ):
        with pytest.raises(RuntimeError, match="forward only"):
            ops.quantize_int8(t)
    with pytest.raises(RuntimeError, match="forward only"):
        ops.int8_linear(xb.clone().requires_grad_(True), w)
    with torch.no_grad():
        ops.quantize_int8(x)
    with torch.autograd.forward_ad.dual_level():
        d = torch.autograd.forward_ad.make_dual(torch.randn(2, 32), torch.randn(2, 32))
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.quantize_int8(d)
