"""The sums of the 4-bit products, at long K where a bound on each element's worst case says little: sums that are
exact, bit for bit, and errors as a whole."""
import pytest
import torch

from tests import _fp4_oracle as oracle

pytestmark = pytest.mark.gpu
dev = "cuda"

SIZES = [(1, 300, 5120), (16, 256, 5120), (100, 1000, 2048), (256, 640, 15360), (129, 257, 1000), (300, 1543, 129),
         (130, 20000, 96), (257, 40000, 4100), (520, 8200, 1543)]


def _ops():
    from dmad_b200 import ops
    assert ops.native_available()
    return ops


def _exact(R, K, fmt, top, seed):
    """Rows of half-integers times a power of two of each block, which their 4-bit form keeps: the first element of a
    block is 6 of its scales."""
    g = torch.Generator(device=dev).manual_seed(seed)
    blk = oracle.BLOCK[fmt]
    nb = -(-K // blk)
    v = torch.tensor(oracle.LEVELS, device=dev)[torch.randint(0, 8, (R, nb, blk), device=dev, generator=g)]
    v[:, :, 0] = 6.0
    v = v * (1.0 - 2.0 * torch.randint(0, 2, v.shape, device=dev, generator=g))
    v = v * 2.0 ** torch.randint(0, top + 1, (R, nb, 1), device=dev, generator=g)
    return v.reshape(R, nb * blk)[:, :K].contiguous()


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_exact_sums_are_rounded_once(fmt, M, N, K):
    """Every product is a multiple of 1/4 and all partial sums stay below 2^22, so fp32 holds each of them whatever their
    order: the result is the sum rounded to bf16, and one wrong scale, code or rounding on the way shows."""
    ops = _ops()
    x, w = _exact(M, K, fmt, 2, M), _exact(N, K, fmt, 1, N + 1)
    b = torch.randint(-8, 9, (N,), device=dev).float() / 4
    xq, wq = ops.quantize_fp4(x, fmt), ops.quantize_fp4(w, fmt)
    assert torch.equal(ops.dequantize_fp4(xq, torch.float32), x) and torch.equal(ops.dequantize_fp4(wq, torch.float32), w)
    assert (x.double().abs() @ w.double().abs().t()).max() + 2 < 2.0 ** 22
    for bias in (None, b):
        y = ops.fp4_linear(xq, wq, bias)
        ref = x.double() @ w.double().t()
        ref = ref if bias is None else ref + bias.double()
        assert torch.equal(y, ref.to(torch.float32).to(torch.bfloat16))  # fp32 holds ref
        assert torch.equal(ops.fp4_linear(x.bfloat16(), wq, bias), y)
    ops.check_device_status()


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("M,N,K", [s for s in SIZES if s[0] * s[1] >= 4000])
def test_errors_as_a_whole(fmt, M, N, K):
    """A bf16 rounding is off by 2^-8 of the value at most and, over evenly spread significands, by 0.42 x 2^-8 in the
    mean square; sums of a thousand and more numbers stay within a few per cent of that, and an accumulator that rounds
    between steps does not.  fp32 sums add a truncation of 2^-23 of the running sum (of the result's size) at each of the
    K / 64 steps."""
    ops = _ops()
    g = torch.Generator(device=dev).manual_seed(K)
    xq = ops.quantize_fp4(torch.randn(M, K, device=dev, generator=g), fmt)
    wq = ops.quantize_fp4(torch.randn(N, K, device=dev, generator=g), fmt)
    ref = ops.dequantize_fp4(xq, torch.float32).double() @ ops.dequantize_fp4(wq, torch.float32).double().t()
    err = ops.fp4_linear(xq, wq).double() - ref
    limit = 0.52 * 2.0 ** -8 + (K / 64 + 8) * 2.0 ** -23
    assert err.norm() <= limit * ref.norm()
    if N >= 1000:
        assert (err.norm(dim=1) <= limit * ref.norm(dim=1)).all()
