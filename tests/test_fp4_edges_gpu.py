"""4-bit products at the edges: kernels that end right after they begin, factors at both ends of fp32, sums that are
exact."""
import pytest
import torch

pytestmark = pytest.mark.gpu
dev = "cuda"


def _ops():
    from dmad_b200 import ops
    assert ops.native_available()
    return ops


def test_one_tile_a_pair_back_to_back_on_two_streams():
    """One tile a pair and one K step a tile: the second CTA of a pair is done as soon as it can be, while the leader's
    last arrivals in its shared memory are on their way; the next kernel takes that memory at once."""
    ops = _ops()
    torch.manual_seed(0)
    w = ops.quantize_fp4(torch.randn(16512, 32, device=dev), "mxfp4")
    xs = [ops.quantize_fp4(torch.randn(256, 32, device=dev), "mxfp4") for _ in range(2)]
    wv = ops.dequantize_fp4(w, torch.float32).double()
    # codes are multiples of half a scale: 32 products and their fp32 sums, then half a bf16 step
    want = [ops.dequantize_fp4(x, torch.float32).double() @ wv.t() for x in xs]
    size = [ops.dequantize_fp4(x, torch.float32).double().abs() @ wv.abs().t() for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(40):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.fp4_linear(xs[i], w))
    torch.cuda.synchronize()
    ops.check_device_status()
    for g, r, s in zip(got, want, size):
        assert ((g[0].double() - r).abs() <= 2.0 ** -8 * r.abs() + 40 * 2.0 ** -23 * s).all()
        assert all(torch.equal(g[0], o) for o in g)


def _ends(M, K, dtype):
    """Rows of 1e34 to 1e37, of 1e-30 to 1e-38 and ordinary ones, in turn."""
    g = torch.Generator(device=dev).manual_seed(M)
    x = torch.randn(M, K, device=dev, generator=g).clamp(-4, 4)
    size = torch.tensor([1e34, 1.0, 1e36, 1e-30, 1e37, 1e-37, 3e28, 1e-21], device=dev)
    return (x * size[torch.arange(M, device=dev) % 8][:, None]).to(dtype)


@pytest.mark.parametrize("M,N,K", [(1, 300, 512), (9, 640, 5120), (200, 1000, 1000), (300, 16500, 700), (520, 8200, 96)])
@pytest.mark.parametrize("wsize,factor", [(0.02, None), (1e-30, None), (1e30, None), (0.02, 1.7e-38), (0.02, 3.3e30),
                                          (0.02, 1e-41)])
def test_factors_at_the_ends_of_fp32(M, N, K, wsize, factor):
    """The row's factor and the weight's multiply without an overflow, or a loss of digits, that the result has not.
    ``factor``: one stored for all rows of the weight."""
    ops = _ops()
    x = ops.quantize_fp4(_ends(M, K, torch.bfloat16), "nvfp4")
    w = ops.quantize_fp4(wsize * torch.randn(N, K, device=dev, generator=torch.Generator(device=dev).manual_seed(N)), "nvfp4")
    if factor is not None:
        w.row_scale = torch.full((N,), factor, device=dev)
    b = torch.randn(N, device=dev)
    for bias in (None, b):
        y = ops.fp4_linear(x, w, bias).double()
        ops.check_device_status()
        # the values in 64 bits from the codes at factors of one
        one = [ops.dequantize_fp4(ops.Fp4Tensor(q.data, q.scales, torch.ones_like(q.row_scale), "nvfp4", q.shape),
                                  torch.float32).double() for q in (x, w)]
        f = x.row_scale.double()[:, None] * w.row_scale.double()
        ref, size = (one[0] @ one[1].t()) * f, (one[0].abs() @ one[1].abs().t()) * f
        if bias is not None:
            ref, size = ref + bias.double(), size + bias.double().abs()
        # half a bf16 step (of a subnormal: 2^-134), a truncation of the running size at each product and the factors, and
        # fp32's own smallest step (2^-149) at two of the multiplications
        bound = 2.0 ** -8 * ref.abs() + 2.0 ** -134 + 2.0 ** -148 + (K + 8) * 2.0 ** -23 * size
        top = torch.finfo(torch.bfloat16).max * (1 + 2.0 ** -9)  # what rounds to infinity
        sure, never = ref.abs() - bound > top, ref.abs() + bound < top
        assert not torch.isnan(y).any()
        assert torch.isinf(y[sure]).all() and (torch.sign(y[sure]) == torch.sign(ref[sure])).all()
        assert torch.isfinite(y[never]).all()
        ok = torch.isfinite(y)
        assert ((y - ref).abs()[ok] <= bound[ok]).all()
        if factor is None and wsize == 0.02:
            assert never.all()


def test_large_rows_match_the_cpu():
    """bf16 rows of 1e36 against weights of 0.02: finite, as on the CPU."""
    ops = _ops()
    x = (torch.randn(3, 1000, generator=torch.Generator().manual_seed(0)) * 1e36).bfloat16()
    w = ops.quantize_fp4(0.02 * torch.randn(300, 1000, generator=torch.Generator().manual_seed(1)), "nvfp4")
    want = ops.fp4_linear(x, w).double()
    got = ops.fp4_linear(x.to(dev), w.to(dev)).double().cpu()
    assert torch.isfinite(want).all() and torch.isfinite(got).all()
    # both round fp32 sums of the same values once: a bf16 step apart at most, and the sums' own rounding
    size = want.abs().amax()
    assert ((got - want).abs() <= 2.0 ** -7 * want.abs() + 1000 * 2.0 ** -22 * size).all()


@pytest.mark.parametrize("M,N,K", [(3, 300, 512), (9, 640, 2048), (300, 16500, 704)])
@pytest.mark.parametrize("wsize", [1e-37, 1e-30, 1e30])
def test_mxfp4_scales_at_the_ends_of_fp32(M, N, K, wsize):
    """Block scales of 2^120 and of 2^-127 on either side: the products are those of the values."""
    ops = _ops()
    x = ops.quantize_fp4(_ends(M, K, torch.bfloat16), "mxfp4")
    w = ops.quantize_fp4(wsize * torch.randn(N, K, device=dev, generator=torch.Generator(device=dev).manual_seed(N)), "mxfp4")
    y = ops.fp4_linear(x, w).double()
    ops.check_device_status()
    xv, wv = (ops.dequantize_fp4(q, torch.float32).double() for q in (x, w))
    ref, size = xv @ wv.t(), xv.abs() @ wv.abs().t()
    # half a bf16 step (2^-134 of the smallest) and a truncation of the running size, or of fp32's smallest step (or its
    # smallest normal number, should the accumulator have no smaller ones), at each product
    bound = 2.0 ** -8 * ref.abs() + 2.0 ** -134 + (K + 8) * (2.0 ** -23 * size + 2.0 ** -126)
    fits = size < 2.0 ** 127  # no partial sum leaves fp32
    assert fits.any() and torch.isfinite(y[fits]).all()
    assert ((y - ref).abs()[fits] <= bound[fits]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_non_finite_blocks_of_16_bit_rows(fmt, dtype):
    """The bytes of rows with infinities, NaN of either sign and zeros, against the CPU."""
    ops = _ops()
    x = torch.randn(200, 100, generator=torch.Generator().manual_seed(0)).to(dtype)
    x[0, 3], x[1, 40], x[2, 99] = float("inf"), -float("inf"), float("nan")
    x[3] = float("nan")
    x[4] = 0.0
    x[5, ::2] = -0.0
    x[6] = torch.finfo(dtype).max
    x[7] = torch.finfo(dtype).smallest_normal / 4
    x.view(torch.int16)[8, 5] = -1  # a NaN with its sign set
    got, want = ops.quantize_fp4(x.to(dev), fmt), ops.quantize_fp4(x, fmt)
    assert torch.equal(got.data.cpu(), want.data) and torch.equal(got.scales.cpu(), want.scales)
    assert want.row_scale is None or torch.equal(got.row_scale.cpu(), want.row_scale)
