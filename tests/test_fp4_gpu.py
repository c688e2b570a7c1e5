"""4-bit kernels: the quantiser's bytes against the CPU restatement, the GEMM against 64 bits, streams, graphs and
refusals."""
import pytest
import torch

from tests import _fp4_oracle as oracle

pytestmark = pytest.mark.gpu
dev = "cuda"


def _ops():
    from dmad_b200 import ops
    assert ops.native_available()
    return ops


def _same(a, b):
    """Equal storage: data, scales, row scales, byte for byte."""
    assert torch.equal(a.data.cpu(), b.data) and torch.equal(a.scales.cpu(), b.scales)
    assert (a.row_scale is None) == (b.row_scale is None)
    if a.row_scale is not None:
        assert torch.equal(a.row_scale.cpu(), b.row_scale)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("R,K,kind", [(1, 1, "normal"), (1, 5120, "normal"), (3, 33, "grid"), (129, 16, "grid"),
                                      (200, 544, "grid"), (5, 1543, "normal"), (2, 16400, "grid"), (2, 40000, "normal")])
def test_quantize_gives_the_cpu_bytes(fmt, dtype, R, K, kind):
    ops = _ops()
    x = oracle.inputs(R, K, dtype, seed=R * 7 + K, kind=kind)
    q = ops.quantize_fp4(x.to(dev), fmt)
    ref = ops.quantize_fp4(x, fmt)
    _same(q, ref)
    for t in (torch.float32, torch.bfloat16):
        assert torch.equal(ops.dequantize_fp4(q, t).cpu(), ops.dequantize_fp4(ref, t))
    assert torch.equal(ops.dequantize_fp4(q, torch.float16).cpu(), ops.dequantize_fp4(ref, torch.float16))


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_extremes_and_strides(fmt, dtype):
    ops = _ops()
    blk = oracle.BLOCK[fmt]
    x = torch.zeros(7, 4 * blk)
    x[1, 0] = 1e-40
    x[2, 0], x[2, blk] = 3.0e38, -1.0e-30
    x[3, 0], x[3, blk], x[3, 2 * blk] = float("inf"), float("nan"), 2.0
    x[4] = -float("inf")
    x[5, 1] = -0.0
    x[6] = torch.randn(4 * blk) * 1e-38
    x = x.to(dtype)
    _same(ops.quantize_fp4(x.to(dev), fmt), ops.quantize_fp4(x, fmt))
    big = torch.randn(40, 300).to(dtype)
    for v in (big[:, 8:136], big[::3, 1:100], big[1:].t(), big[:, :64].expand(40, 64), big[0].expand(5, 300)):
        _same(ops.quantize_fp4(v.to(dev) if v.is_contiguous() else big.to(dev).as_strided(v.shape, v.stride(),
                                                                                    v.storage_offset()), fmt),
              ops.quantize_fp4(v.contiguous(), fmt))


def _check_linear(ops, M, N, K, fmt, dtype, bias, seed=0):
    x = oracle.inputs(M, K, torch.float32, seed=seed) / 4
    x = x.clamp(-200, 200).to(dtype)
    w = torch.randn(N, K, generator=torch.Generator().manual_seed(seed + 1)).mul(K ** -0.5).to(dtype)
    b = torch.randn(N).to(bias) if bias is not None else None
    xq, wq = ops.quantize_fp4(x.to(dev), fmt), ops.quantize_fp4(w.to(dev), fmt)
    y = ops.fp4_linear(x.to(dev), wq, b.to(dev) if b is not None else None)
    assert torch.equal(ops.fp4_linear(xq, wq, b.to(dev) if b is not None else None, out_dtype=dtype), y)
    torch.cuda.synchronize()
    ops.check_device_status()
    xv = ops.dequantize_fp4(xq, torch.float32).double()
    wv = ops.dequantize_fp4(wq, torch.float32).double()
    ref, size = xv @ wv.t(), xv.abs() @ wv.abs().t()
    if b is not None:
        ref, size = ref + b.to(dev).double(), size + b.to(dev).double().abs()
    # half a step of the output, fp16's smallest step, and one truncation (2^-23) of the running size at each of the
    # K products, the bias and the row factors
    bound = torch.finfo(dtype).eps / 2 * ref.abs() + torch.finfo(dtype).smallest_normal * 2.0 ** -10 + (K + 8) * 2.0 ** -23 * size
    assert y.shape == (M, N) and y.dtype == dtype
    assert ((y.double() - ref).abs() <= bound).all()


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("M,N,K", [(128, 256, 256), (1, 8, 32), (1, 1, 1), (2, 5120, 1536), (16, 256, 5120), (17, 333, 65),
                                   (77, 392, 200), (129, 257, 1000), (300, 1543, 129), (1000, 1536, 1536),
                                   (256, 640, 15360), (130, 20000, 96)])
def test_linear_matches_64_bits(fmt, M, N, K):
    _check_linear(_ops(), M, N, K, fmt, torch.bfloat16, torch.float32, seed=M)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("M,N,K,dtype", [(700, 4500, 1000, torch.bfloat16), (1100, 3001, 520, torch.bfloat16),
                                         (520, 8200, 65, torch.float16), (2500, 5120, 1536, torch.bfloat16),
                                         (385, 16387, 257, torch.float16), (257, 40000, 4100, torch.bfloat16)])
def test_linear_of_many_tiles(fmt, M, N, K, dtype):
    """Sizes that the kernel for pairs of CTAs takes: several tiles a pair, tails of every kind, rows of the output that
    are no multiples of 16 bytes."""
    _check_linear(_ops(), M, N, K, fmt, dtype, torch.float32 if N % 2 else dtype, seed=M)


@pytest.mark.parametrize("M,N", [(127, 128), (128, 129), (129, 128), (129, 4096), (129, 16384), (128, 16512), (256, 8192)])
def test_linear_on_both_sides_of_the_kernel_choice(M, N):
    _check_linear(_ops(), M, N, 320, "nvfp4", torch.bfloat16, None, seed=N)


@pytest.mark.parametrize("fmt,dtype,bias", [("mxfp4", torch.float16, None), ("nvfp4", torch.float16, torch.float16),
                                            ("nvfp4", torch.bfloat16, torch.bfloat16)])
def test_linear_types(fmt, dtype, bias):
    _check_linear(_ops(), 150, 520, 264, fmt, dtype, bias)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("M,N", [(3, 300), (700, 300), (700, 5000)])
def test_linear_non_finite_rows_stay_in_their_rows(fmt, M, N):
    ops = _ops()
    x = torch.randn(M, 512).bfloat16()
    x[1, 5] = float("inf")
    w = torch.randn(N, 512)
    w[7, 100] = float("nan")
    y = ops.fp4_linear(x.to(dev), ops.quantize_fp4(w.to(dev), fmt)).cpu()
    bad = torch.zeros(M, N, dtype=torch.bool)
    bad[1], bad[:, 7] = True, True
    assert torch.equal(torch.isnan(y), bad)


def test_linear_row_factors_of_any_size():
    """A stored weight with one tensor-wide factor that is no power of two."""
    ops = _ops()
    w = ops.quantize_fp4(torch.randn(96, 128, device=dev), "nvfp4")
    x = torch.randn(40, 128, device=dev).bfloat16()
    w.row_scale = torch.full((96,), 0.0137, device=dev)
    y = ops.fp4_linear(x, w).double()
    xv = ops.dequantize_fp4(ops.quantize_fp4(x, "nvfp4"), torch.float32).double()
    wv = ops.dequantize_fp4(w, torch.float32).double()
    ref, size = xv @ wv.t(), xv.abs() @ wv.abs().t()
    assert ((y - ref).abs() <= 2.0 ** -8 * ref.abs() + (128 + 8) * 2.0 ** -23 * size).all()


def test_streams_graphs_and_two_calls_at_once():
    ops = _ops()
    w = ops.quantize_fp4(torch.randn(1536, 1536, device=dev) / 40, "nvfp4")
    xs = [torch.randn(m, 1536, device=dev).bfloat16() for m in (5, 300)]
    want = [ops.fp4_linear(x, w) for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = ops.fp4_linear(xs[i], w)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = xs[1].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.fp4_linear(static, w)
    for x in (xs[1], -xs[1]):
        static.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.fp4_linear(x, w))
    ops.check_device_status()


def test_refusals_on_the_gpu():
    ops = _ops()
    w = ops.quantize_fp4(torch.randn(8, 64, device=dev), "nvfp4")
    x = torch.randn(4, 64, device=dev).bfloat16()
    with pytest.raises(ValueError):
        ops.fp4_linear(x.cpu(), w)
    with pytest.raises(ValueError):
        ops.fp4_linear(x, w, torch.zeros(8))
    with pytest.raises(ValueError):
        ops.dequantize_fp4(ops.Fp4Tensor(w.data, w.scales.cpu(), w.row_scale, "nvfp4", (8, 64)))
    with pytest.raises(ValueError):  # a start that TMA cannot read
        ops.fp4_linear(x, ops.Fp4Tensor(torch.zeros(8 * 32 + 8, dtype=torch.uint8, device=dev)[8:].view(8, 32), w.scales,
                                        w.row_scale, "nvfp4", (8, 64)))
    for f in (lambda: ops.fp4_linear(x[:, :32], w), lambda: ops.fp4_linear(x.float(), w),
              lambda: ops.fp4_linear(ops.quantize_fp4(x[:, :32], "nvfp4"), w), lambda: ops.quantize_fp4(x.double()),
              lambda: ops.quantize_fp4(x[:, :0]), lambda: ops.fp4_linear(x, w, torch.zeros(7, device=dev)),
              lambda: ops.fp4_linear(x, w, torch.zeros(8, device=dev, dtype=torch.double)),
              lambda: ops.dequantize_fp4(ops.Fp4Tensor(w.data, w.scales, None, "nvfp4", (8, 64)))):
        with pytest.raises(ValueError):
            f()
